// Products of rows of 8-bit codes, out[m, n] = (X W^T)[m, n] x_scales[m] w_scales[n] and its epilogues, and scores of given tokens straight from a head's product.
//
// The sums are whole numbers of 32 bits on the tensor cores (tcgen05 kind::i8): exact in any order, so parts of K add up to the same bits however they are cut.  Both operands
// lie in rows along K and come as blocks of 128 bytes of 128 or 256 rows, TMA's 128-byte swizzle: 128 codes, or 64 entries of bf16 where the head's scores take those.
//
// tile_kernel: persistent, one block (or a pair of blocks, cta_group::2) per SM; warp 0 loads, warp 1 multiplies, sixteen warps (eight for bf16) take the sums from tensor memory,
// which holds two tiles' so that one tile's epilogue lies behind the next one's products.
//   Scores: thread = row, so that a row's running maximum m, S = sum e^(z - m) and U = sum (z - m) e^(z - m) need no other thread; tiles leave three numbers per row
//   and group of columns instead of its logits, and join_scores_kernel puts them together: lp = z_t - m - log S, entropy = log S - U / S.
//   few_scores_kernel: up to 64 rows, W's rows the 128 of a product and X's its columns, so that none of the products is for nothing; a lane has a column of logits.
// split_kernel: few tiles.  The blocks of a cluster share K and add their whole numbers through distributed shared memory.  W's rows are the 128 of a product there and X's its
//   columns, as many as there are: products of rows that nobody wants would take power, and with it clock.
//
// Waits are bounded (q8_wait_cycles): one that runs out ends the kernel with NaN in place of what it was for, and q8_status says so.
#include <math.h>

#include <algorithm>
#include <atomic>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "tma_host.h"

namespace hb {
namespace {

constexpr int TM = 128;                    // rows of X of a block
constexpr int KB = 128;                    // bytes of K of a block of operands: one span of the swizzle
constexpr int kStaging = TM * 128;         // 128 rows of 128 bytes on their way out
constexpr int EPI_SCORES = 100;
constexpr float kLog2e = 1.4426950408889634f;

__device__ unsigned wait_ran_out;  // set by a block that gave up a wait: q8_status

// False where the barrier has not turned after so many cycles (below 0: it is not looked at).  Warps come here whole.
__device__ __forceinline__ bool wait_turn(uint64_t* bar, uint32_t parity, long long cycles) {
  bool ok = cycles >= 0 && mbar_try_wait(bar, parity);
  if (!ok && cycles > 0) {
    const long long t0 = clock64();
    while (!(ok = mbar_try_wait(bar, parity)) && clock64() - t0 < cycles) {
    }
  }
  return __all_sync(0xffffffffu, ok);
}
// True for all of the barrier's threads if it is for each
__device__ __forceinline__ bool all_of(uint32_t id, uint32_t nthreads, bool mine) {
  uint32_t r;
  asm volatile(
      "{\n"
      ".reg .pred p, q;\n"
      "setp.ne.u32 p, %3, 0;\n"
      "barrier.cta.red.and.pred q, %1, %2, p;\n"
      "selp.u32 %0, 1, 0, q;\n"
      "}\n"
      : "=r"(r)
      : "r"(id), "r"(nthreads), "r"((uint32_t)mine)
      : "memory");
  return r != 0;
}
// bytes that count as arrived (for copies that were announced and never asked for)
__device__ __forceinline__ void mbar_complete_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ void prefetch_l1(const void* p) { asm volatile("prefetch.global.L1 [%0];" ::"l"(p)); }
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// x Phi(x) = max(x, 0) - |x| erfc(|x| / sqrt 2) / 2 for two values, erfc by Abramowitz and Stegun 7.1.26 (off by 1.5e-7 at most; nothing is left of it at 16)
__device__ __forceinline__ void gelu_erf2(float& x0, float& x1) {
  auto c2 = [](float c) { return f2_pack(c, c); };
  const uint64_t ax = f2_pack(fminf(fabsf(x0), 16.f), fminf(fabsf(x1), 16.f)), z = f2_mul(ax, c2(0.70710678118654752f));
  float a0, a1, e0, e1;
  f2_unpack(f2_fma(z, c2(0.3275911f), c2(1.f)), a0, a1);
  const uint64_t t = f2_pack(rcp_fast(a0), rcp_fast(a1));
  uint64_t p = f2_fma(t, c2(-0.5f * 1.061405429f), c2(0.5f * 1.453152027f));
  p = f2_fma(p, t, c2(-0.5f * 1.421413741f));
  p = f2_fma(p, t, c2(0.5f * 0.284496736f));
  p = f2_mul(f2_fma(p, t, c2(-0.5f * 0.254829592f)), t);
  f2_unpack(f2_mul(f2_mul(z, z), c2(-kLog2e)), e0, e1);
  p = f2_mul(p, f2_pack(exp2_fast(e0), exp2_fast(e1)));
  asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(x0));
  asm("max.NaN.f32 %0, %0, 0f00000000;" : "+f"(x1));
  f2_unpack(f2_fma(ax, p, f2_pack(x0, x1)), x0, x1);
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
struct Cap {
  float cap, inv;  // cap 0: none
};
// cap tanh(x / cap) for two values: 1 - 2 / (e^2y + 1), and where that cancels (|y| < 1/4) the series, whose next term is 2^-26 of it
__device__ __forceinline__ void cap2(const Cap& c, float& x0, float& x1) {
  auto c2 = [](float c) { return f2_pack(c, c); };
  const uint64_t x = f2_pack(x0, x1), y = f2_mul(x, c2(c.inv)), u = f2_mul(y, y);
  float a0, a1, u0, u1, s0, s1;
  f2_unpack(f2_mul(y, c2(2.f * kLog2e)), a0, a1);
  f2_unpack(f2_add(f2_pack(exp2_fast(a0), exp2_fast(a1)), c2(1.f)), a0, a1);
  f2_unpack(f2_mul(f2_fma(f2_pack(rcp_fast(a0), rcp_fast(a1)), c2(-2.f), c2(1.f)), c2(c.cap)), a0, a1);
  uint64_t p = f2_fma(u, c2(62.f / 2835.f), c2(-17.f / 315.f));
  p = f2_fma(p, u, c2(2.f / 15.f));
  p = f2_mul(f2_fma(p, u, c2(-1.f / 3.f)), u);
  f2_unpack(f2_fma(p, x, x), s0, s1);
  f2_unpack(u, u0, u1);
  x0 = u0 < 0.0625f ? s0 : a0;
  x1 = u1 < 0.0625f ? s1 : a1;
}
__device__ __forceinline__ float silu(float x) { return x * rcp_fast(1.f + exp2_fast(-kLog2e * x)); }

__host__ __device__ constexpr bool has_bias(int epi) { return epi == EPI_BIAS || epi == EPI_BIAS_GELU || epi == EPI_BIAS_RESID; }
__host__ __device__ constexpr bool has_resid(int epi) { return epi == EPI_RESID || epi == EPI_BIAS_RESID; }

struct TileArgs {
  const float *xs, *ws;       // scales of rows and columns (codes)
  const bf16* bias;
  const bf16* r;
  void* out;
  int ldo, ldr;
  int M, N;
  int kbs;                    // blocks along K
  int grp, group_n;           // order of tiles
  int box_rows;               // rows of a block of X that are loaded
  const int32_t* targets;     // scores
  float *part, *at;           // [slot][3][M], [M]
  float scale;
  Cap cap;
  int carry;                  // scores: a block's tiles are of the same rows
  long long wait_cycles;
};

// Sums of bf16 products lose their last bits each time that more are added to them on the tensor cores (they are cut off, not rounded): after so many blocks they are taken out and
// added in fp32.  In one piece scores of H = 4096 are off by 3e-6 of themselves, in pieces of 512 terms by 2.2e-7 (entropies 3.6e-7), of 256 by 1.1e-7 (1.6e-7), of 128 by 7e-8.
// Up to 128 rows the weights' way from memory takes longer than either (us in pieces of 512 | 256 | 128, a 1 GB head: 1 row 167 | 167 | 171, 64 rows 175 | 178 | 193, 100 rows
// 176 | 177 | 186), above it does not (2048 rows 1422 | 1488 | 1657, 1000 rows of 30522 x 768 41.6 | 48.3 | 60.4).  Whole numbers lose nothing.
constexpr int kPiece = 8, kFewPiece = 4;  // blocks of 64 terms: above 128 rows, up to them

template <bool I8>
__device__ __forceinline__ int k_at(int kb) {  // a block's first entry
  return kb * (I8 ? KB : KB / 2);
}

template <bool I8, int BN, int CG, int EPI>
struct Cfg {
  static constexpr int EG = I8 ? 4 : 2;  // groups of four warps behind the products (two where a thread holds sums of 128 columns)
  static constexpr int THREADS = 64 + EG * 128;
  static constexpr int X_BYTES = TM * KB, W_BYTES = BN / CG * KB;
  static constexpr int STAGE = X_BYTES + W_BYTES;
  // Products: teams of groups, a staging buffer each, take chunks of 128 bytes per row in turn: two teams of two groups, or three of one where there are three chunks (192 columns)
  static constexpr int TEAMS = EPI == EPI_SCORES ? EG : BN == 192 && EPI != EPI_F32 ? 3 : 2, MEMBERS = EPI == EPI_SCORES || TEAMS == 3 ? 1 : 2;
  static constexpr int STAGING = EPI == EPI_SCORES ? 0 : TEAMS * kStaging;
  static constexpr int FIXED = STAGING + 1024 + 512;  // alignment, barriers
  static constexpr int RAW = (227 * 1024 - FIXED) / STAGE;
  static constexpr int STAGES = RAW > 10 ? 10 : RAW;
  static constexpr int SMEM = STAGES * STAGE + FIXED;
  static constexpr int COLS = 2 * BN > 256 ? 512 : 2 * BN > 128 ? 256 : 128;  // of tensor memory (allocated in powers of two)
};

__device__ __forceinline__ void tile_at(const TileArgs& a, int t, int num_m, int num_n, int& mi, int& ni) {
  const int num_a = a.group_n ? num_n : num_m, num_b = a.group_n ? num_m : num_n;  // grouped and swept dimension
  const int per = a.grp * num_b, g = t / per, r = t % per, first = g * a.grp, ga = min(a.grp, num_a - first);
  const int x = first + r % ga, y = r / ga;
  mi = a.group_n ? y : x;
  ni = a.group_n ? x : y;
}

// NC whole numbers of a row times both scales
template <int NC>
__device__ __forceinline__ void values_of(const uint32_t (&v)[NC], const TileArgs& a, float sx, int n0, float (&f)[NC]) {
  if (n0 + NC <= a.N) {
    const uint64_t s2 = f2_pack(sx, sx);
#pragma unroll
    for (int j = 0; j < NC; j += 4) {
      const float4 w = __ldg(reinterpret_cast<const float4*>(a.ws + n0 + j));
      f2_unpack(f2_mul(f2_mul(f2_pack((float)(int)v[j], (float)(int)v[j + 1]), f2_pack(w.x, w.y)), s2), f[j], f[j + 1]);
      f2_unpack(f2_mul(f2_mul(f2_pack((float)(int)v[j + 2], (float)(int)v[j + 3]), f2_pack(w.z, w.w)), s2), f[j + 2], f[j + 3]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < NC; ++j) f[j] = __fmul_rn(__fmul_rn((float)(int)v[j], n0 + j < a.N ? __ldg(a.ws + n0 + j) : 0.f), sx);  // (each rounded, as above and in split_kernel)
  }
}
// 32 bf16 values of a row (of which `left` are there) added
__device__ __forceinline__ void add_32(const bf16* p, int left, float (&f)[32]) {
  if (left >= 32) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float b[8];
      unpack_bf16x8(*(reinterpret_cast<const uint4*>(p) + j), b);
#pragma unroll
      for (int k = 0; k < 8; k += 2) f2_unpack(f2_add(f2_pack(f[8 * j + k], f[8 * j + k + 1]), f2_pack(b[k], b[k + 1])), f[8 * j + k], f[8 * j + k + 1]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < left) f[j] = __fadd_rn(f[j], __bfloat162float(p[j]));
  }
}

template <bool I8, int BN, int CG, int EPI>
__global__ void __launch_bounds__(Cfg<I8, BN, CG, EPI>::THREADS, 1)
tile_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_c,
            const __grid_constant__ TileArgs a) {
  using C = Cfg<I8, BN, CG, EPI>;
  constexpr int STAGES = C::STAGES, EG = C::EG, TILE_M = TM * CG, PIECE = BN == 128 ? kFewPiece : kPiece;
  constexpr bool kScores = EPI == EPI_SCORES, kGlu = EPI == EPI_SWIGLU, kF32 = EPI == EPI_F32;
  constexpr int OUT_BN = kGlu ? BN / 2 : BN, CHUNK = kF32 ? 32 : 64, NCHUNK = OUT_BN / CHUNK;
  static_assert(!kGlu || BN == 256, "[128 gate|128 up]");
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0u;
  const int worker = blockIdx.x / CG, workers = gridDim.x / CG;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);
  uint8_t* smem_x = smem;
  uint8_t* smem_w = smem + STAGES * C::X_BYTES;
  uint8_t* staging = smem + STAGES * C::STAGE;
  uint64_t* full = reinterpret_cast<uint64_t*>(staging + C::STAGING);  // [STAGES]
  uint64_t* empty = full + STAGES;                                     // [STAGES]
  uint64_t* sums_full = empty + STAGES;                                // [2]
  uint64_t* sums_empty = sums_full + 2;                                // [2]
  uint64_t* all_done = sums_empty + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(all_done + 1);
  int* issued_ptr = reinterpret_cast<int*>(tmem_ptr + 1);
  int* bad_ptr = issued_ptr + 1;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int num_m = (a.M + TILE_M - 1) / TILE_M, num_n = (a.N + BN - 1) / BN, tiles = num_m * num_n;

  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    if (!kScores) tma_prefetch_desc(&map_c);
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(&full[i], CG);  // (a pair's bytes all count on the first block's)
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sums_full[i], 1);
      mbar_init(&sums_empty[i], 4 * C::TEAMS * C::MEMBERS * CG);
    }
    mbar_init(all_done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      tmem_alloc_2sm(tmem_ptr, C::COLS);
      tmem_relinquish_2sm();
    } else {
      tmem_alloc(tmem_ptr, C::COLS);
      tmem_relinquish();
    }
    pdl_launch_dependents();  // (launch.h)
  }
  if constexpr (CG == 1) {
    // rows of X that are not loaded are zeros: their products take less of the power that the card's clock goes by (32 rows of a bf16 head, run for seconds: 202 -> 191 us)
    const int fill = (TM - a.box_rows) * (KB / 16);
    for (int i = threadIdx.x; i < STAGES * fill; i += C::THREADS)
      *reinterpret_cast<uint4*>(smem_x + i / fill * C::X_BYTES + a.box_rows * KB + i % fill * 16) = make_uint4(0, 0, 0, 0);
    fence_proxy_async_smem();
  }
  tc_fence_before();
  if constexpr (CG == 2) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0);
  pdl_wait();

  bool ok = true;
  if (warp == 0) {
    const bool elected = elect_one_sync();
    int s = 0, issued = 0;
    uint32_t phase = 0;
    for (int t = worker; t < tiles && ok; t += workers) {
      int mi, ni;
      tile_at(a, t, num_m, num_n, mi, ni);
      for (int kb = 0; kb < a.kbs; ++kb) {
        if (!(ok = wait_turn(&empty[s], phase ^ 1, a.wait_cycles))) break;
        if (elected) {
          if constexpr (CG == 2) {
            if (rank == 0) mbar_arrive_expect_tx(&full[s], 2 * C::STAGE);
            else mbar_arrive_cluster(&full[s], 0);
            tma_load_2d_2sm(smem_x + s * C::X_BYTES, &map_x, &full[s], k_at<I8>(kb), mi * TILE_M + (int)rank * TM);
            tma_load_2d_2sm(smem_w + s * C::W_BYTES, &map_w, &full[s], k_at<I8>(kb), ni * BN + (int)rank * (BN / 2));
          } else {
            mbar_arrive_expect_tx(&full[s], a.box_rows * KB + C::W_BYTES);
            tma_load_2d(smem_x + s * C::X_BYTES, &map_x, &full[s], k_at<I8>(kb), mi * TILE_M);
            tma_load_2d(smem_w + s * C::W_BYTES, &map_w, &full[s], k_at<I8>(kb), ni * BN);
          }
        }
        ++issued;
        if (++s == STAGES) { s = 0; phase ^= 1; }
      }
    }
    if (lane == 0) *issued_ptr = issued;
  } else if (warp == 1) {
    if (rank == 0) {
      const bool elected = elect_one_sync();
      constexpr uint32_t idesc = I8 ? umma_idesc_i8(TILE_M, BN) : umma_idesc_bf16(TILE_M, BN);
      int s = 0, it = 0;
      uint32_t phase = 0;
      for (int t = worker; t < tiles && ok; t += workers) {
        uint32_t d = 0;
        for (int kb = 0; kb < a.kbs; ++kb) {
          const bool first = I8 ? kb == 0 : kb % PIECE == 0;
          if (first) {
            if (!(ok = wait_turn(&sums_empty[it & 1], ((it >> 1) & 1) ^ 1, a.wait_cycles))) break;
            tc_fence_after();
            d = tmem + (it & 1) * BN;
          }
          if (!(ok = wait_turn(&full[s], phase, a.wait_cycles))) break;
          tc_fence_after();
          const uint32_t xa = smem_u32(smem_x + s * C::X_BYTES), wa = smem_u32(smem_w + s * C::W_BYTES);
          if (elected) {
#pragma unroll
            for (int k = 0; k < KB; k += 32) {  // a product takes 32 bytes of K
              const uint64_t dx = umma_desc_kmajor_sw128(xa + k), dw = umma_desc_kmajor_sw128(wa + k);
              const uint32_t more = !first || k != 0;
              if constexpr (I8 && CG == 2) umma_i8_ss_2sm(d, dx, dw, idesc, more);
              else if constexpr (I8) umma_i8_ss(d, dx, dw, idesc, more);
              else if constexpr (CG == 2) umma_f16_ss_2sm(d, dx, dw, idesc, more);
              else umma_f16_ss(d, dx, dw, idesc, more);
            }
            if constexpr (CG == 2) umma_commit_2sm_mc(&empty[s], 0x3); else umma_commit(&empty[s]);
          }
          if (++s == STAGES) { s = 0; phase ^= 1; }
          if (kb + 1 == a.kbs || (!I8 && kb % PIECE == PIECE - 1)) {
            if (elected) {
              if constexpr (CG == 2) umma_commit_2sm_mc(&sums_full[it & 1], 0x3); else umma_commit(&sums_full[it & 1]);
            }
            ++it;
          }
        }
      }
    }
  } else if ((warp - 2) >> 2 < C::TEAMS * C::MEMBERS) {
    const int q = warp & 3, row = q * 32 + lane;  // row of the block's 128, lane of tensor memory
    const int grp = (warp - 2) >> 2;
    // products: a team's groups share a chunk, half each; scores: each group has its columns
    constexpr int TEAMS = C::TEAMS, MEMBERS = C::MEMBERS, TEAM = 128 * MEMBERS;
    const int team = grp / MEMBERS, half0 = MEMBERS == 2 ? grp & 1 : 0, half1 = MEMBERS == 2 ? half0 + 1 : 2;  // halves of a chunk that are this group's
    const bool leader = (threadIdx.x - 64) % TEAM == 0;
    uint8_t* const buf = staging + team * kStaging;
    uint8_t* const my_row = buf + row * 128;
    float m = -INFINITY, S = 0.f, U = 0.f;  // scores
    const bool carry = a.carry != 0;        // a row's sums go on through the block's tiles
    int it = 0;
    for (int t = worker; t < tiles && ok; t += workers) {
      int mi, ni;
      tile_at(a, t, num_m, num_n, mi, ni);
      const int m0 = mi * TILE_M + (int)rank * TM, row_g = m0 + row;
      const bool live = row_g < a.M, any = m0 + q * 32 < a.M;  // this row, one of the warp's is there
      float sx = 1.f;
      if constexpr (I8) sx = live ? __ldg(a.xs + row_g) : 0.f;
      int target = -1;
      if constexpr (kScores) {
        sx *= a.scale;
        if (live && a.targets) target = __ldg(a.targets + row_g);
      }
      uint32_t t_row = 0;
      int as = 0;
      auto sums_there = [&] {
        as = it & 1;
        ok = all_of(1 + team, TEAM, wait_turn(&sums_full[as], (it >> 1) & 1, a.wait_cycles));
        tc_fence_after();
        t_row = tmem + as * BN + (static_cast<uint32_t>(q * 32) << 16);
        ++it;
        return ok;
      };
      auto release = [&] {  // this warp has read what it needs of the tile's sums
        tc_fence_before();
        __syncwarp();
        if (lane == 0) { if (CG == 2) mbar_arrive_cluster(&sums_empty[as], 0); else mbar_arrive(&sums_empty[as]); }
      };
      if constexpr (kScores) {
        constexpr int MINE = BN / EG;  // a thread's columns of its row
        float sums[I8 ? 1 : MINE];
        if constexpr (!I8) {
#pragma unroll
          for (int j = 0; j < MINE; ++j) sums[j] = 0.f;
          for (int k0 = 0; k0 < a.kbs; k0 += PIECE) {
            if (!sums_there()) break;
            if (any) {
#pragma unroll
              for (int c = 0; c < MINE; c += 32) {
                uint32_t v[32];
                tmem_ld_32x32b_x32(t_row + grp * MINE + c, v);
                tmem_ld_wait();
#pragma unroll
                for (int j = 0; j < 32; ++j) sums[c + j] += __uint_as_float(v[j]);
              }
            }
            release();
          }
        } else {
          const int n0 = ni * BN + grp * MINE + lane * 32;
          if (lane < MINE / 32 && n0 < a.N) prefetch_l1(a.ws + n0);  // (on its way while the tile's products are made)
          sums_there();
        }
        if (!ok) break;
        // 32 columns from n0 on
        auto take = [&](float(&f)[32], int n0) {
          if (n0 >= a.N) return;
          if constexpr (!I8) {
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] *= sx;
          }
          if (a.cap.cap > 0.f) {
#pragma unroll
            for (int j = 0; j < 32; j += 2) cap2(a.cap, f[j], f[j + 1]);
          }
          if ((unsigned)target - (unsigned)n0 < 32u) {
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) z = target - n0 == j ? f[j] : z;
            a.at[row_g] = z;  // (one tile has the target; whether it is below N is asked where it is read)
          }
          const int left = a.N - n0;
          if (left < 32) {
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = j < left ? f[j] : -INFINITY;
          }
          float top = f[0];
#pragma unroll
          for (int j = 1; j < 31; j += 2) top = max3(top, f[j], f[j + 1]);
          top = fmaxf(top, f[31]);
          if (top > m) {
            if (m > -INFINITY) {
              const float d = m - top, w = exp2_fast(d * kLog2e);
              U = w > 0.f ? w * fmaf(d, S, U) : 0.f;
              S *= w;
            }
            m = top;
          }
          float base = m > -INFINITY ? m : 0.f;
          if (left < 32) {  // (the distance itself, as a large m less 1e4 is m again)
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = j < left ? f[j] - base : -1e4f;
            base = 0.f;
          }
          // A logit of -inf has a weight of 0, and 0 times its distance is to be 0: no distance is below -1e4 there.  Codes, which hardly ever have one, look for the NaN instead and take
          // these 32 again (us of each clamped | looked for: 700 x 151936 x 1536 of codes 127.9 | 125.0, with a cap 154.4 | 153.6; 200 x 30522 x 768 in bf16 19.4 | 19.9)
          const uint64_t off = f2_pack(-base, -base), log2e = f2_pack(kLog2e, kLog2e);
          uint64_t s2 = f2_pack(0.f, 0.f), u2 = s2;  // two at a time
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            const uint64_t d = f2_add(f2_pack(f[j], f[j + 1]), off);
            float x0, x1;
            f2_unpack(f2_mul(d, log2e), x0, x1);
            const uint64_t w = f2_pack(exp2_fast(x0), exp2_fast(x1));
            s2 = f2_add(s2, w);
            if constexpr (I8) {
              u2 = f2_fma(w, d, u2);
            } else {
              float d0, d1;
              f2_unpack(d, d0, d1);
              u2 = f2_fma(w, f2_pack(fmaxf(d0, -1e4f), fmaxf(d1, -1e4f)), u2);
            }
          }
          float lo, hi;
          f2_unpack(s2, lo, hi);
          S += lo + hi;
          f2_unpack(u2, lo, hi);
          lo += hi;
          if (I8 && __builtin_expect(lo != lo, 0)) {
            lo = 0.f;
#pragma unroll
            for (int j = 0; j < 32; ++j) lo = fmaf(exp2_fast((f[j] - base) * kLog2e), fmaxf(f[j] - base, -1e4f), lo);
          }
          U += lo;
        };
        const int n_first = ni * BN + grp * MINE;
        if (!any) {
          if constexpr (I8) release();
        } else if constexpr (I8) {
#pragma unroll 1
          for (int c = 0; c < MINE; c += 32) {
            uint32_t v[32];
            float f[32];
            tmem_ld_32x32b_x32(t_row + grp * MINE + c, v);
            tmem_ld_wait();
            if (c + 32 == MINE) release();
            values_of(v, a, sx, n_first + c, f);
            take(f, n_first + c);
          }
        } else {
#pragma unroll
          for (int c = 0; c < MINE; c += 32) {
            float f[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) f[j] = sums[c + j];
            take(f, n_first + c);
          }
        }
        if (!carry || t + workers >= tiles) {
          if (live) {
            float* p = a.part + (size_t)((carry ? worker / num_m : ni) * EG + grp) * 3 * a.M + row_g;
            p[0] = m;
            p[a.M] = S;
            p[2 * (size_t)a.M] = U;
          }
          m = -INFINITY;
          S = U = 0.f;
        }
      } else {
        const int n_out0 = ni * OUT_BN, n_out = kGlu ? a.N / 2 : a.N;
        // what the columns are multiplied by and what is added is on its way while the tile's products are made
        for (int c = team; c < NCHUNK; c += TEAMS) {
          const int col = c * CHUNK + half0 * (CHUNK / 2), n0 = ni * BN + col;
          if (lane == 0 && n0 < a.N) prefetch_l1(a.ws + n0);
          if (kGlu && lane == 1) prefetch_l1(a.ws + n0 + 128);
          if (has_bias(EPI) && lane == 2 && n0 < a.N) prefetch_l1(a.bias + n0);
          if (has_resid(EPI) && live && n0 < n_out) prefetch_l2_line(a.r + (size_t)row_g * a.ldr + n0);
        }
        if (!sums_there()) break;
#pragma unroll 1
        for (int c = team; c < NCHUNK; c += TEAMS) {
          const bool last = c + TEAMS >= NCHUNK;
          if (leader) tma_store_wait_read<0>();  // the team's store before has read `buf`
          if constexpr (kF32) {
            const int col = c * 32 + half0 * 16;
            uint32_t v[16];
            float f[16];
            tmem_ld_32x32b_x16(t_row + col, v);
            tmem_ld_wait();
            if (last) release();
            values_of(v, a, sx, n_out0 + col, f);
            bar_sync(1 + team, TEAM);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              *reinterpret_cast<float4*>(my_row + (((half0 * 4 + j) ^ (row & 7)) << 4)) = make_float4(f[4 * j], f[4 * j + 1], f[4 * j + 2], f[4 * j + 3]);
          } else {
#pragma unroll 1
            for (int half = half0; half < half1; ++half) {
              const int col = c * 64 + half * 32, n0 = n_out0 + col;
              float f[32];
              if constexpr (kGlu) {
#pragma unroll
                for (int h = 0; h < 32; h += 16) {
                  uint32_t v[16], u[16];
                  float g[16], x[16];
                  tmem_ld_32x32b_x16(t_row + col + h, v);
                  tmem_ld_32x32b_x16(t_row + 128 + col + h, u);
                  tmem_ld_wait();
                  if (h == 16 && last && half + 1 == half1) release();
                  values_of(v, a, sx, ni * BN + col + h, g);
                  values_of(u, a, sx, ni * BN + 128 + col + h, x);
#pragma unroll
                  for (int j = 0; j < 16; ++j) f[h + j] = silu(g[j]) * x[j];
                }
              } else {
                uint32_t v[32];
                tmem_ld_32x32b_x32(t_row + col, v);
                tmem_ld_wait();
                if (last && half + 1 == half1) release();
                values_of(v, a, sx, n0, f);
              }
              if constexpr (has_bias(EPI)) add_32(a.bias + n0, n_out - n0, f);
              if constexpr (EPI == EPI_BIAS_GELU) {
#pragma unroll
                for (int j = 0; j < 32; j += 2) gelu_erf2(f[j], f[j + 1]);
              }
              if constexpr (has_resid(EPI)) {
                if (live) add_32(a.r + (size_t)row_g * a.ldr + n0, n_out - n0, f);
              }
              if (half == half0) bar_sync(1 + team, TEAM);
#pragma unroll
              for (int j = 0; j < 4; ++j) {
                uint4 o;
                o.x = pack_bf16x2(f[8 * j], f[8 * j + 1]);
                o.y = pack_bf16x2(f[8 * j + 2], f[8 * j + 3]);
                o.z = pack_bf16x2(f[8 * j + 4], f[8 * j + 5]);
                o.w = pack_bf16x2(f[8 * j + 6], f[8 * j + 7]);
                *reinterpret_cast<uint4*>(my_row + (((half * 4 + j) ^ (row & 7)) << 4)) = o;
              }
            }
          }
          const int n0 = n_out0 + c * CHUNK;
          if (n0 + CHUNK > n_out && n_out % (kF32 ? 4 : 8) != 0) {  // (a copy ends on 16 bytes: it would write zeros behind the last column)
            if (live) {
              for (int j = half0 * (CHUNK / 2); j < half1 * (CHUNK / 2) && n0 + j < n_out; ++j) {
                const int at = ((j / (kF32 ? 4 : 8)) ^ (row & 7)) << 4, in = j % (kF32 ? 4 : 8);
                if constexpr (kF32) static_cast<float*>(a.out)[(size_t)row_g * a.ldo + n0 + j] = reinterpret_cast<const float*>(my_row + at)[in];
                else static_cast<bf16*>(a.out)[(size_t)row_g * a.ldo + n0 + j] = reinterpret_cast<const bf16*>(my_row + at)[in];
              }
            }
            continue;
          }
          fence_proxy_async_smem();
          bar_sync(1 + team, TEAM);
          if (leader) {
            tma_store_2d(&map_c, buf, n0, m0);
            tma_store_commit();
          }
        }
      }
    }
    if (!kScores && leader) tma_store_wait_all<0>();
    __syncwarp();
  }

  tc_fence_before();
  bool bad = __syncthreads_or(!ok);
  if constexpr (CG == 2) {
    if (threadIdx.x == 0) *bad_ptr = bad;
    __syncthreads();
    cluster_sync_all();
    bad |= *cluster_ptr<2>(bad_ptr, rank ^ 1) != 0;
  }
  if (bad) {
    // what is in flight ends before its room is given back
    if (warp == 0) {
      const int mine = *issued_ptr, other = CG == 2 ? *cluster_ptr<2>(issued_ptr, rank ^ 1) : mine;
      if (rank == 0) {
        if (lane == 0) {
          if constexpr (CG == 2) {
            for (int i = min(mine, other); i < max(mine, other); ++i) {  // blocks that one of the pair asked for and the other did not: the other's part is made up for
              if (other > mine) {
                mbar_arrive_expect_tx(&full[i % STAGES], C::STAGE);
              } else {
                mbar_complete_tx(&full[i % STAGES], C::STAGE);
                mbar_arrive(&full[i % STAGES]);
              }
            }
          }
        }
        __syncwarp();
        for (int i = max(0, max(mine, other) - STAGES); i < max(mine, other); ++i) wait_turn(&full[i % STAGES], (i / STAGES) & 1, HB_WAIT_TIMEOUT_CYCLES);
      }
    }
    if (warp == 1) {
      if (rank == 0 && elect_one_sync()) {
        if constexpr (CG == 2) umma_commit_2sm_mc(all_done, 0x3); else umma_commit(all_done);
      }
      __syncwarp();
      wait_turn(all_done, 0, HB_WAIT_TIMEOUT_CYCLES);
    }
    const float nan = __uint_as_float(0x7fffffffu);
    for (int t = worker; t < tiles; t += workers) {
      int mi, ni;
      tile_at(a, t, num_m, num_n, mi, ni);
      const int m0 = mi * TILE_M + (int)rank * TM;
      if constexpr (kScores) {
        for (int i = threadIdx.x; i < TM * EG; i += C::THREADS) {
          const int r = m0 + i % TM;
          if (r < a.M) a.part[(size_t)((a.carry ? worker / num_m : ni) * EG + i / TM) * 3 * a.M + (size_t)a.M + r] = nan;
        }
      } else {
        const int n_out = kGlu ? a.N / 2 : a.N;
        for (int i = threadIdx.x; i < TM * OUT_BN; i += C::THREADS) {
          const int r = m0 + i / OUT_BN, n = ni * OUT_BN + i % OUT_BN;
          if (r < a.M && n < n_out) {
            if constexpr (kF32) static_cast<float*>(a.out)[(size_t)r * a.ldo + n] = nan;
            else static_cast<bf16*>(a.out)[(size_t)r * a.ldo + n] = __float2bfloat16(nan);
          }
        }
      }
    }
    if (threadIdx.x == 0) wait_ran_out = 1;
    __syncthreads();
  }
  if constexpr (CG == 2) cluster_sync_all();
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 2) tmem_dealloc_2sm(tmem, C::COLS); else tmem_dealloc(tmem, C::COLS);
  }
}

// ------------------------------------------------------------------ a row's sums of all tiles
// kJoinRows rows per block, their threads side by side
template <int kJoinThreads, int kJoinRows>
__global__ void __launch_bounds__(kJoinThreads) join_scores_kernel(const float* __restrict__ part, const float* __restrict__ at, const int32_t* __restrict__ targets,
                                                                  float* __restrict__ lp, float* __restrict__ entropy, int slots, int T, int V) {
  __shared__ float sm[3][kJoinThreads];
  pdl_wait();
  pdl_launch_dependents();
  const int r = threadIdx.x % kJoinRows, g = threadIdx.x / kJoinRows;  // neighbouring threads read neighbouring rows
  const int row = blockIdx.x * kJoinRows + r;
  float m = -INFINITY, s = 0.f, u = 0.f;
  auto add = [&](float m2, float s2, float u2) {
    const float top = fmaxf(m, m2);
    auto weight = [&](float x, float& d) {
      d = x == top ? 0.f : fmaxf(x - top, -200.f);
      return d > -200.f ? exp2_fast(d * kLog2e) : 0.f;
    };
    float d1, d2;
    const float w1 = weight(m, d1), w2 = weight(m2, d2);
    u = (w1 > 0.f ? w1 * fmaf(d1, s, u) : 0.f) + (w2 > 0.f ? w2 * fmaf(d2, s2, u2) : 0.f);
    s = fmaf(w1, s, w2 * s2);  // (a NaN times 0 stays one)
    m = top;
  };
  if (row < T) {
    constexpr int kAhead = 5;
    for (int i = g; i < slots; i += kAhead * (kJoinThreads / kJoinRows)) {
      float v[kAhead][3];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int slot = i + k * (kJoinThreads / kJoinRows);
#pragma unroll
        for (int c = 0; c < 3; ++c) v[k][c] = slot < slots ? part[((size_t)slot * 3 + c) * T + row] : (c == 0 ? -INFINITY : 0.f);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) add(v[k][0], v[k][1], v[k][2]);
    }
  }
  sm[0][threadIdx.x] = m;
  sm[1][threadIdx.x] = s;
  sm[2][threadIdx.x] = u;
  for (int o = kJoinThreads / 2; o >= kJoinRows; o >>= 1) {
    __syncthreads();
    if ((int)threadIdx.x < o) {
      add(sm[0][threadIdx.x + o], sm[1][threadIdx.x + o], sm[2][threadIdx.x + o]);
      sm[0][threadIdx.x] = m;
      sm[1][threadIdx.x] = s;
      sm[2][threadIdx.x] = u;
    }
  }
  if ((int)threadIdx.x < kJoinRows && row < T) {
    const bool none = s == 0.f;  // nothing but -inf
    const float log_s = logf(s);
    const int t = targets ? targets[row] : -1;
    if (lp) lp[row] = t >= 0 && t < V && !none ? at[row] - m - log_s : -INFINITY;
    if (entropy) entropy[row] = none ? 0.f : log_s - u / s;
  }
}

// ------------------------------------------------------------------ few tiles: K shared by a cluster
constexpr int SN = 128;                  // rows of W of a tile (a gated unit's: 64 of the gate, 64 beside them)
constexpr int kDump = SN + 4;            // whole numbers of a row on their way through shared memory
constexpr int kSplitThreads = 320;       // warp 0 loads, warp 1 multiplies, eight take the sums out

struct SplitArgs {
  const float *xs, *ws;
  const bf16 *bias, *r;
  void* out;
  int ldo, ldr, M, N, kbs, epi;
  int box_rows, columns, stages;  // rows of X that are loaded (a multiple of 16), columns of tensor memory for them
  long long wait_cycles;
};

__global__ void __launch_bounds__(kSplitThreads) split_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w,
                                                              const __grid_constant__ SplitArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[12], empty[12], sums_full, all_done;
  __shared__ uint32_t tmem_at;
  __shared__ int bad_flag;
  __shared__ float s_xs[TM], s_ws[SN], s_bias[SN];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);
  const int x_bytes = a.box_rows * KB, stages = a.stages;
  uint8_t* smem_w = smem + stages * x_bytes;
  int* dump = reinterpret_cast<int*>(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int parts = gridDim.x, part = blockIdx.x;
  const int kb0 = (int)((long long)a.kbs * part / parts), kb1 = (int)((long long)a.kbs * (part + 1) / parts);
  const bool glu = a.epi == EPI_SWIGLU;
  const int m0 = blockIdx.z * TM;
  const int w0 = glu ? blockIdx.y / 2 * 256 + blockIdx.y % 2 * 64 : blockIdx.y * SN, w1 = w0 + (glu ? 128 : 64);  // rows of W: 64 from each
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    mbar_init(&sums_full, 1);
    mbar_init(&all_done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_at, a.columns);
    tmem_relinquish();
    pdl_launch_dependents();  // (launch.h)
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_at, 0);
  // W is on its way into L2 (nothing of it is read) while the kernel before ends: 13 x 4096 x 14336 15.1 -> 13.9 us back to back, 32 x 28672 x 4096 gated 23.2 -> 21.3; with more rows
  // of X these come late behind the others (128 x 4096 x 4096 10.7 -> 10.9)
  if (a.box_rows <= 64 && warp == 0 && elect_one_sync()) {
    for (int kb = kb0; kb < min(kb1, kb0 + stages); ++kb) {
      tma_prefetch_l2_2d(&map_w, kb * KB, w0);
      tma_prefetch_l2_2d(&map_w, kb * KB, w1);
    }
  }
  __syncwarp();
  pdl_wait();

  bool ok = true;
  int issued = 0;
  if (warp == 0) {
    const bool elected = elect_one_sync();
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!(ok = wait_turn(&empty[s], phase ^ 1, a.wait_cycles))) break;
      if (elected) {
        mbar_arrive_expect_tx(&full[s], x_bytes + SN * KB);
        tma_load_2d(smem_w + s * SN * KB, &map_w, &full[s], kb * KB, w0, kEvictFirst);
        tma_load_2d(smem_w + s * SN * KB + 64 * KB, &map_w, &full[s], kb * KB, w1, kEvictFirst);
        tma_load_2d(smem + s * x_bytes, &map_x, &full[s], kb * KB, m0, kEvictLast);
      }
      ++issued;
      if (++s == stages) { s = 0; phase ^= 1; }
    }
  } else if (warp == 1) {
    const bool elected = elect_one_sync();
    const uint32_t idesc = umma_idesc_i8(SN, a.box_rows);
    int s = 0;
    uint32_t phase = 0;
    for (int kb = kb0; kb < kb1; ++kb) {
      if (!(ok = wait_turn(&full[s], phase, a.wait_cycles))) break;
      tc_fence_after();
      const uint32_t xa = smem_u32(smem + s * x_bytes), wa = smem_u32(smem_w + s * SN * KB);
      if (elected) {
#pragma unroll
        for (int k = 0; k < KB; k += 32) umma_i8_ss(tmem, umma_desc_kmajor_sw128(wa + k), umma_desc_kmajor_sw128(xa + k), idesc, kb > kb0 || k != 0);
        umma_commit(&empty[s]);
      }
      if (++s == stages) { s = 0; phase ^= 1; }
    }
    if (ok && elected) umma_commit(&sums_full);
    __syncwarp();
  } else {
    // scales and bias come while the products are made
    for (int i = threadIdx.x - 64; i < 3 * 128; i += kSplitThreads - 64) {
      const int j = i & 127, n = j < 64 ? w0 + j : w1 + j - 64;
      if (i < 128) s_ws[j] = n < a.N ? __ldg(a.ws + n) : 0.f;
      else if (i < 256) s_xs[j] = m0 + j < a.M ? __ldg(a.xs + m0 + j) : 0.f;
      else s_bias[j] = a.bias && n < a.N ? __bfloat162float(a.bias[n]) : 0.f;
    }
    ok = wait_turn(&sums_full, 0, a.wait_cycles);
    const int q = warp & 3;
    if (ok) {  // (all operands have been read: their room takes the sums, a row of X after the other)
      tc_fence_after();
      for (int c = warp < 6 ? 0 : 16; c < a.box_rows; c += 32) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(q * 32) << 16) + c, v);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < 16; ++j) dump[(c + j) * kDump + q * 32 + lane] = (int)v[j];
      }
    }
  }
  tc_fence_before();
  bool bad = __syncthreads_or(!ok);
  if (bad) {
    if (warp == 0)
      for (int i = max(0, issued - stages); i < issued; ++i) wait_turn(&full[i % stages], (i / stages) & 1, HB_WAIT_TIMEOUT_CYCLES);
    if (warp == 1) {
      if (elect_one_sync()) umma_commit(&all_done);
      __syncwarp();
      wait_turn(&all_done, 0, HB_WAIT_TIMEOUT_CYCLES);
    }
    if (threadIdx.x == 0) wait_ran_out = 1;
  }
  if (parts > 1) {
    if (threadIdx.x == 0) bad_flag = bad;
    __syncthreads();
    cluster_sync_all();
    bad = __syncthreads_or((int)threadIdx.x < parts && *cluster_ptr<2>(&bad_flag, threadIdx.x) != 0);
  }
  const int rows = min(a.M - m0, TM), quads = glu ? SN / 8 : SN / 4, n_out = glu ? a.N / 2 : a.N;
  for (int i = part * kSplitThreads + threadIdx.x; i < rows * quads; i += parts * kSplitThreads) {
    const int r = i / quads, c = i % quads * 4, m = m0 + r, n = blockIdx.y * (quads * 4) + c;
    if (n >= n_out) continue;
    float resid[4] = {};
    if (a.r) {
      const bf16* at = a.r + (size_t)m * a.ldr + n;
      if (n + 4 <= n_out) {
        const uint2 u = *reinterpret_cast<const uint2*>(at);
        const float2 lo = unpack_bf16x2(u.x), hi = unpack_bf16x2(u.y);
        resid[0] = lo.x; resid[1] = lo.y; resid[2] = hi.x; resid[3] = hi.y;
      } else {
        for (int e = 0; n + e < n_out; ++e) resid[e] = __bfloat162float(at[e]);
      }
    }
    auto sum_at = [&](int col, int(&sum)[4]) {  // all parts' numbers at once, added in any order
      int4 v[8];
#pragma unroll
      for (int p = 0; p < 8; ++p)
        if (p < parts) v[p] = *reinterpret_cast<const int4*>((parts == 1 ? dump : cluster_ptr<2>(dump, p)) + r * kDump + col);
      sum[0] = v[0].x; sum[1] = v[0].y; sum[2] = v[0].z; sum[3] = v[0].w;
#pragma unroll
      for (int p = 1; p < 8; ++p)
        if (p < parts) {
          sum[0] += v[p].x; sum[1] += v[p].y; sum[2] += v[p].z; sum[3] += v[p].w;
        }
    };
    const float sx = s_xs[r];
    int acc[4];
    float f[4];
    sum_at(c, acc);
    if (glu) {
      int up[4];
      sum_at(64 + c, up);
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(silu(__fmul_rn(__fmul_rn((float)acc[e], s_ws[c + e]), sx)), __fmul_rn(__fmul_rn((float)up[e], s_ws[64 + c + e]), sx));
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = __fmul_rn(__fmul_rn((float)acc[e], s_ws[c + e]), sx);  // (roundings as in tile_kernel, nothing added where that adds nothing: zeros keep their signs)
      if (a.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __fadd_rn(f[e], s_bias[c + e]);
      }
      if (a.epi == EPI_BIAS_GELU) {
        gelu_erf2(f[0], f[1]);
        gelu_erf2(f[2], f[3]);
      }
      if (a.r) {
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = __fadd_rn(f[e], resid[e]);
      }
    }
    if (bad) f[0] = f[1] = f[2] = f[3] = __uint_as_float(0x7fffffffu);
    if (a.epi == EPI_F32) {
      float* o = static_cast<float*>(a.out) + (size_t)m * a.ldo + n;
      if (n + 4 <= n_out) *reinterpret_cast<float4*>(o) = make_float4(f[0], f[1], f[2], f[3]);
      else
        for (int e = 0; n + e < n_out; ++e) o[e] = f[e];
    } else {
      bf16* o = static_cast<bf16*>(a.out) + (size_t)m * a.ldo + n;
      if (n + 4 <= n_out) *reinterpret_cast<uint2*>(o) = make_uint2(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]));
      else
        for (int e = 0; n + e < n_out; ++e) o[e] = __float2bfloat16(f[e]);
    }
  }
  if (parts > 1) {
    __syncwarp();
    cluster_sync_all();  // others may still read this block's sums
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, a.columns);
  }
}

// ------------------------------------------------------------------ scores of few rows
// Shared memory: us of 1 | 16 | 32 | 64 rows of a 1 GB head with 130 KB 167 | 169 | 173 | 180, 165 KB 163 | 164 | 167 | 176, 184 KB 164 | 166 | 166 | 173, 200 KB 166 | 168 | 165 | 171 (32 | 16 rows
// with 100 KB 181 | 176, 225 KB 173 | 174)
constexpr int kFewRows = 64, kFewThreads = 64 + 4 * 128, kFewSmem = 184 * 1024;

struct FewArgs {
  const float *xs, *ws;
  int T, V, kbs;
  int box_rows, columns, stages;  // as in SplitArgs; the columns hold two tiles' sums
  const int32_t* targets;
  float *part, *at;
  float scale;
  Cap cap;
  long long wait_cycles;
};

template <bool I8>
__global__ void __launch_bounds__(kFewThreads, 1) few_scores_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w, const __grid_constant__ FewArgs a) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[12], empty[12], sums_full[2], sums_empty[2], all_done;
  __shared__ uint32_t tmem_at;
  __shared__ __align__(16) float s_xs[kFewRows];
  __shared__ __align__(16) int s_targets[kFewRows];
  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);
  const int x_bytes = a.box_rows * KB, stages = a.stages;
  uint8_t* smem_w = smem + stages * x_bytes;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (a.V + SN - 1) / SN, groups = a.box_rows / 16;  // sixteen rows of X for each group of four warps
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w);
    for (int i = 0; i < stages; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&sums_full[i], 1);
      mbar_init(&sums_empty[i], 4 * groups);
    }
    mbar_init(&all_done, 1);
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(&tmem_at, a.columns);
    tmem_relinquish();
    pdl_launch_dependents();  // (launch.h)
  }
  if (warp == 2 && elect_one_sync())  // W is on its way into L2 (nothing of it is read) while the kernel before ends
    for (int kb = 0; kb < min(a.kbs, stages); ++kb) tma_prefetch_l2_2d(&map_w, k_at<I8>(kb), blockIdx.x * SN);
  __syncwarp();
  pdl_wait();
  if (threadIdx.x < kFewRows) {
    const int t = threadIdx.x;
    s_xs[t] = t < a.T ? (I8 ? __ldg(a.xs + t) : 1.f) * a.scale : 0.f;
    s_targets[t] = t < a.T && a.targets ? __ldg(a.targets + t) : -1;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_at, 0);

  bool ok = true;
  int issued = 0;
  if (warp == 0) {
    const bool elected = elect_one_sync();
    int s = 0;
    uint32_t phase = 0;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x)
      for (int kb = 0; kb < a.kbs; ++kb) {
        if (!(ok = wait_turn(&empty[s], phase ^ 1, a.wait_cycles))) break;
        if (elected) {
          mbar_arrive_expect_tx(&full[s], x_bytes + SN * KB);
          tma_load_2d(smem_w + s * SN * KB, &map_w, &full[s], k_at<I8>(kb), t * SN);
          tma_load_2d(smem + s * x_bytes, &map_x, &full[s], k_at<I8>(kb), 0);
        }
        ++issued;
        if (++s == stages) { s = 0; phase ^= 1; }
      }
  } else if (warp == 1) {
    const bool elected = elect_one_sync();
    const uint32_t idesc = I8 ? umma_idesc_i8(SN, a.box_rows) : umma_idesc_bf16(SN, a.box_rows);
    int s = 0, it = 0;
    uint32_t phase = 0, d = 0;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x)
      for (int kb = 0; kb < a.kbs; ++kb) {
        const bool first = I8 ? kb == 0 : kb % kFewPiece == 0;
        if (first) {
          if (!(ok = wait_turn(&sums_empty[it & 1], ((it >> 1) & 1) ^ 1, a.wait_cycles))) break;
          tc_fence_after();
          d = tmem + (it & 1) * a.box_rows;
        }
        if (!(ok = wait_turn(&full[s], phase, a.wait_cycles))) break;
        tc_fence_after();
        const uint32_t xa = smem_u32(smem + s * x_bytes), wa = smem_u32(smem_w + s * SN * KB);
        if (elected) {
#pragma unroll
          for (int k = 0; k < KB; k += 32) {
            const uint64_t dw = umma_desc_kmajor_sw128(wa + k), dx = umma_desc_kmajor_sw128(xa + k);
            if constexpr (I8) umma_i8_ss(d, dw, dx, idesc, !first || k != 0);
            else umma_f16_ss(d, dw, dx, idesc, !first || k != 0);
          }
          umma_commit(&empty[s]);
        }
        if (++s == stages) { s = 0; phase ^= 1; }
        if (kb + 1 == a.kbs || (!I8 && kb % kFewPiece == kFewPiece - 1)) {
          if (elected) umma_commit(&sums_full[it & 1]);
          ++it;
        }
      }
    __syncwarp();
  } else if ((warp - 2) >> 2 < groups) {
    // a lane has a column of logits, its sixteen rows' sums go on through the block's tiles
    const int q = warp & 3, r0 = ((warp - 2) >> 2) * 16;
    float m[16], S[16], U[16];
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      m[j] = -INFINITY;
      S[j] = U[j] = 0.f;
    }
    int it = 0;
    for (int t = blockIdx.x; t < tiles && ok; t += gridDim.x) {
      const int n = t * SN + q * 32 + lane;
      float z[16];
      auto take = [&] {  // the next sums of this warp's lanes
        ok = wait_turn(&sums_full[it & 1], (it >> 1) & 1, a.wait_cycles);
        if (!ok) return;
        tc_fence_after();
        uint32_t v[16];
        tmem_ld_32x32b_x16(tmem + (static_cast<uint32_t>(q * 32) << 16) + (it & 1) * a.box_rows + r0, v);
        tmem_ld_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sums_empty[it & 1]);
        ++it;
        const float w = I8 && n < a.V ? __ldg(a.ws + n) : 0.f;
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if constexpr (I8) z[j] = __fmul_rn((float)(int)v[j], w);
          else z[j] += __uint_as_float(v[j]);
        }
      };
      if constexpr (I8) {
        take();
      } else {
#pragma unroll
        for (int j = 0; j < 16; ++j) z[j] = 0.f;
        for (int k0 = 0; k0 < a.kbs && ok; k0 += kFewPiece) take();
      }
      __syncwarp();
      if (ok && n < a.V) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          const float4 x = *reinterpret_cast<const float4*>(s_xs + r0 + j);
          z[j] = __fmul_rn(z[j], x.x);
          z[j + 1] = __fmul_rn(z[j + 1], x.y);
          z[j + 2] = __fmul_rn(z[j + 2], x.z);
          z[j + 3] = __fmul_rn(z[j + 3], x.w);
        }
        if (a.cap.cap > 0.f) {
#pragma unroll
          for (int j = 0; j < 16; j += 2) cap2(a.cap, z[j], z[j + 1]);
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          if (s_targets[r0 + j] == n) a.at[r0 + j] = z[j];
          if (z[j] - m[j] > 8.f) {  // (m need not be the maximum: it follows when it is left far behind)
            if (m[j] > -INFINITY) {
              const float d = m[j] - z[j], w = exp2_fast(d * kLog2e);
              U[j] = w > 0.f ? w * fmaf(d, S[j], U[j]) : 0.f;
              S[j] *= w;
            }
            m[j] = z[j];
          }
          const float d = z[j] - (m[j] > -INFINITY ? m[j] : 0.f), w = exp2_fast(d * kLog2e);
          S[j] += w;
          U[j] = fmaf(w, fmaxf(d, -1e4f), U[j]);  // (a logit of -inf: 0 times what is no infinity)
        }
      }
      __syncwarp();
    }
    // the lanes' sums: each row's brought to one m, then half of the rows to each half of the lanes, and so on
    const int j0 = lane >> 1;  // the row that this lane ends up with
    float mine = -INFINITY;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const uint32_t u = __float_as_uint(m[j]);
      const uint32_t key = __reduce_max_sync(0xffffffffu, u & 0x80000000u ? ~u : u | 0x80000000u);
      const float top = __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key);
      const float d = m[j] == top ? 0.f : m[j] - top, w = exp2_fast(d * kLog2e);  // (no infinity less itself)
      U[j] = w > 0.f ? w * fmaf(d, S[j], U[j]) : 0.f;
      S[j] *= w;
      mine = j == j0 ? top : mine;
    }
#pragma unroll
    for (int half = 8; half > 0; half >>= 1) {
      const bool upper = lane & 2 * half;
#pragma unroll
      for (int j = 0; j < half; ++j) {
        const float s = upper ? S[j] : S[j + half], u = upper ? U[j] : U[j + half];
        S[j] = (upper ? S[j + half] : S[j]) + __shfl_xor_sync(0xffffffffu, s, 2 * half);
        U[j] = (upper ? U[j + half] : U[j]) + __shfl_xor_sync(0xffffffffu, u, 2 * half);
      }
    }
    S[0] += __shfl_xor_sync(0xffffffffu, S[0], 1);
    U[0] += __shfl_xor_sync(0xffffffffu, U[0], 1);
    if (!(lane & 1) && r0 + j0 < a.T) {
      float* p = a.part + (size_t)(blockIdx.x * 4 + q) * 3 * a.T + r0 + j0;
      p[0] = mine;
      p[a.T] = S[0];
      p[2 * a.T] = U[0];
    }
    __syncwarp();
  }
  tc_fence_before();
  if (__syncthreads_or(!ok)) {
    if (warp == 0)
      for (int i = max(0, issued - stages); i < issued; ++i) wait_turn(&full[i % stages], (i / stages) & 1, HB_WAIT_TIMEOUT_CYCLES);
    if (warp == 1) {
      if (elect_one_sync()) umma_commit(&all_done);
      __syncwarp();
      wait_turn(&all_done, 0, HB_WAIT_TIMEOUT_CYCLES);
    }
    for (int i = threadIdx.x; i < 4 * a.T; i += kFewThreads) a.part[(size_t)(blockIdx.x * 4 + i / a.T) * 3 * a.T + a.T + i % a.T] = __uint_as_float(0x7fffffffu);
    if (threadIdx.x == 0) wait_ran_out = 1;
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, a.columns);
  }
}

// ------------------------------------------------------------------ host
std::atomic<long long> wait_limit{HB_WAIT_TIMEOUT_CYCLES};

int device_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return effective_sms(sms);
}
// More than 48 KB of shared memory wants to be asked for once per device
template <typename F>
cudaError_t ask_smem(F kernel, int bytes, std::atomic<uint64_t>& asked) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(asked.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  }
  return e;
}
struct Launch {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[2];
  Launch(dim3 grid, int threads, int smem, cudaStream_t stream, int cluster) {
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    int n = 0;
    if (pdl_enabled()) {
      attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[n++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (cluster > 1) {
      attr[n].id = cudaLaunchAttributeClusterDimension;
      attr[n].val.clusterDim.x = cluster;
      attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
      ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
  }
};

struct Operand {
  const void* p;
  int ld, rows;
};
template <bool I8>
bool operand_map(CUtensorMap* map, const Operand& o, int K, int box_rows) {
  return make_tmap_2d(map, o.p, I8 ? TM_U8 : TM_BF16, (uint64_t)K, (uint64_t)o.rows, (uint64_t)o.ld * (I8 ? 1 : 2), I8 ? KB : KB / 2, box_rows);
}

template <bool I8, int BN, int CG, int EPI>
cudaError_t launch_tiles(cudaStream_t stream, TileArgs a, const Operand& x, const Operand& w, int K, int sms, int* slots = nullptr) {
  using C = Cfg<I8, BN, CG, EPI>;
  static std::atomic<uint64_t> asked{0};
  cudaError_t e = ask_smem(tile_kernel<I8, BN, CG, EPI>, C::SMEM, asked);
  if (e != cudaSuccess) return e;
  constexpr int TILE_M = TM * CG;
  const int n_out = EPI == EPI_SWIGLU ? a.N / 2 : a.N;
  a.box_rows = CG == 2 ? TM : std::min(TM, (a.M + 7) / 8 * 8);
  CUtensorMap mx, mw, mc;
  if (!operand_map<I8>(&mx, x, K, a.box_rows) || !operand_map<I8>(&mw, w, K, BN / CG)) return cudaErrorInvalidValue;
  mc = mx;
  if (EPI != EPI_SCORES &&
      !make_tmap_2d(&mc, a.out, EPI == EPI_F32 ? TM_F32 : TM_BF16, (uint64_t)n_out, (uint64_t)a.M, (uint64_t)a.ldo * (EPI == EPI_F32 ? 4 : 2), EPI == EPI_F32 ? 32 : 64, TM))
    return cudaErrorInvalidValue;
  const int bytes_k = I8 ? K : 2 * K;
  a.kbs = (bytes_k + KB - 1) / KB;
  const int num_m = (a.M + TILE_M - 1) / TILE_M, num_n = (a.N + BN - 1) / BN;
  if ((long long)num_m * num_n > INT32_MAX / 2) return cudaErrorInvalidValue;
  // Order of tiles: some 32 MB of one operand stay in L2 while the other passes by
  const double x_tile = (double)TILE_M * bytes_k, w_tile = (double)BN * bytes_k, X = x_tile * num_m, W = w_tile * num_n;
  const int gm = (int)std::max(1.0, std::min((double)num_m, floor(32e6 / x_tile))), gn = (int)std::max(1.0, std::min((double)num_n, floor(32e6 / w_tile)));
  a.group_n = W + X * ceil((double)num_n / gn) < X + W * ceil((double)num_m / gm);
  a.grp = a.group_n ? gn : gm;
  a.wait_cycles = wait_limit.load(std::memory_order_relaxed);
  int workers = std::max(1, std::min(num_m * num_n, sms / CG));
  if constexpr (EPI == EPI_SCORES) {
    // Each block keeps to one tile of rows where that costs no round of tiles: its sums are joined on the way, and few are left to be joined behind it
    const int per = workers / num_m;
    a.carry = per > 0 && (num_n + per - 1) / per <= (num_m * num_n + workers - 1) / workers;
    if (a.carry) {
      workers = per * num_m;
      a.group_n = 0;
      a.grp = num_m;
    }
    if (slots) *slots = (a.carry ? per : num_n) * C::EG;
  }
  Launch l(dim3(workers * CG), C::THREADS, C::SMEM, stream, CG);
  return cudaLaunchKernelEx(&l.cfg, tile_kernel<I8, BN, CG, EPI>, mx, mw, mc, a);
}

template <bool I8>
cudaError_t launch_few(cudaStream_t stream, const HeadScoresArgs& g, const TileArgs& t, int sms, int* slots) {
  static std::atomic<uint64_t> asked{0};
  cudaError_t e = ask_smem(few_scores_kernel<I8>, kFewSmem, asked);
  if (e != cudaSuccess) return e;
  const int box = (g.T + 15) / 16 * 16, stage = (box + SN) * KB, stages = std::min(12, (kFewSmem - 1024) / stage);
  CUtensorMap mx, mw;
  if (!operand_map<I8>(&mx, {g.x, g.ldx, g.T}, g.H, box) || !operand_map<I8>(&mw, {g.w, g.ldw, g.V}, g.H, SN)) return cudaErrorInvalidValue;
  const FewArgs a{g.x_scales, g.w_scales, g.T, g.V, ((I8 ? g.H : 2 * g.H) + KB - 1) / KB, box, 2 * box <= 32 ? 32 : 2 * box <= 64 ? 64 : 128, stages, t.targets, t.part, t.at, t.scale, t.cap,
                  wait_limit.load(std::memory_order_relaxed)};
  const int workers = std::min((g.V + SN - 1) / SN, sms);
  *slots = workers * 4;
  Launch l(dim3(workers), kFewThreads, stages * stage + 1024, stream, 1);
  return cudaLaunchKernelEx(&l.cfg, few_scores_kernel<I8>, mx, mw, a);
}

// K in parts: the blocks of a cluster.  More parts while all clusters are resident at once: with two blocks per SM (up to 64 rows of X, 108 KB) some 260 blocks, with one some 130,
// as a cluster lies within one group of SMs (us in 4 | 5 | 6 parts, 1 x 6144 x 4096: 8.7 | 8.9 | 13.9, 300 x 1024 x 8192: 12.1 | 11.1 | 17.1), and four blocks of K are left for each.
struct SplitPlan {
  int parts, stages, smem, rounds;
};
SplitPlan split_plan(int M, int N, int kbs, int sms) {
  const int box = std::min(TM, (M + 15) / 16 * 16);
  const long long tiles = (long long)((M + TM - 1) / TM) * ((N + SN - 1) / SN), room = std::max(1LL, (long long)((box <= 64 ? 2 : 1) * 0.88 * sms));
  int parts = 1;
  while (parts < 8 && tiles * (parts + 1) <= room && kbs >= 4 * (parts + 1)) ++parts;
  const int stage = box * KB + SN * KB, most = (kbs + parts - 1) / parts;
  const int stages = std::min(std::min(most, 12), (box <= 64 ? 108 : 216) * 1024 / stage);
  return {parts, stages, std::max(stages * stage, box * kDump * 4) + 1024, (int)std::min<long long>((tiles * parts + room - 1) / room, INT32_MAX)};
}
double split_us(int M, int N, int kbs, int sms, double load_us, bool resid) {  // (fitted as below)
  const SplitPlan p = split_plan(M, N, kbs, sms);
  return std::max(p.rounds * ((kbs + p.parts - 1) / p.parts * 0.26 + std::min(M, TM) * (resid ? 0.076 : 0.034) / p.parts), load_us) + 3.5 + std::min(M, TM) / 40.0;
}

cudaError_t launch_split(cudaStream_t stream, const GemmQ8Args& g, int sms) {
  static std::atomic<uint64_t> asked{0};
  cudaError_t e = ask_smem(split_kernel, 220 * 1024, asked);
  if (e != cudaSuccess) return e;
  const int kbs = (g.K + KB - 1) / KB, box = std::min(TM, (g.M + 15) / 16 * 16);
  const SplitPlan p = split_plan(g.M, g.N, kbs, sms);
  CUtensorMap mx, mw;
  if (!operand_map<true>(&mx, {g.x, g.ldx, g.M}, g.K, box) || !operand_map<true>(&mw, {g.w, g.ldw, g.N}, g.K, 64)) return cudaErrorInvalidValue;
  const SplitArgs a{g.x_scales, g.w_scales, has_bias(g.epi) ? g.bias : nullptr, has_resid(g.epi) ? g.r : nullptr, g.out, g.ldo, g.ldr, g.M, g.N, kbs, (int)g.epi, box, box <= 32 ? 32 : box <= 64 ? 64 : 128, p.stages,
                    wait_limit.load(std::memory_order_relaxed)};
  Launch l(dim3(p.parts, (g.N + SN - 1) / SN, (g.M + TM - 1) / TM), kSplitThreads, p.smem, stream, p.parts);
  return cudaLaunchKernelEx(&l.cfg, split_kernel, mx, mw, a);
}

// Which kernel, which tiles: the one whose rounds end first.  Per shape: us per block of K of one tile, the least that a round takes (what follows the products: plain | gelu, gated
// units and residuals), what a launch takes beside them (a pair starts later, a wide last tile is longer on its way out); 3.6 (4.8 for the latter kind) for all.  Fitted to 1690 runs of
// 283 products, 1 x 2048 x 2048 to 13800 x 2304 x 768: what it chooses takes 0.3% more than the fastest there on the mean.  Some of these (us):
//                            256 x 256 pair  192 pair  128 pair  128 x 256  128 x 192  128 x 128  parts of K
//   8192 x 28672 x  4096            575         639       796       651        736        889
//   1100 x  4096 x 14336 (R)         73.9        63.0      86.5      53.4       79.8       67.9
//    512 x  2048 x  8192             24.3        21.6      20.6      28.2       26.6       22.0
//  13800 x  2304 x   768 (bias)      32.8        29.5      33.7      31.3       30.6       34.7
//  13800 x   768 x   768 (R)         25.5        20.8      22.5      25.1       21.0       22.3
//  13800 x  2304 x   768 (gelu)      47.0        42.6      44.8      43.0       42.9       45.2
//    777 x  8960 x  1536 (gelu)      19.9        20.4      21.4      19.1       21.0       21.7
//    200 x  4096 x  4096             15.4        14.0      13.1      16.8       15.6       13.4      19.3
//    128 x  4096 x  4096                                   13.2      17.3                  13.4      10.7
//     32 x 28672 x  4096                                   36.0      24.2                  26.2      22.6
//    200 x   512 x 14336                                   31.2      44.9                  34.3      10.8
// A row's sums are whole numbers: its bits do not depend on the choice.
struct TileShape {
  int bn, cg;
  double kb, floor, deep_floor, beside;
};
constexpr TileShape kShapes[] = {{256, 2, 0.352, 3.6, 6.2, 2.05}, {192, 2, 0.295, 2.75, 4.15, 1.9}, {128, 2, 0.239, 2.1, 2.7, 1.75}, {256, 1, 0.439, 4.0, 5.9, 0.65}, {192, 1, 0.414, 3.2, 4.4, 0.5}, {128, 1, 0.317, 2.35, 3.1, 0.35}};

template <int EPI>
cudaError_t launch_product(cudaStream_t stream, const GemmQ8Args& g, int sms) {
  constexpr bool kGlu = EPI == EPI_SWIGLU, kDeep = kGlu || EPI == EPI_BIAS_GELU || has_resid(EPI);
  const int kbs = (g.K + KB - 1) / KB;
  const double load_us = (double)g.N * g.K / 6.2e6 + 0.9;  // (few rows: W's way from memory)
  const TileShape* pick = nullptr;
  double best = 1e30;
  for (const TileShape& t : kShapes) {
    if ((t.cg == 2 && sms < 2) || (kGlu && t.bn != 256)) continue;
    const long long tiles = (long long)((g.M + TM * t.cg - 1) / (TM * t.cg)) * ((g.N + t.bn - 1) / t.bn), workers = sms / t.cg;
    const double us = std::max((double)((tiles + workers - 1) / workers) * std::max(kbs * t.kb, kDeep ? t.deep_floor : t.floor), load_us) + t.beside + (kDeep ? 4.8 : 3.6);
    if (us < best) {
      best = us;
      pick = &t;
    }
  }
  if (g.N <= 65535 * SN && g.M <= 65535 * TM && split_us(g.M, g.N, kbs, sms, load_us, has_resid(EPI)) < best) return launch_split(stream, g, sms);
  TileArgs a{};
  a.xs = g.x_scales;
  a.ws = g.w_scales;
  a.bias = g.bias;
  a.r = g.r;
  a.out = g.out;
  a.ldo = g.ldo;
  a.ldr = g.ldr;
  a.M = g.M;
  a.N = g.N;
  const Operand x{g.x, g.ldx, g.M}, w{g.w, g.ldw, g.N};
  switch (pick->bn * 10 + pick->cg) {
    case 2562: return launch_tiles<true, 256, 2, EPI>(stream, a, x, w, g.K, sms);
    case 2561: return launch_tiles<true, 256, 1, EPI>(stream, a, x, w, g.K, sms);
    case 1922:
      if constexpr (!kGlu) return launch_tiles<true, 192, 2, EPI>(stream, a, x, w, g.K, sms);
      break;
    case 1921:
      if constexpr (!kGlu) return launch_tiles<true, 192, 1, EPI>(stream, a, x, w, g.K, sms);
      break;
    case 1282:
      if constexpr (!kGlu) return launch_tiles<true, 128, 2, EPI>(stream, a, x, w, g.K, sms);
      break;
    case 1281:
      if constexpr (!kGlu) return launch_tiles<true, 128, 1, EPI>(stream, a, x, w, g.K, sms);
      break;
  }
  return cudaErrorInvalidValue;
}

constexpr int kMostK = 131056;  // 127^2 K stays below 2^31 (codes of -128 that a caller may have: 128^2 K too)

}  // namespace

long long q8_wait_cycles(long long cycles) { return wait_limit.exchange(cycles); }
cudaError_t q8_status() {
  unsigned ran_out = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&ran_out, wait_ran_out, sizeof ran_out);
  if (e != cudaSuccess || !ran_out) return e;
  const unsigned none = 0;
  e = cudaMemcpyToSymbol(wait_ran_out, &none, sizeof none);
  return e == cudaSuccess ? cudaErrorLaunchTimeout : e;
}

cudaError_t gemm_q8(cudaStream_t stream, const GemmQ8Args& g) {
  const bool f32 = g.epi == EPI_F32, glu = g.epi == EPI_SWIGLU;
  if (g.epi < EPI_NONE || g.epi > EPI_F32 || g.M < 0 || g.M > (1 << 30) || g.N < 1 || g.N > (1 << 30) || g.K < 1 || g.K > kMostK || (glu && g.N % 256)) return cudaErrorInvalidValue;
  if (g.M == 0) return cudaSuccess;
  if (!g.x || ((uintptr_t)g.x & 15) || g.ldx < g.K || g.ldx % 16 || !g.w || ((uintptr_t)g.w & 15) || g.ldw < g.K || g.ldw % 16) return cudaErrorInvalidValue;
  if (!g.x_scales || ((uintptr_t)g.x_scales & 3) || !g.w_scales || ((uintptr_t)g.w_scales & 15)) return cudaErrorInvalidValue;
  const int n_out = glu ? g.N / 2 : g.N;
  if (!g.out || ((uintptr_t)g.out & 15) || g.ldo < n_out || g.ldo % (f32 ? 4 : 8)) return cudaErrorInvalidValue;
  if ((has_bias(g.epi) && (!g.bias || ((uintptr_t)g.bias & 15))) || (has_resid(g.epi) && (!g.r || ((uintptr_t)g.r & 15) || g.ldr < n_out || g.ldr % 8))) return cudaErrorInvalidValue;
  const int sms = device_sms();
  if (sms <= 0) return cudaErrorNoDevice;
  switch (g.epi) {
    case EPI_NONE: return launch_product<EPI_NONE>(stream, g, sms);
    case EPI_BIAS: return launch_product<EPI_BIAS>(stream, g, sms);
    case EPI_BIAS_GELU: return launch_product<EPI_BIAS_GELU>(stream, g, sms);
    case EPI_RESID: return launch_product<EPI_RESID>(stream, g, sms);
    case EPI_BIAS_RESID: return launch_product<EPI_BIAS_RESID>(stream, g, sms);
    case EPI_SWIGLU: return launch_product<EPI_SWIGLU>(stream, g, sms);
    default: return launch_product<EPI_F32>(stream, g, sms);
  }
}

namespace {
bool score_sizes_ok(int T, int V) { return T >= 0 && T <= (1 << 28) && V >= 1 && V <= (1 << 30); }
// Above 128 rows: pairs' tiles of 256 rows or blocks' of 128, whichever rounds end first: us per block of K, the least of a round (what follows the products), the pair's later start,
// as in kShapes.  (us of pairs | blocks: 200 x 128256 x 4096 in bf16 210 | 231, 300 rows 353 | 322, 300 rows of codes, H = 1536, with a cap 84 | 73, 384 x 30522 x 768 in bf16 28.0 | 24.8,
// 512 x 50000 x 2048 78 | 88, 1000 x 128256 x 1536 268 | 296, 1100 x 30522 x 768 50.8 | 48.8, 700 x 151936 x 1536 of codes with a cap 146 | 151: what follows the products of a block takes a
// little longer the more of them there are beside it, 0.03 us per block of K by these runs.)
bool pairs_score(int T, int V, int kbs, bool i8, bool cap, int sms) {
  const long long wide = (V + 255) / 256, pairs = sms / 2;
  const double least = (i8 ? 3.2 : 4.9) + (cap ? 2.3 : 0.0);
  const double two = (double)((wide * ((T + 255) / 256) + pairs - 1) / pairs) * std::max(kbs * 0.37, least) + 1.4;
  const double one = (double)((wide * ((T + 127) / 128) + sms - 1) / sms) * std::max(kbs * 0.46, least + kbs * 0.03);
  return two <= one;
}
int score_slots(int T, int V) { return T <= TM ? (V + 127) / 128 * 4 : (V + 255) / 256 * 4; }  // at most
}  // namespace

size_t head_scores_workspace_floats(int T, int V) { return score_sizes_ok(T, V) ? (size_t)T * (3 * (size_t)score_slots(T, V) + 1) : 0; }

cudaError_t head_scores(cudaStream_t stream, const HeadScoresArgs& g) {
  const bool i8 = g.x_scales != nullptr;
  if (!score_sizes_ok(g.T, g.V) || g.H < 1 || g.H > (i8 ? kMostK : 1 << 29) || i8 != (g.w_scales != nullptr) || !(fabsf(g.scale) < INFINITY) || !(g.softcap >= 0.f) ||
      !(g.softcap < INFINITY))
    return cudaErrorInvalidValue;
  if (g.T == 0) return cudaSuccess;
  const int step = i8 ? 16 : 8;
  if (!g.x || ((uintptr_t)g.x & 15) || g.ldx < g.H || g.ldx % step || !g.w || ((uintptr_t)g.w & 15) || g.ldw < g.H || g.ldw % step) return cudaErrorInvalidValue;
  if (((uintptr_t)g.x_scales & 3) || ((uintptr_t)g.w_scales & 15) || ((uintptr_t)g.targets & 3) || ((uintptr_t)g.lp & 3) || ((uintptr_t)g.entropy & 3)) return cudaErrorInvalidValue;
  if (!g.workspace || ((uintptr_t)g.workspace & 3) || (g.lp && !g.targets) || (!g.lp && !g.entropy)) return cudaErrorInvalidValue;
  const int sms = device_sms();
  if (sms <= 0) return cudaErrorNoDevice;
  TileArgs a{};
  a.xs = g.x_scales;
  a.ws = g.w_scales;
  a.M = g.T;
  a.N = g.V;
  a.targets = g.lp ? g.targets : nullptr;
  a.part = g.workspace;
  a.at = g.workspace + 3 * (size_t)score_slots(g.T, g.V) * g.T;
  a.scale = g.scale;
  a.cap = {g.softcap, std::min(1.f / g.softcap, 3.4028235e38f)};  // (a logit of 0 stays 0 under the smallest caps)
  const Operand x{g.x, g.ldx, g.T}, w{g.w, g.ldw, g.V};
  if (sms < 2) return cudaErrorInvalidConfiguration;
  cudaError_t e;
  int slots = 0;
  if (g.T <= kFewRows) e = i8 ? launch_few<true>(stream, g, a, sms, &slots) : launch_few<false>(stream, g, a, sms, &slots);
  else if (g.T <= TM) e = i8 ? launch_tiles<true, 128, 1, EPI_SCORES>(stream, a, x, w, g.H, sms, &slots) : launch_tiles<false, 128, 1, EPI_SCORES>(stream, a, x, w, g.H, sms, &slots);
  else if (pairs_score(g.T, g.V, ((i8 ? 1 : 2) * g.H + KB - 1) / KB, i8, g.softcap > 0.f, sms))
    e = i8 ? launch_tiles<true, 256, 2, EPI_SCORES>(stream, a, x, w, g.H, sms, &slots) : launch_tiles<false, 256, 2, EPI_SCORES>(stream, a, x, w, g.H, sms, &slots);
  else
    e = i8 ? launch_tiles<true, 256, 1, EPI_SCORES>(stream, a, x, w, g.H, sms, &slots) : launch_tiles<false, 256, 1, EPI_SCORES>(stream, a, x, w, g.H, sms, &slots);
  if (e != cudaSuccess) return e;
  // Few sums: many threads per row (a row of a head of 151936 x 1536 in codes 51.5 -> 47.8 us).  Blocks that wait beside the kernel before for its end cost it more than their start
  // is worth once there are more than a few (us started early | behind it: 4 rows of a 1 GB head 187.9 | 189.9, 16 rows 195.8 | 188.5, 128 rows 196.9 | 191.8)
  const bool early = g.T <= 8;
  if (slots <= 600)
    return launch_k(join_scores_kernel<128, 2>, dim3((g.T + 1) / 2), dim3(128), 0, stream, early, (const float*)a.part, (const float*)a.at, g.targets, g.lp, g.entropy, slots, g.T, g.V);
  return launch_k(join_scores_kernel<512, 8>, dim3((g.T + 7) / 8), dim3(512), 0, stream, early, (const float*)a.part, (const float*)a.at, g.targets, g.lp, g.entropy, slots, g.T, g.V);
}

}  // namespace hb

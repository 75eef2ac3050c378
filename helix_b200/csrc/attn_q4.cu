// Attention of the last rows of each sequence over a 4-bit paged cache (layout: quant4.cuh): single tokens, and portions of several rows.
//
//   o = sum_j p_j v_j,  p = softmax over the visible j of s_j,  s = scale q.k (capped: cap tanh(s / cap)),  a sink adds exp(sink) to the denominator
//
// The columns of a block are (row, query head) pairs of one kv head.  Two kernels: up to 16 columns per block, for single tokens and short portions, and 128
// (attn_q4_wide_kernel below) where a sequence and kv head may have 256 or more.
//
// The first takes eight columns per product: S^T[16 positions x 8 columns] = K q^T and O^T[16 entries x 8 columns] += V^T P^T as warp-wide 16 x 8 x 16 products.
// Both operands that come from the cache are then the 16-row one, the codes go straight from their words to its registers, and no cached byte passes through
// shared memory twice.  (The tensor-memory path wants the widened entries in shared memory: four times the cache's bytes written there and read again.)
// Instructions bound it (HBM gives a position of a kv head of 128 entries 25 issue slots), the products least of all.
//   c - 8 is exact in fp16.  (Codes as they are, numbers below fp16's smallest normal one, with the 8 taken off by a further product, save three
//      of eight instructions per word, but such products are summed to some 14 bits only: results whose codes are near 8 were off by 2^-15 of a group's weight.)
//   S: the products of a group of 32 entries are summed by themselves, then times the key group's scale in fp32.
//   O: the value group's scale depends on the position, which is summed over: it goes into P^T, one operand per group, fp16 (bf16 would add as much
//      error as the output's own rounding; here two roundings of at most 2^-11 each, and 2^-35 of the largest weight for weights far below it).  A
//      group's scales are brought near 1 by a power of two that follows their largest finite one so far, as the running maximum does for the
//      scores; a share in which some lie below 2^-16 of it is done again in fp32 (share_in_fp32).
//   q: fp16 after a power of two per column (bf16 has fewer bits; entries 2^-27 of the column's largest and below lose some).
// Softmax statistics and sums are fp32.  A warp takes every fourth page of the block's share by itself; the four meet at the end.
//
// A sequence of more than `split` pages is cut into as few even shares as none is larger, so a row's bits depend on its own sequence, `split` and whether
// the launch allows 256 columns, not on who shares it.
// Sequences of more than one share leave (O, m, l) per share in the workspace, which a second kernel joins in order.
//
// Measured (8 kv heads of 128 entries, 32 query heads): 32 sequences of 1.5k to 2.2k positions 25 us (68 MB, 41 % of the copy rate: two blocks on most SMs
// and one on the others, some 5 us of launch, first loads and last sums), 74 of 2k 39 us, 32 of 8k 66 us (302 MB, 70 %: 18.5 instructions per position and kv
// head at 65 % of the issue slots; parts left out in a copy, at 2k: 7 % less without the loads, 12 % without the 8 taken off the codes, 2 % without V's
// products), three of 9k to 131k 60 us (242 MB, 61 %; 67 on another GPU).  Also tried: scores in shared memory and rolled loops (a fifth more instructions), e4m3 products (widened to
// fp16 by further instructions on this chip: 41 -> 52), pages dealt evenly over all blocks by the launch's lengths (two runs of pages per block: 26 -> 37), clusters
// that join their sums through distributed shared memory (one sequence of 2k 6.4 -> 7.2, 32 of 8k 66 -> 77).
#include <math.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "quant4.cuh"

namespace hb {
namespace {

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int PAGE = q4::kPage;
constexpr int kWideCols = 128;  // columns of a block of the kernel for portions
constexpr int SLOTS = 3;  // halves (K or V) of pages that a warp has in shared memory
constexpr float kLog2e = 1.4426950408889634f;
// Powers of two that a share's value scales of one group may differ by, beyond which share_in_fp32 takes it.  A weight times its scale is an fp16 operand of at most
// 2^15: scales 2^-16 of the largest still have all their bits, weights down to 2^-12 of the largest all of theirs, and smaller ones are off by 2^-23 of it at
// most.  Where models' values lie: 2^4 between neighbours, 2^8 between a first position and the others.
constexpr int kRange = 16;

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// cap tanh(x / cap) as log2 of a weight.  tanh(y) = 1 - 2 / (e^2y + 1) takes two transcendentals and is off by some 2^-21 of the cap however small the score: 2^-15 of a
// weight at kCapByExp, and more than the score itself from a cap of 10^7 on.  Above, tanh itself.
constexpr float kCapByExp = 64.f;
struct Cap {
  float in, out;
  __device__ __forceinline__ explicit Cap(float cap) : in(fminf(2.f * kLog2e / cap, 3e38f)), out(cap * kLog2e) {}  // (of a subnormal cap: no infinity, 0 stays 0)
  __device__ __forceinline__ float by_exp(float x) const { return fmaf(-2.f * out, __fdividef(1.f, exp2_fast(x * in) + 1.f), out); }
};
__device__ __noinline__ float capped_far(float x, float cap) { return cap * tanhf(x / cap) * kLog2e; }

// What a tile of columns of one sequence and kv head covers
struct Tile {
  int row0;            // its first packed row; column c belongs to row0 + (rest + c) / G, head (rest + c) % G
  int rest;
  int cols;            // columns of the tile
  int pos0;            // position of row0
  int lo, hi;          // positions that some column sees
  int page0, pages;    // pages that hold them
  int splits;          // shares: pages page0 + pages s / splits and on
};
__device__ __forceinline__ int div_g(const AttnQ4Args& a, int x) { return (int)((unsigned long long)x * a.inv_group >> 32); }
__device__ __forceinline__ Tile tile_of(const AttnQ4Args& a, int b, int ct, int cols_per_tile) {
  Tile t;
  const int first = a.cu_seqlens ? min(max(a.cu_seqlens[b], 0), a.T) : b;
  const int rows = a.cu_seqlens ? min(min(max(a.cu_seqlens[b + 1], 0), a.T) - first, a.max_q_len) : 1;
  const int kv = min(max(a.kv_lens[b], 0), a.kv_bound);
  const int col0 = ct * cols_per_tile;
  const int i0 = a.max_q_len == 1 && a.group <= cols_per_tile ? 0 : col0 / a.group;
  t.row0 = first + i0;
  t.rest = col0 - i0 * a.group;
  t.cols = min(max(rows, 0) * a.group - col0, cols_per_tile);
  t.pos0 = kv - rows + i0;
  t.hi = min(max(t.pos0 + div_g(a, t.rest + max(t.cols, 1) - 1) + 1, 0), kv);
  t.lo = a.window > 0 ? max(t.pos0 - a.window + 1, 0) : 0;
  t.page0 = t.lo / PAGE;
  t.pages = t.cols > 0 ? max((t.hi + PAGE - 1) / PAGE - t.page0, 0) : 0;
  t.splits = t.pages <= a.split_pages ? min(t.pages, 1) : (t.pages + a.split_pages - 1) / a.split_pages;
  return t;
}

template <int D, int NT>
struct Cfg {
  static constexpr int J = D / q4::kGroup;
  static constexpr int BLOCK = q4::block_bytes(D);
  static constexpr int COLS = 8 * NT;
  static constexpr int PER_WARP = SLOTS * BLOCK;
  static constexpr int RING = kWarps * PER_WARP;
  static constexpr int MERGE = kWarps * COLS * (D + 4) * 4;  // [warp][column]: D sums, maximum, sum of weights, and 8 bytes that keep the rows aligned
  static constexpr int SMEM = RING > MERGE ? RING : MERGE;
  static constexpr int BLOCKS = NT == 2 ? (D == 128 ? 2 : 3) : (D == 128 ? 4 : 5);  // per SM, by registers and shared memory
};

// the 16 (D = 128), 8 (D = 64) or 4 (D = 32: half as many) bytes that a lane takes of a row or pair
template <int D>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[D / 32]) {
  if constexpr (D == 128) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else if constexpr (D == 64) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
// the bf16 scales of one position
template <int D>
__device__ __forceinline__ void load_scales(const uint8_t* p, float (&s)[D / 32]) {
  if constexpr (D == 128) {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    s[0] = q4::bf16_lo(u.x); s[1] = q4::bf16_hi(u.x); s[2] = q4::bf16_lo(u.y); s[3] = q4::bf16_hi(u.y);
  } else {
    const uint32_t u = *reinterpret_cast<const uint32_t*>(p);
    s[0] = q4::bf16_lo(u); s[1] = q4::bf16_hi(u);
  }
}

__device__ __forceinline__ void store4(bf16* dst, float4 x, float sum) {
  const float y[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) dst[i] = __float2bfloat16(sum == 0.f ? 0.f : y[i] / sum);
}

// the larger magnitude of two bf16 entries that is finite, as its bits
__device__ __forceinline__ uint32_t finite_top(uint32_t u) {
  const uint32_t lo = u & 0x7fffu, hi = (u >> 16) & 0x7fffu;
  return max(lo < 0x7f80u ? lo : 0u, hi < 0x7f80u ? hi : 0u);
}
template <int D>
__device__ __forceinline__ void zero_columns(const AttnQ4Args& a, const Tile& tile, int kvh) {
  for (int i = threadIdx.x; i < tile.cols * D; i += kThreads) {
    const int c = i / D, r = div_g(a, tile.rest + c);
    a.out[(size_t)(tile.row0 + r) * a.ldo + (size_t)(kvh * a.group + tile.rest + c - r * a.group) * D + i % D] = __float2bfloat16(0.f);
  }
}

// The smallest finite scale other than 0 of each value group that a lane has met, two groups to a word, as the signed 16-bit number (bits - 1) - 2^15: 0 and what
// is not seen become 2^15 - 1, above all of them.
constexpr uint32_t kNoScale = 0x7fff7fffu;
__device__ __forceinline__ uint32_t smallest_scale(uint32_t low, uint32_t x, uint32_t y) {
  return __vmins2(__vmins2(low, (x | 0x80008000u) - 0x00010001u), (y | 0x80008000u) - 0x00010001u);
}
// Whether some scale of group j is less than 2^-range of the group's largest (exponent field `top`)
__device__ __forceinline__ bool out_of_range(uint32_t low, int j, int top, int range) {
  return (((int)(short)(j & 1 ? low >> 16 : low) + 32769) >> 7) + range < top;
}

// A share by itself in fp32, whatever its scales: for those whose value scales differ so much that the operands of the kernels below would lose bits of the small ones.
// They are brought to fp16 under the largest of the tile's positions, and that one may be of a position that a row does not see, or of next to no weight.  A warp takes
// four columns at a time, so that a page is widened once for them: for the scores a lane takes two neighbouring positions, for the sums the entries 32 j + lane.
// Models do not come here, so it is short, not fast (8 kv heads of 128 entries, 4 query heads each): 32 rows of one sequence of 4096 take 385 us instead of 23,
// 512 rows 4800 instead of 97, single tokens of 32 sequences of 2k 735 instead of 30.
template <int D, bool CAP>
__device__ __noinline__ void share_in_fp32(const AttnQ4Args& a, int ct, int cols_per_tile, int share) {
  constexpr int J = D / q4::kGroup, N = 4;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.z, kvh = blockIdx.y % a.Hkv;
  const Tile tile = tile_of(a, b, ct, cols_per_tile);
  const int p_begin = tile.page0 + (int)((long long)tile.pages * share / tile.splits);
  const int p_end = tile.page0 + (int)((long long)tile.pages * (share + 1) / tile.splits);
  const int32_t* table = a.page_table + (size_t)b * a.max_pages;
  for (int c = warp * N; c < tile.cols; c += blockDim.x / 32 * N) {
    int row[N], head[N], last[N], first[N];
    const bf16* q[N];
    float m[N], l[N], o[N][J];
#pragma unroll
    for (int n = 0; n < N; ++n) {  // (behind the tile's last column: that one again, not stored)
      const int at = tile.rest + min(c + n, tile.cols - 1), r = div_g(a, at);
      row[n] = tile.row0 + r;
      head[n] = kvh * a.group + at - r * a.group;
      last[n] = tile.pos0 + r;
      first[n] = a.window > 0 ? last[n] - a.window + 1 : 0;
      q[n] = a.q + (size_t)row[n] * a.ldq + (size_t)head[n] * D;
      m[n] = -INFINITY;
      l[n] = 0.f;
#pragma unroll
      for (int j = 0; j < J; ++j) o[n][j] = 0.f;
    }
    for (int p = p_begin; p < p_end; ++p) {
      const int id = table[p], pos = p * PAGE + 2 * lane;
      if (id < 0 || id >= a.num_pages) continue;
      const uint8_t* kb = a.k_cache + ((size_t)id * a.Hkv + kvh) * q4::block_bytes(D);
      const uint8_t* vb = a.v_cache + ((size_t)id * a.Hkv + kvh) * q4::block_bytes(D);
      float s[2][N] = {};
      uint32_t seen[2][N];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        for (int j = 0; j < J; ++j) {
          float group[N] = {};
          for (int t = 0; t < 4; ++t) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(kb + (2 * lane + h) * (D / 2) + t * (D / 8) + 4 * j);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const float code = (float)((int)(w >> (4 * (i / 2 + 4 * (i & 1))) & 15u) - 8);
#pragma unroll
              for (int n = 0; n < N; ++n) group[n] = fmaf(__bfloat162float(q[n][32 * j + 8 * t + i]), code, group[n]);
            }
          }
          const float d = __bfloat162float(*reinterpret_cast<const bf16*>(kb + q4::code_bytes(D) + ((2 * lane + h) * J + j) * 2));
#pragma unroll
          for (int n = 0; n < N; ++n) s[h][n] = fmaf(d, group[n], s[h][n]);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
          float x = s[h][n] * a.scale;
          x = CAP ? capped_far(x, a.softcap) : x * kLog2e;
          const bool sees = pos + h >= first[n] && pos + h <= last[n];
          s[h][n] = sees ? x : -INFINITY;
          seen[h][n] = __ballot_sync(0xffffffffu, sees);
        }
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        float top = fmaxf(s[0][n], s[1][n]);
#pragma unroll
        for (int w = 1; w < 32; w <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, w));
        top = fmaxf(m[n], top);
        const float f = m[n] == top ? 1.f : exp2_fast(m[n] - top), ref = top == -INFINITY ? 0.f : top;
        m[n] = top;
        s[0][n] = exp2_fast(s[0][n] - ref);
        s[1][n] = exp2_fast(s[1][n] - ref);
        l[n] = fmaf(l[n], f, s[0][n] + s[1][n]);  // (a lane's own positions)
#pragma unroll
        for (int j = 0; j < J; ++j) o[n][j] *= f;
      }
      for (int x = 0; x < PAGE / 2; ++x)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[J];
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const uint32_t word = *reinterpret_cast<const uint32_t*>(vb + x * D + ((lane >> 2) ^ q4::place_xor(D, x)) * (D / 8) + 4 * j);
            const float d = __bfloat162float(*reinterpret_cast<const bf16*>(vb + q4::code_bytes(D) + ((2 * x + h) * J + j) * 2));
            v[j] = d * (float)((int)(word >> (4 * (lane & 3) + 16 * h) & 15u) - 8);
          }
#pragma unroll
          for (int n = 0; n < N; ++n) {
            const float w = __shfl_sync(0xffffffffu, s[h][n], x);
            if (!(seen[h][n] >> x & 1)) continue;
#pragma unroll
            for (int j = 0; j < J; ++j) o[n][j] = fmaf(w, v[j], o[n][j]);
          }
        }
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
#pragma unroll
      for (int w = 1; w < 32; w <<= 1) l[n] += __shfl_xor_sync(0xffffffffu, l[n], w);
      if (c + n >= tile.cols) continue;
      if (tile.splits == 1) {
        const float sink = a.sink ? __bfloat162float(a.sink[head[n]]) * kLog2e : -INFINITY;
        const float top = fmaxf(m[n], sink), ref = top == -INFINITY ? 0.f : top, f = exp2_fast(m[n] - ref), sum = fmaf(l[n], f, exp2_fast(sink - ref));
#pragma unroll
        for (int j = 0; j < J; ++j) a.out[(size_t)row[n] * a.ldo + (size_t)head[n] * D + 32 * j + lane] = __float2bfloat16(sum == 0.f ? 0.f : o[n][j] * f / sum);
      } else {
        float* part = a.workspace + (((size_t)row[n] * a.Hq + head[n]) * a.max_splits + share) * (D + 4);
#pragma unroll
        for (int j = 0; j < J; ++j) part[32 * j + lane] = o[n][j];
        if (lane == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m[n], l[n]);
      }
    }
  }
}

template <int D, int NT, bool CAP>
__global__ void __launch_bounds__(kThreads, Cfg<D, NT>::BLOCKS) attn_q4_kernel(const __grid_constant__ AttnQ4Args a) {
  using C = Cfg<D, NT>;
  constexpr int J = C::J;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = a.group;
  const int b = blockIdx.z, ct = a.tile0 + blockIdx.y / a.Hkv, kvh = blockIdx.y % a.Hkv;
  const Tile tile = tile_of(a, b, ct, C::COLS);
  if (tile.cols <= 0) return;
  auto row_of = [&](int c) { return div_g(a, tile.rest + c); };  // row of column c
  const int shares = tile.splits;
  if (tile.pages == 0) {  // nothing to see
    if (blockIdx.x == 0) zero_columns<D>(a, tile, kvh);
    return;
  }
  if ((int)blockIdx.x >= shares) return;
  const int p_begin = tile.page0 + (int)((long long)tile.pages * blockIdx.x / shares);
  const int p_end = tile.page0 + (int)((long long)tile.pages * (blockIdx.x + 1) / shares);

  uint8_t* ring = smem + warp * C::PER_WARP;
  const int32_t* table = a.page_table + (size_t)b * a.max_pages;
  const size_t block0 = (size_t)kvh * C::BLOCK + lane * 16, page_stride = (size_t)a.Hkv * C::BLOCK;
  // The warp's pages are p_begin + warp + 4 i.  Lane i % 32 holds the number of page i, -1 for one that is none: its positions are not seen.
  // Halves of pages go through the slots in order, K_0 V_0 K_1 V_1 ..., each a copy group of its own.
  const int n_mine = (p_end - p_begin - warp + kWarps - 1) / kWarps;
  int ids = -1;
  auto number_of = [&](int i) {
    if ((i & 31) == 0) {
      ids = -1;
      if (i + lane < n_mine) {
        const int id = table[p_begin + warp + kWarps * (i + lane)];
        if (id >= 0 && id < a.num_pages) ids = id;
      }
    }
    const int id = __shfl_sync(0xffffffffu, ids, i & 31);
    return i < n_mine ? id : -1;
  };
  auto fetch = [&](const uint8_t* plane, int id, int slot) {
    if (id >= 0) {
      const uint8_t* src = plane + (size_t)id * page_stride + block0;
      uint8_t* dst = ring + slot * C::BLOCK + lane * 16;
#pragma unroll
      for (int c = 0; c < C::BLOCK; c += 512)
        if (c + 512 <= C::BLOCK || c + lane * 16 < C::BLOCK) copy16(dst + c, src + c);
    }
    copy_commit();
  };
  int id = number_of(0);
  fetch(a.k_cache, id, 0);
  fetch(a.v_cache, id, 1);
  int id_next = number_of(1);
  fetch(a.k_cache, id_next, 2);

  // q as the 8-column operand: lane (g, t) holds entries 32 j + 8 t .. + 7 of column g
  uint32_t qr[NT][J][4];
  float mul[NT][2];               // what brings a column's sums to log2 of its weights (to scores, where they are capped)
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const int c = n * 8 + g;
    uint4 raw[J];
#pragma unroll
    for (int j = 0; j < J; ++j) raw[j] = make_uint4(0, 0, 0, 0);
    if (c < tile.cols) {
      const int r = row_of(c);
      const bf16* src = a.q + (size_t)(tile.row0 + r) * a.ldq + (size_t)(kvh * G + tile.rest + c - r * G) * D + t * 8;
#pragma unroll
      for (int j = 0; j < J; ++j) raw[j] = *reinterpret_cast<const uint4*>(src + j * 32);
    }
    uint32_t mag = 0;  // largest finite magnitude: an infinity or NaN passes as it is and takes no other entry with it
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) mag = max(mag, finite_top(w[i]));
    }
    mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 1));
    mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, 2));
    // the largest becomes [2^10, 2^11): exponent field e -> factor 2^(137 - e), kept a normal number at both ends
    const int e = max((int)(mag >> 7), 20);
    const float up = __uint_as_float((uint32_t)(264 - e) << 23), down = __uint_as_float((uint32_t)(e - 10) << 23);
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const uint32_t w[4] = {raw[j].x, raw[j].y, raw[j].z, raw[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) qr[n][j][i] = q4::pack_f16x2(q4::bf16_lo(w[i]) * up, q4::bf16_hi(w[i]) * up);
    }
    // the sign of the scale goes into q, so that the largest sum is the largest score
    const float scale = CAP ? fabsf(a.scale) : fabsf(a.scale) * kLog2e;
    if (a.scale < 0.f) {
#pragma unroll
      for (int j = 0; j < J; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) qr[n][j][i] ^= 0x80008000u;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      mul[n][i] = fmaxf(__shfl_sync(0xffffffffu, down, 4 * (2 * t + i)) * scale, 1e-37f);  // (a scale of 0 still leaves what is not seen at -inf)
  }
  auto last_of = [&](int c) { return c < tile.cols ? tile.pos0 + row_of(c) : -1; };  // positions a column sees: first_of <= j <= last_of
  auto first_of = [&](int last) { return a.window > 0 ? last - a.window + 1 : 0; };
  // every column sees a page whole that lies in [all_lo, all_hi]
  const int all_hi = tile.pos0, all_lo = first_of(tile.pos0 + row_of(tile.cols - 1));

  float o[J][2][NT][4];
  float m[NT][2], l[NT][2];  // running maximum (log2 of a weight) and sum of weights times 2^10
  int ex[J];                 // exponent field of a value group's largest scale so far
  uint32_t low[J / 2];       // and its smallest
#pragma unroll
  for (int j = 0; j < J; ++j) {
    ex[j] = 12;
    low[j / 2] = kNoScale;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][h][n][i] = 0.f;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      m[n][i] = -INFINITY;
      l[n][i] = 0.f;
    }

  int slot = 0;  // of the page's K; its V lies in the next one
  int i = 0;
  // One page.  `whole`: every column sees all of it
  auto page = [&](const int pos, auto whole_t) {
    constexpr bool whole = decltype(whole_t)::value;
    uint8_t* kb = ring + slot * C::BLOCK;
    uint8_t* vb = ring + (slot == SLOTS - 1 ? 0 : slot + 1) * C::BLOCK;
    float s[4][NT][4];
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      const int r0 = blk * 16 + g;
      uint32_t k0[J], k1[J];
      float d0[J], d1[J];
      load_words<D>(kb + r0 * (D / 2) + t * (D / 8), k0);
      load_words<D>(kb + (r0 + 8) * (D / 2) + t * (D / 8), k1);
      load_scales<D>(kb + q4::code_bytes(D) + r0 * J * 2, d0);
      load_scales<D>(kb + q4::code_bytes(D) + (r0 + 8) * J * 2, d1);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t a0[4], a1[4];
        q4::codes_f16(k0[j], a0);
        q4::codes_f16(k1[j], a1);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          float c[4];
          q4::mma_f16_first(c, a0[0], a1[0], a0[1], a1[1], qr[n][j][0], qr[n][j][1]);
          q4::mma_f16(c, a0[2], a1[2], a0[3], a1[3], qr[n][j][2], qr[n][j][3]);
#pragma unroll
          for (int h = 0; h < 4; ++h) s[blk][n][h] = j == 0 ? (h < 2 ? d0 : d1)[j] * c[h] : fmaf((h < 2 ? d0 : d1)[j], c[h], s[blk][n][h]);
        }
      }
    }
    __syncwarp();  // K's slot is free: the next page's V
    fetch(a.v_cache, id_next, slot);
    if constexpr (CAP) {  // as log2 of a weight
      const Cap cap(a.softcap);
      if (a.softcap <= kCapByExp) {
#pragma unroll
        for (int blk = 0; blk < 4; ++blk)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 4; ++h) s[blk][n][h] = cap.by_exp(s[blk][n][h] * mul[n][h & 1]);
      } else {
#pragma unroll
        for (int blk = 0; blk < 4; ++blk)
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 4; ++h) s[blk][n][h] = capped_far(s[blk][n][h] * mul[n][h & 1], a.softcap);
      }
    }
    if constexpr (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int last = last_of(n * 8 + 2 * t + h), hi = last - pos - g, lo = first_of(last) - pos - g;
#pragma unroll
          for (int blk = 0; blk < 4; ++blk) {
            if (blk * 16 > hi || blk * 16 < lo) s[blk][n][h] = -INFINITY;
            if (blk * 16 + 8 > hi || blk * 16 + 8 < lo) s[blk][n][h + 2] = -INFINITY;
          }
        }
    }
    // running maximum
    bool moved = false;
    float keep[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float x = fmaxf(s[0][n][h], s[0][n][h + 2]);
#pragma unroll
        for (int blk = 1; blk < 4; ++blk) x = fmaxf(x, fmaxf(s[blk][n][h], s[blk][n][h + 2]));
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
        if constexpr (!CAP) x *= mul[n][h];
        x = fmaxf(m[n][h], x);
        moved |= x != m[n][h];
        keep[n][h] = m[n][h];
        m[n][h] = x;
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float f = m[n][h] == keep[n][h] ? 1.f : exp2_fast(keep[n][h] - m[n][h]);  // (-inf before: 0)
          l[n][h] *= f;
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              o[j][q][n][h] *= f;
              o[j][q][n][h + 2] *= f;
            }
        }
    }
    copy_wait<2>();
    __syncwarp();
    // value scales: a lane takes those of positions 2 lane and 2 lane + 1, follows each group's largest exponent, and puts them back as
    // fp16 pairs of the two positions with the largest in [2^4, 2^5)
    {
      uint32_t w[J], pair[J];
      uint8_t* mine = vb + q4::code_bytes(D) + lane * (J * 4);
      load_words<D>(mine, w);
      const int at = pos + 2 * lane;
      uint32_t x[J / 2], y[J / 2];
      bool grow = false;
#pragma unroll
      for (int k = 0; k < J / 2; ++k) {
        x[k] = whole || (at >= tile.lo && at < tile.hi) ? w[k] & 0x7fff7fffu : 0u;
        y[k] = whole || (at + 1 >= tile.lo && at + 1 < tile.hi) ? w[J / 2 + k] & 0x7fff7fffu : 0u;
        const uint32_t fits = (uint32_t)(ex[2 * k] << 7 | ex[2 * k + 1] << 23) | 0x007f007fu;  // the largest numbers of the present exponents
        grow |= __vmaxu2(__vmaxu2(x[k], y[k]), fits) != fits;
        low[k] = smallest_scale(low[k], x[k], y[k]);
      }
      if (__any_sync(0xffffffffu, grow)) {
        auto finite = [](uint32_t u) {  // infinities and NaN: 0 (they reach their columns through the weights)
          return ((u & 0xffffu) < 0x7f80u ? u & 0xffffu : 0u) | ((u >> 16) < 0x7f80u ? u & 0xffff0000u : 0u);
        };
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const uint32_t z = __vmaxu2(finite(x[j / 2]), finite(y[j / 2]));
          const int e = max((int)(__reduce_max_sync(0xffffffffu, j & 1 ? z >> 16 : z & 0xffffu) >> 7), ex[j]);
          const float less = exp2f((float)(ex[j] - e));
          ex[j] = e;
#pragma unroll
          for (int q = 0; q < 2; ++q)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
              for (int r = 0; r < 4; ++r) o[j][q][n][r] *= less;
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float near1 = __uint_as_float((uint32_t)(258 - ex[j]) << 23);  // 2^(131 - ex)
        const uint32_t u = w[j / 2], v = w[J / 2 + j / 2];
        pair[j] = q4::pack_f16x2((j & 1 ? q4::bf16_hi(u) : q4::bf16_lo(u)) * near1, (j & 1 ? q4::bf16_hi(v) : q4::bf16_lo(v)) * near1);
      }
      if constexpr (J == 4) *reinterpret_cast<uint4*>(mine) = make_uint4(pair[0], pair[1], pair[2], pair[3]);
      else *reinterpret_cast<uint2*>(mine) = make_uint2(pair[0], pair[1]);
      __syncwarp();
    }
    float base[NT][2];  // weights times 2^10: fp16 then holds them to 2^-35 of the largest, and their products with scales to 2^-40
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int h = 0; h < 2; ++h) base[n][h] = 10.f - (m[n][h] == -INFINITY ? 0.f : m[n][h]);
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      const int p0 = blk * 8 + t;
      uint32_t v0[J], v1[J], s0[J], s1[J], b0[NT], b1[NT], see0[NT], see1[NT];
      load_words<D>(vb + p0 * D + (g ^ q4::place_xor(D, p0)) * (D / 8), v0);
      load_words<D>(vb + (p0 + 4) * D + (g ^ q4::place_xor(D, p0 + 4)) * (D / 8), v1);
      load_words<D>(vb + q4::code_bytes(D) + p0 * (J * 4), s0);
      load_words<D>(vb + q4::code_bytes(D) + (p0 + 4) * (J * 4), s1);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          w[h] = exp2_fast(CAP ? s[blk][n][h] + base[n][h & 1] : fmaf(s[blk][n][h], mul[n][h & 1], base[n][h & 1]));
          l[n][h & 1] += w[h];
        }
        b0[n] = q4::transpose8(q4::pack_f16x2(w[0], w[1]));
        b1[n] = q4::transpose8(q4::pack_f16x2(w[2], w[3]));
        if constexpr (!whole) {  // what a column does not see has no part in it, whatever its bytes say
          const int hi = last_of(n * 8 + g), lo = first_of(hi);
          auto seen = [&](int at) { return (at >= lo && at <= hi ? 0xffffu : 0u) | (at + 1 >= lo && at + 1 <= hi ? 0xffff0000u : 0u); };
          see0[n] = seen(pos + 2 * p0);
          see1[n] = seen(pos + 2 * p0 + 8);
        }
      }
#pragma unroll
      for (int j = 0; j < J; ++j) {
        uint32_t a0[4], a1[4];
        q4::codes_f16(v0[j], a0);
        q4::codes_f16(v1[j], a1);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          uint32_t w0 = q4::hmul2(b0[n], s0[j]), w1 = q4::hmul2(b1[n], s1[j]);
          if constexpr (!whole) {
            w0 &= see0[n];
            w1 &= see1[n];
          }
          q4::mma_f16(o[j][0][n], a0[0], a0[1], a1[0], a1[1], w0, w1);
          q4::mma_f16(o[j][1][n], a0[2], a0[3], a1[2], a1[3], w0, w1);
        }
      }
    }
  };
  for (; i < n_mine; ++i) {
    const int pos = (p_begin + warp + kWarps * i) * PAGE;
    copy_wait<2>();
    __syncwarp();
    if (id < 0) fetch(a.v_cache, id_next, slot);  // none of it is seen
    else if (pos >= all_lo && pos + PAGE - 1 <= all_hi) page(pos, std::true_type{});
    else page(pos, std::false_type{});
    __syncwarp();  // V's slot is free: the K of the page after next
    id = id_next;
    id_next = number_of(i + 2);
    fetch(a.k_cache, id_next, slot == SLOTS - 1 ? 0 : slot + 1);
    slot = slot == 0 ? SLOTS - 1 : slot - 1;  // two on
  }
  copy_wait<0>();
  bool wide_range = false;
#pragma unroll
  for (int j = 0; j < J; ++j) wide_range |= out_of_range(low[j / 2], j, ex[j], kRange);
  if (__syncthreads_or(wide_range)) {
    share_in_fp32<D, CAP>(a, ct, C::COLS, blockIdx.x);
    return;
  }

  // the four warps meet
  float* sm = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float* dst = sm + (warp * C::COLS + n * 8 + 2 * t + i) * (D + 4);
      float sum = l[n][i];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float back = __uint_as_float((uint32_t)(ex[j] - 4) << 23);  // 2^(ex - 131)
        *reinterpret_cast<float4*>(dst + 32 * j + 4 * g) = make_float4(o[j][0][n][i] * back, o[j][0][n][i + 2] * back, o[j][1][n][i] * back, o[j][1][n][i + 2] * back);
      }
      if (g == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(m[n][i], sum);
    }
  __syncthreads();
  for (int i = threadIdx.x; i < tile.cols * (D / 4); i += kThreads) {
    const int c = i / (D / 4), d = i % (D / 4) * 4;
    const int r = row_of(c), row = tile.row0 + r, head = kvh * G + tile.rest + c - r * G;
    const bool done = shares == 1;
    float2 ml[kWarps];
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      ml[w] = *reinterpret_cast<const float2*>(sm + (w * C::COLS + c) * (D + 4) + D);
      mt = fmaxf(mt, ml[w].x);
    }
    const float sink = done && a.sink ? __bfloat162float(a.sink[head]) * kLog2e : -INFINITY;
    const float top = fmaxf(mt, sink), ref = top == -INFINITY ? 0.f : top;
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = exp2_fast(sink - ref);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(sm + (w * C::COLS + c) * (D + 4) + d);
      const float f = exp2_fast(ml[w].x - ref - 10.f);  // (sums are 2^10 times what they stand for)
      acc = make_float4(fmaf(x.x, f, acc.x), fmaf(x.y, f, acc.y), fmaf(x.z, f, acc.z), fmaf(x.w, f, acc.w));
      sum = fmaf(ml[w].y, f, sum);
    }
    if (done) {
      store4(a.out + (size_t)row * a.ldo + (size_t)head * D + d, acc, sum);
    } else {
      float* dst = a.workspace + (((size_t)row * a.Hq + head) * a.max_splits + blockIdx.x) * (D + 4);
      *reinterpret_cast<float4*>(dst + d) = acc;
      if (d == 0) *reinterpret_cast<float2*>(dst + D) = make_float2(mt, sum);
    }
  }
}

// Portions.  A block has 128 columns, and every page of its share is widened once for all of them: codes times scales, exact in fp16 (a code has 3 bits
// beside its sign, a bf16 scale 8), into shared memory, where the tensor cores take them from.  S[128 columns x 64 positions] = Q K^T and
// O[128 columns x D] += P V, with S, P (over S) and O in tensor memory; P is fp16 by one rounding of at most 2^-11.
//   warps 0-3   a column per lane: scores, running maximum, weights; O is scaled by them where a maximum has moved far or a value scale has
//   warps 4-7   a page's words from global memory to registers to shared memory, one page ahead of the columns
// S of a page whose keys are there is issued by warps 4 to 6 in turn, the products with V by warp 7 (an issuing lane is held up for as long as the products
// before it take, and the columns' warps have the longest way as it is).
//   K: [position][entry], scaled by a power of two per position that the scores take back (largest scale in [2^11, 2^12); scales below 2^-25 of a position's
//      largest lose bits).
//   V: [entry][position], as pairs of positions lie together in the words; its power of two is per group and follows its largest finite scale so far (a
//      share with scales below 2^-25 of it: share_in_fp32).
// Both are rows of 128 bytes with 16-byte chunks at the places that the 128-byte swizzle gives them; every store of eight lanes meets all banks.
// Measured (32 query heads over 8 kv heads of 128 entries), with the kernel above beside it: 512 rows behind 3584 positions 97 us (206), a prompt of 2048 rows
// 125 (252), 128 rows of four sequences of 4096 99 (182), 64 rows of one of 8192 39 (56), but of 16 sequences of 1024 47 (38); 32 rows, 128 columns, of four
// of 4096 37 (36).
// No unit is busy half of its time: a page takes 1100 issue slots per SM quarter, the chain scores - weights - V - scores of the page after next some
// 2600 cycles with two blocks per SM.  Sixteen columns per warp from one widened page with the warp-wide products took 197 us for the 512 rows.
template <int D>
struct Wide {
  static constexpr int COLS = kWideCols;
  static constexpr int THREADS = 256;
  static constexpr int BLOCK = q4::block_bytes(D);
  static constexpr int Q_BYTES = COLS * D * 2, HALF = PAGE * D * 2;  // widened K or V
  static constexpr int J = D / q4::kGroup;
  static constexpr int RANGE = 25;  // as kRange: the widened values alone are fp16 here, below 2^15, and a code times a scale has 11 bits
  struct Page {  // what a widened page is besides
    float factor[PAGE];
    float less[4];  // the groups' factors for O so far
    int ex[4];
    int id, grow, bad;
  };
  static constexpr int KEYS = Q_BYTES, VALUES = KEYS + 2 * HALF, PAGES = VALUES + 2 * HALF, PAIRS = PAGES + 4 * 512, BARS = PAIRS + 4 * PAGE / 2 * J * 4,
                       MULS = BARS + 128, END = MULS + COLS * 4;
  static constexpr int SMEM = (END > 80 * 1024 ? END : 80 * 1024) + 1024;  // (two blocks per SM: tensor memory has room for no more)
  static_assert(sizeof(Page) <= 512 && COLS * (D + 4) * 4 <= PAGES);  // (the sums leave through the room of Q and the widened pages)
};
// Set by a block that gave up a wait: attn_q4_status.  Its rows are NaN, its products in flight are waited for before their operands' room and its columns are given back.
__device__ unsigned wait_ran_out;
// False where the barrier has not turned after so many cycles (below 0: it is not looked at)
__device__ __forceinline__ bool wait_turn(uint64_t* bar, uint32_t parity, long long cycles) {
  bool ok = cycles >= 0 && mbar_try_wait(bar, parity);
  if (!ok && cycles > 0) {
    const long long t0 = clock64();
    while (!(ok = mbar_try_wait(bar, parity)) && clock64() - t0 < cycles) {
    }
  }
  return __all_sync(0xffffffffu, ok);
}

template <int D, bool CAP>
__global__ void __launch_bounds__(Wide<D>::THREADS, 2) attn_q4_wide_kernel(const __grid_constant__ AttnQ4Args a) {
  using C = Wide<D>;
  constexpr int J = C::J;
  extern __shared__ uint8_t smem_raw[];
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int G = a.group;
  const int b = blockIdx.z, ct = a.tile0 + blockIdx.y / a.Hkv, kvh = blockIdx.y % a.Hkv;
  const Tile tile = tile_of(a, b, ct, C::COLS);
  if (tile.cols <= 0) return;
  auto row_of = [&](int c) { return div_g(a, tile.rest + c); };
  const int shares = tile.splits;
  if (tile.pages == 0) {
    if (blockIdx.x == 0) zero_columns<D>(a, tile, kvh);
    return;
  }
  if ((int)blockIdx.x >= shares) return;
  const int p_begin = tile.page0 + (int)((long long)tile.pages * blockIdx.x / shares);
  const int n_pages = tile.page0 + (int)((long long)tile.pages * (blockIdx.x + 1) / shares) - p_begin;

  uint8_t* smem = smem_raw + (-smem_u32(smem_raw) & 1023);
  auto info_of = [&](int i) { return reinterpret_cast<typename C::Page*>(smem + C::PAGES + (i & 3) * 512); };  // (read till P is there, written when S two pages before is)
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::BARS);
  // keys there (page i: i & 3), values, scores, weights there, page done with (i & 1)
  uint64_t *k_full = bars, *v_full = bars + 4, *s_full = bars + 6, *p_full = bars + 8, *pv_done = bars + 10;
  uint64_t* all_done = bars + 12;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(bars + 13);
  if (threadIdx.x == 128) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&k_full[i], 4);
      mbar_init(&k_full[i + 2], 4);
      mbar_init(&v_full[i], 4);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(all_done, 4);
    fence_barrier_init();
  }
  if (warp == 7) {
    tmem_alloc(tmem_ptr, 256);
    tmem_relinquish();
  }
  const int all_hi = tile.pos0, all_lo = a.window > 0 ? tile.pos0 + row_of(tile.cols - 1) - a.window + 1 : 0;
  auto whole_at = [&](int pos) { return pos >= all_lo && pos + PAGE - 1 <= all_hi; };  // every column sees all of the page at pos
  float* muls = reinterpret_cast<float*>(smem + C::MULS);  // what brings a column's sums to log2 of its weights (to scores, where they are capped)
  {  // q: a column's row as fp16, its largest entry in [2^10, 2^11)
    constexpr int PER_ROW = D / 8, AT_ONCE = 32 / PER_ROW;
    const int x = lane % PER_ROW;
    const uint32_t sign = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll 4
    for (int c = warp * 16 + lane / PER_ROW; c < warp * 16 + 16; c += AT_ONCE) {
      uint4 w = make_uint4(0, 0, 0, 0);
      if (c < tile.cols) {
        const int r = row_of(c);
        w = *reinterpret_cast<const uint4*>(a.q + (size_t)(tile.row0 + r) * a.ldq + (size_t)(kvh * G + tile.rest + c - r * G) * D + 8 * x);
      }
      uint32_t mag = max(max(finite_top(w.x), finite_top(w.y)), max(finite_top(w.z), finite_top(w.w)));
#pragma unroll
      for (int y = 1; y < PER_ROW; y <<= 1) mag = max(mag, __shfl_xor_sync(0xffffffffu, mag, y));
      const int e = max((int)(mag >> 7), 20);
      const float up = __uint_as_float((uint32_t)(264 - e) << 23), down = __uint_as_float((uint32_t)(e - 10) << 23);
      w.x = q4::pack_f16x2(q4::bf16_lo(w.x) * up, q4::bf16_hi(w.x) * up) ^ sign;
      w.y = q4::pack_f16x2(q4::bf16_lo(w.y) * up, q4::bf16_hi(w.y) * up) ^ sign;
      w.z = q4::pack_f16x2(q4::bf16_lo(w.z) * up, q4::bf16_hi(w.z) * up) ^ sign;
      w.w = q4::pack_f16x2(q4::bf16_lo(w.w) * up, q4::bf16_hi(w.w) * up) ^ sign;
      *reinterpret_cast<uint4*>(smem + (x >> 3) * (C::COLS * 128) + c * 128 + (((x & 7) ^ (c & 7)) << 4)) = w;
      if (x == 0) muls[c] = fmaxf(down * (CAP ? fabsf(a.scale) : fabsf(a.scale) * kLog2e), 1e-37f);
    }
    fence_proxy_async_smem();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  pdl_launch_dependents();  // (its columns are held: launch.h)
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_ptr, 0), tmem_o = tmem + 2 * PAGE;  // columns: two pages of S, then O
  constexpr uint32_t f16 = ~((1u << 7) | (1u << 10));  // (the descriptors' types)
  constexpr uint32_t idesc_s = umma_idesc_bf16(C::COLS, PAGE) & f16, idesc_o = umma_idesc_bf16(C::COLS, D) & f16;
  const bool leader = elect_one_sync();
  bool ok = true, wide_range = false;
  float m = -INFINITY, l = 0.f;
  const uint32_t tmem_row = (uint32_t)(warp & 3) << 21;  // the warp's 32 lanes

  if (warp < 4) {
    const int c = threadIdx.x;
    const float mul = muls[c];
    const int last = c < tile.cols ? tile.pos0 + row_of(c) : -1, first = a.window > 0 ? last - a.window + 1 : 0;
    for (int i = 0; i < n_pages; ++i) {
      const int st = i & 1, ph = (i >> 1) & 1, pos = (p_begin + i) * PAGE;
      if (!(ok = wait_turn(&k_full[i & 3], (i >> 2) & 1, a.wait_cycles) && wait_turn(&s_full[st], ph, a.wait_cycles))) break;
      tc_fence_after();
      const typename C::Page& pg = *info_of(i);
      float s[PAGE];
      {
        uint32_t(&lo)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[0]);
        uint32_t(&hi)[32] = *reinterpret_cast<uint32_t(*)[32]>(&s[32]);
        tmem_ld_32x32b_x32(tmem + tmem_row + st * PAGE, lo);
        tmem_ld_32x32b_x32(tmem + tmem_row + st * PAGE + 32, hi);
        tmem_ld_wait();
      }
#pragma unroll
      for (int x = 0; x < PAGE; x += 4) {
        const float4 f = *reinterpret_cast<const float4*>(&pg.factor[x]);
        f2_unpack(f2_mul(f2_pack(s[x], s[x + 1]), f2_pack(f.x, f.y)), s[x], s[x + 1]);
        f2_unpack(f2_mul(f2_pack(s[x + 2], s[x + 3]), f2_pack(f.z, f.w)), s[x + 2], s[x + 3]);
      }
      if constexpr (CAP) {
        const Cap cap(a.softcap);
        if (a.softcap <= kCapByExp) {
#pragma unroll
          for (int x = 0; x < PAGE; ++x) s[x] = cap.by_exp(s[x] * mul);
        } else {
#pragma unroll
          for (int x = 0; x < PAGE; ++x) s[x] = capped_far(s[x] * mul, a.softcap);
        }
      }
      if (pg.id < 0 || !whole_at(pos)) {
        const int hi = pg.id < 0 ? -1 : last - pos, lo = first - pos;
#pragma unroll
        for (int x = 0; x < PAGE; ++x)
          if (x > hi || x < lo) s[x] = -INFINITY;
      }
      float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int x = 4; x < PAGE; ++x) top[x & 3] = fmaxf(top[x & 3], s[x]);
      float x = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
      if constexpr (!CAP) x *= mul;
      // weights up to 2^15 fit fp16, so what they are relative to moves seldom
      const bool moved = x > m + 5.f;
      if (__any_sync(0xffffffffu, moved) || pg.grow) {
        x = fmaxf(m, x);
        const float f = m == x ? 1.f : exp2_fast(m - x);  // (-inf before: 0)
        m = x;
        l *= f;
        if (i > 0) {
          if (!(ok = wait_turn(&pv_done[st ^ 1], ((i - 1) >> 1) & 1, a.wait_cycles))) break;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const float by = f * pg.less[j];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint32_t o[16];
              tmem_ld_32x32b_x16(tmem_o + tmem_row + 32 * j + 16 * h, o);
              tmem_ld_wait();
#pragma unroll
              for (int y = 0; y < 16; ++y) o[y] = __float_as_uint(__uint_as_float(o[y]) * by);
              tmem_st_32x32b_x16(tmem_o + tmem_row + 32 * j + 16 * h, o);
            }
          }
        }
      }
      const float base = 10.f - (m == -INFINITY ? 0.f : m);
      uint64_t sums[2] = {0, 0};
#pragma unroll
      for (int y = 0; y < PAGE; y += 32) {
        uint32_t w[16];
#pragma unroll
        for (int z = 0; z < 16; ++z) {
          float p0 = s[y + 2 * z] + base, p1 = s[y + 2 * z + 1] + base;
          if constexpr (!CAP) f2_unpack(f2_fma(f2_pack(s[y + 2 * z], s[y + 2 * z + 1]), f2_pack(mul, mul), f2_pack(base, base)), p0, p1);
          p0 = exp2_fast(p0);
          p1 = exp2_fast(p1);
          sums[z & 1] = f2_add(sums[z & 1], f2_pack(p0, p1));
          w[z] = q4::pack_f16x2(p0, p1);
        }
        tmem_st_32x32b_x16(tmem + tmem_row + st * PAGE + y / 2, w);
      }
      {
        float x0, x1;
        f2_unpack(f2_add(sums[0], sums[1]), x0, x1);
        l += x0 + x1;
      }
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_full[st]);
      if (pg.bad) {  // infinities and NaN among value scales that not every column sees were widened as 0: for the columns that do, after the products
        if (!(ok = wait_turn(&pv_done[st], ph, a.wait_cycles))) break;
        tc_fence_after();
        const uint8_t* vb = a.v_cache + ((size_t)pg.id * a.Hkv + kvh) * C::BLOCK;
        for (int j = 0; j < J; ++j)
          for (int h = 0; h < 2; ++h) {
            uint32_t o[16];
            tmem_ld_32x32b_x16(tmem_o + tmem_row + 32 * j + 16 * h, o);
            tmem_ld_wait();
            for (int p = max(first - pos, 0); p <= min(last - pos, PAGE - 1); ++p) {
              const uint32_t d = *reinterpret_cast<const uint16_t*>(vb + q4::code_bytes(D) + (p * J + j) * 2);
              if ((d & 0x7fffu) < 0x7f80u) continue;
#pragma unroll
              for (int y = 0; y < 16; ++y) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(vb + (p >> 1) * D + ((4 * h + (y >> 2)) ^ q4::place_xor(D, p >> 1)) * (D / 8) + 4 * j);
                const int code = w >> (4 * (y & 3) + 16 * (p & 1)) & 15;
                o[y] = __float_as_uint(__uint_as_float(o[y]) + __uint_as_float(d << 16) * (float)(code - 8));
              }
            }
            __syncwarp();
            tmem_st_32x32b_x16(tmem_o + tmem_row + 32 * j + 16 * h, o);
          }
        tmem_st_wait();
        tc_fence_before();  // (the next weights say that O may be added to)
      }
    }
    if (ok) ok = wait_turn(&pv_done[(n_pages - 1) & 1], ((n_pages - 1) >> 1) & 1, a.wait_cycles);
  } else {
    const int id_x = threadIdx.x - 128;
    const int32_t* table = a.page_table + (size_t)b * a.max_pages + p_begin;
    uint32_t* pairs = reinterpret_cast<uint32_t*>(smem + C::PAIRS) + (warp - 4) * (PAGE / 2 * J);
    int ids = -1;  // lane i % 32 holds the number of page i, -1 for one that is none
    auto number_of = [&](int i) {
      if ((i & 31) == 0) {
        ids = -1;
        if (i + lane < n_pages) {
          const int id = table[i + lane];
          if (id >= 0 && id < a.num_pages) ids = id;
        }
      }
      const int id = __shfl_sync(0xffffffffu, ids, i & 31);
      return i < n_pages ? id : -1;
    };
    // keys: quarter u of rows p and p + 32; values: half a chunk of four pairs
    const int l8 = lane >> 2, u = lane & 3, p = (warp - 4) * 8 + ((l8 & 1) << 2 | l8 >> 1);
    const int p8 = lane & 7, chunk = id_x >> 4, half = (id_x >> 3) & 1;
    constexpr int W = J / 2;
    uint32_t kw[2][J], ks[2][W], vw[4][W], vs[J];  // (of a page that is none: page 0's, not used)
    auto load_keys = [&](int id) {
      const uint8_t* kb = a.k_cache + ((size_t)max(id, 0) * a.Hkv + kvh) * C::BLOCK;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        load_words<D>(kb + (p + 32 * h) * (D / 2) + u * (D / 8), kw[h]);
        load_words<D / 2>(kb + q4::code_bytes(D) + (p + 32 * h) * J * 2, ks[h]);
      }
    };
    auto load_values = [&](int id) {
      const uint8_t* vb = a.v_cache + ((size_t)max(id, 0) * a.Hkv + kvh) * C::BLOCK;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int n = 4 * p8 + k;
        load_words<D / 2>(vb + n * D + (chunk ^ q4::place_xor(D, n)) * (D / 8) + half * (D / 16), vw[k]);
      }
      load_words<D>(vb + q4::code_bytes(D) + lane * (J * 4), vs);
    };
    int ex[J];
    uint32_t low[W];
#pragma unroll
    for (int j = 0; j < J; ++j) {
      ex[j] = 12;
      low[j / 2] = kNoScale;
    }
    auto add_values = [&](int i) {  // O += P V of page i
      const int st = i & 1, ph = (i >> 1) & 1;
      if (!wait_turn(&p_full[st], ph, a.wait_cycles) || !wait_turn(&v_full[st], ph, a.wait_cycles)) return false;
      tc_fence_after();
      if (leader) {
        const uint64_t vd = umma_desc_kmajor_sw128(smem_u32(smem + C::VALUES + st * C::HALF));
#pragma unroll
        for (int k = 0; k < PAGE / 16; ++k) umma_f16_ts(tmem_o, tmem + st * PAGE + k * 8, vd + (k * 32 >> 4), idesc_o, i > 0 || k != 0);
        umma_commit(&pv_done[st]);
      }
      __syncwarp();
      return true;
    };
    int id = number_of(0);
    load_keys(id);
    load_values(id);
    for (int i = 0; i < n_pages; ++i) {
      const int st = i & 1, pos = (p_begin + i) * PAGE;
      const bool whole = whole_at(pos);
      const int id_next = number_of(i + 1);
      if (i >= 2 && !(ok = wait_turn(&s_full[st], ((i - 2) >> 1) & 1, a.wait_cycles))) break;
      typename C::Page& pg = *info_of(i);
      uint8_t* keys = smem + C::KEYS + st * C::HALF;
      uint8_t* values = smem + C::VALUES + st * C::HALF;
      if (id < 0) {  // no column sees it, and whatever the weights' zeros are multiplied with is finite
#pragma unroll
        for (int j = 0; j < J; ++j) vs[j] = 0;
      }
      bool bad = false, grow = false;
      float less[J];
#pragma unroll
      for (int j = 0; j < J; ++j) less[j] = 1.f;
      {  // a lane takes the scales of positions 2 lane and 2 lane + 1
        const int at = pos + 2 * lane;
        uint32_t x[W], y[W];
#pragma unroll
        for (int k = 0; k < W; ++k) {
          if (!whole && !(at >= tile.lo && at < tile.hi)) vs[k] = 0;
          if (!whole && !(at + 1 >= tile.lo && at + 1 < tile.hi)) vs[W + k] = 0;
          x[k] = vs[k] & 0x7fff7fffu;
          y[k] = vs[W + k] & 0x7fff7fffu;
          const uint32_t fits = (uint32_t)(ex[2 * k] << 7 | ex[2 * k + 1] << 23) | 0x007f007fu;  // the largest numbers of the present exponents
          grow |= __vmaxu2(__vmaxu2(x[k], y[k]), fits) != fits;
          low[k] = smallest_scale(low[k], x[k], y[k]);
        }
        grow = __any_sync(0xffffffffu, grow);
        if (grow) {
          bool odd = false;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const uint32_t v0 = j & 1 ? x[j / 2] >> 16 : x[j / 2] & 0xffffu, v1 = j & 1 ? y[j / 2] >> 16 : y[j / 2] & 0xffffu;
            odd |= max(v0, v1) >= 0x7f80u;
            if (!whole && v0 >= 0x7f80u) vs[j / 2] &= j & 1 ? 0xffffu : 0xffff0000u;
            if (!whole && v1 >= 0x7f80u) vs[W + j / 2] &= j & 1 ? 0xffffu : 0xffff0000u;
            const int e = max((int)(__reduce_max_sync(0xffffffffu, max(v0 < 0x7f80u ? v0 : 0u, v1 < 0x7f80u ? v1 : 0u)) >> 7), ex[j]);
            less[j] = exp2f((float)(ex[j] - e));
            ex[j] = e;
          }
          bad = __any_sync(0xffffffffu, odd && !whole);
        }
        uint32_t w[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const float near1 = __uint_as_float((uint32_t)(265 - ex[j]) << 23);
          const uint32_t v0 = vs[j / 2], v1 = vs[W + j / 2];
          w[j] = q4::pack_f16x2((j & 1 ? q4::bf16_hi(v0) : q4::bf16_lo(v0)) * near1, (j & 1 ? q4::bf16_hi(v1) : q4::bf16_lo(v1)) * near1);
        }
        __syncwarp();
        if constexpr (J == 4) *reinterpret_cast<uint4*>(pairs + lane * J) = make_uint4(w[0], w[1], w[2], w[3]);
        else *reinterpret_cast<uint2*>(pairs + lane * J) = make_uint2(w[0], w[1]);
        __syncwarp();
      }
      if (id_x == 0) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          pg.less[j] = less[j];
          pg.ex[j] = ex[j];
        }
        pg.id = id;
        pg.grow = grow;
        pg.bad = bad;
      }
      if (id >= 0) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int r = p + 32 * h;
          float d[J];
          uint32_t mag = 0;
#pragma unroll
          for (int j = 0; j < J; ++j) {
            d[j] = j & 1 ? q4::bf16_hi(ks[h][j / 2]) : q4::bf16_lo(ks[h][j / 2]);
            if (j & 1) mag = max(mag, finite_top(ks[h][j / 2]));
          }
          const int e = max((int)(mag >> 7), 12);
          const float near1 = __uint_as_float((uint32_t)(265 - e) << 23);  // 2^(138 - e)
          if (u == 0) pg.factor[r] = __uint_as_float((uint32_t)(e - 11) << 23);
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const uint32_t sc = q4::pack_f16x2(d[j] * near1, d[j] * near1);
            uint32_t x[4];
            q4::codes_f16(kw[h][j], x);
            *reinterpret_cast<uint4*>(keys + (j >> 1) * (PAGE * 128) + r * 128 + (((4 * (j & 1) + u) ^ (r & 7)) << 4)) =
                make_uint4(q4::hmul2(x[0], sc), q4::hmul2(x[1], sc), q4::hmul2(x[2], sc), q4::hmul2(x[3], sc));
          }
        }
      }
      load_keys(id_next);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&k_full[i & 3]);
      if (i >= 2 && warp == 7 && !(ok = add_values(i - 2))) break;
      if (i >= 2 && !(ok = wait_turn(&pv_done[st], ((i - 2) >> 1) & 1, a.wait_cycles))) break;
      if (warp == 4 + i % 3) {
        if (!(ok = wait_turn(&k_full[i & 3], (i >> 2) & 1, a.wait_cycles))) break;
        tc_fence_after();
        if (leader) {
          const uint64_t qd = umma_desc_kmajor_sw128(smem_u32(smem)), kd = umma_desc_kmajor_sw128(smem_u32(keys));
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            umma_f16_ss(tmem + st * PAGE, qd + (((k >> 2) * (C::COLS * 128) + (k & 3) * 32) >> 4), kd + (((k >> 2) * (PAGE * 128) + (k & 3) * 32) >> 4), idesc_s, k != 0);
          umma_commit(&s_full[st]);
        }
        __syncwarp();
      }
#pragma unroll
      for (int j = 0; j < W; ++j) {
        uint32_t x[4][4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          q4::codes_f16(vw[k][j], x[k]);
          const uint32_t sc = pairs[(4 * p8 + k) * J + half * W + j];
#pragma unroll
          for (int y = 0; y < 4; ++y) x[k][y] = q4::hmul2(x[k][y], sc);
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const int entry = 32 * (half * W + j) + 4 * chunk + y;
          *reinterpret_cast<uint4*>(values + entry * 128 + ((p8 ^ (entry & 7)) << 4)) = make_uint4(x[0][y], x[1][y], x[2][y], x[3][y]);
        }
      }
      load_values(id_next);
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&v_full[st]);
      id = id_next;
    }
    for (int i = max(n_pages - 2, 0); i < n_pages && ok && warp == 7; ++i) ok = add_values(i);
#pragma unroll
    for (int j = 0; j < J; ++j) wide_range |= out_of_range(low[j / 2], j, ex[j], C::RANGE);
  }
  tc_fence_before();
  if (__syncthreads_or(!ok)) {
    if (warp >= 4 && leader) umma_commit(all_done);  // (turns when all that these four lanes have issued is done)
    __syncwarp();
    wait_turn(all_done, 0, HB_WAIT_TIMEOUT_CYCLES);
    tc_fence_after();
    const float nan = __uint_as_float(0x7fffffffu);
    for (int i = threadIdx.x; i < tile.cols * (D + 2); i += C::THREADS) {
      const int c = i / (D + 2), d = i % (D + 2), r = row_of(c), row = tile.row0 + r, head = kvh * G + tile.rest + c - r * G;
      if (shares > 1) a.workspace[(((size_t)row * a.Hq + head) * a.max_splits + blockIdx.x) * (D + 4) + d] = nan;
      else if (d < D) a.out[(size_t)row * a.ldo + (size_t)head * D + d] = __float2bfloat16(nan);
    }
    if (threadIdx.x == 0) wait_ran_out = 1;
    tc_fence_before();
    __syncthreads();
    if (warp == 7) {
      tc_fence_after();
      tmem_dealloc(tmem, 256);
    }
    return;
  }
  if (__syncthreads_or(wide_range)) {
    tc_fence_after();
    if (warp == 7) tmem_dealloc(tmem, 256);
    share_in_fp32<D, CAP>(a, ct, C::COLS, blockIdx.x);
    return;
  }
  tc_fence_after();
  float* sums = reinterpret_cast<float*>(smem);  // [column]: D sums, maximum, sum of weights, and 8 bytes that keep the rows aligned
  const bool done = shares == 1;
  if (warp < 4) {
    const int c = threadIdx.x, r = row_of(c);
    const float sink = done && a.sink && c < tile.cols ? __bfloat162float(a.sink[kvh * G + tile.rest + c - r * G]) * kLog2e : -INFINITY;
    const float top = fmaxf(m, sink), ref = top == -INFINITY ? 0.f : top;
    const float f = exp2_fast(m - ref - 10.f);  // (sums are 2^10 times what they stand for)
#pragma unroll
    for (int j = 0; j < 2 * J; ++j) {
      uint32_t o[16];
      tmem_ld_32x32b_x16(tmem_o + tmem_row + 16 * j, o);
      tmem_ld_wait();
      const float back = __uint_as_float((uint32_t)(info_of(n_pages - 1)->ex[j / 2] - 11) << 23);  // 2^(ex - 138)
      float x[16];
#pragma unroll
      for (int y = 0; y < 16; ++y) x[y] = __uint_as_float(o[y]) * back * f;
#pragma unroll
      for (int y = 0; y < 16; y += 4) *reinterpret_cast<float4*>(sums + c * (D + 4) + 16 * j + y) = make_float4(x[y], x[y + 1], x[y + 2], x[y + 3]);
    }
    *reinterpret_cast<float2*>(sums + c * (D + 4) + D) = make_float2(m, fmaf(l, f, exp2_fast(sink - ref)));
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tile.cols * (D / 4); i += C::THREADS) {
    const int c = i / (D / 4), d = i % (D / 4) * 4, r = row_of(c), row = tile.row0 + r, head = kvh * G + tile.rest + c - r * G;
    const float4 x = *reinterpret_cast<const float4*>(sums + c * (D + 4) + d);
    const float2 ml = *reinterpret_cast<const float2*>(sums + c * (D + 4) + D);
    if (done) {
      store4(a.out + (size_t)row * a.ldo + (size_t)head * D + d, x, ml.y);
    } else {
      float* part = a.workspace + (((size_t)row * a.Hq + head) * a.max_splits + blockIdx.x) * (D + 4);
      *reinterpret_cast<float4*>(part + d) = x;
      if (d == 0) *reinterpret_cast<float2*>(part + D) = ml;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 7) {
    tc_fence_after();
    tmem_dealloc(tmem, 256);
  }
}

// What more than one block has worked on is joined: four sums of every fourth share each, then these, in order.  PER = 4 warps to a (row, head) take one each;
// where there are many (row, head)s one warp takes all four, with the same bits (512 rows of 32 heads in two shares: the call takes 97 us with one, 116 with four;
// eight sequences of 2k with 32 heads, eight shares: 10.2 with four, 11.9 with one).
template <int D, int PER>
__global__ void __launch_bounds__(kThreads) attn_q4_join_kernel(const AttnQ4Args a, int cols_per_tile) {
  constexpr int V = D / 32, SUMS = 4;
  __shared__ float s_part[SUMS][D + 2];
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int at = blockIdx.x * (kWarps / PER) + warp / PER, i = at / a.Hq, head = at - i * a.Hq;
  // (lengths are settled: the blocks of the kernel before let this one start only once they had waited for the kernels ahead of them)
  const int ct = (i * a.group + head % a.group) / cols_per_tile;
  const Tile tile = tile_of(a, b, ct, cols_per_tile);
  const int c = i * a.group + head % a.group - ct * cols_per_tile;
  const int shares = tile.splits, row = tile.row0 + div_g(a, tile.rest + c);
  const float* src = a.workspace + ((size_t)row * a.Hq + head) * a.max_splits * (D + 4);
  pdl_wait();
  pdl_launch_dependents();
  if (c >= tile.cols || shares <= 1) return;
  const float sink = a.sink ? __bfloat162float(a.sink[head]) * kLog2e : -INFINITY;
  struct Sum {
    float m, sum, acc[V];
  };
  auto sum_of = [&](int first) {  // up to eight of the shares at a time
    Sum r = {-INFINITY, 0.f, {}};
    for (int s0 = first; s0 < shares; s0 += 8 * SUMS) {
      float x[8][V];
      float2 ml[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        ml[k] = make_float2(-INFINITY, 0.f);
        if (s0 + k * SUMS < shares) {
          const float* p = src + (size_t)(s0 + k * SUMS) * (D + 4);
          ml[k] = *reinterpret_cast<const float2*>(p + D);
#pragma unroll
          for (int v = 0; v < V; ++v) x[k][v] = p[lane + 32 * v];
        } else {
#pragma unroll
          for (int v = 0; v < V; ++v) x[k][v] = 0.f;
        }
      }
      float top = r.m;
#pragma unroll
      for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
      const float ref = top == -INFINITY ? 0.f : top, old = exp2_fast(r.m - ref);
      r.m = top;
      r.sum = __fmul_rn(r.sum, old);
#pragma unroll
      for (int v = 0; v < V; ++v) r.acc[v] = __fmul_rn(r.acc[v], old);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const float f = exp2_fast(ml[k].x - ref);
        r.sum = fmaf(ml[k].y, f, r.sum);
#pragma unroll
        for (int v = 0; v < V; ++v) r.acc[v] = fmaf(x[k][v], f, r.acc[v]);
      }
    }
    return r;
  };
  bf16* out = a.out + (size_t)row * a.ldo + (size_t)head * D;
  if constexpr (PER == 1) {
    Sum part[SUMS];
    if (shares <= SUMS) {  // (one each: all loads at once)
#pragma unroll
      for (int w = 0; w < SUMS; ++w) {
        part[w] = Sum{-INFINITY, 0.f, {}};
        if (w < shares) {
          const float* p = src + (size_t)w * (D + 4);
          part[w].m = p[D];
          part[w].sum = p[D + 1];
#pragma unroll
          for (int v = 0; v < V; ++v) part[w].acc[v] = p[lane + 32 * v];
        }
      }
    } else {
#pragma unroll
      for (int w = 0; w < SUMS; ++w) part[w] = sum_of(w);
    }
    float top = sink;
#pragma unroll
    for (int w = 0; w < SUMS; ++w) top = fmaxf(top, part[w].m);
    const float ref = top == -INFINITY ? 0.f : top;
    float y[V] = {}, all = exp2_fast(sink - ref);
#pragma unroll
    for (int w = 0; w < SUMS; ++w) {
      const float f = exp2_fast(part[w].m - ref);
      all = fmaf(part[w].sum, f, all);
#pragma unroll
      for (int v = 0; v < V; ++v) y[v] = fmaf(part[w].acc[v], f, y[v]);
    }
#pragma unroll
    for (int v = 0; v < V; ++v) out[lane + 32 * v] = __float2bfloat16(all == 0.f ? 0.f : y[v] / all);
  } else {
    const Sum part = sum_of(warp);
#pragma unroll
    for (int v = 0; v < V; ++v) s_part[warp][lane + 32 * v] = part.acc[v];
    if (lane == 0) {
      s_part[warp][D] = part.m;
      s_part[warp][D + 1] = part.sum;
    }
    __syncthreads();
    if (threadIdx.x < D) {
      float top = sink;
#pragma unroll
      for (int w = 0; w < SUMS; ++w) top = fmaxf(top, s_part[w][D]);
      const float ref = top == -INFINITY ? 0.f : top;
      float y = 0.f, all = exp2_fast(sink - ref);
#pragma unroll
      for (int w = 0; w < SUMS; ++w) {
        const float f = exp2_fast(s_part[w][D] - ref);
        y = fmaf(s_part[w][threadIdx.x], f, y);
        all = fmaf(s_part[w][D + 1], f, all);
      }
      out[threadIdx.x] = __float2bfloat16(all == 0.f ? 0.f : y / all);
    }
  }
}

constexpr int kMostGridY = 65535;
struct Plan {
  int split_pages, max_splits, tiles, cols;
};
// By the rule (split_pages 0) a tile's pages are cut into so many shares that there are some 1.67 blocks per SM, and that none has more than 32 pages,
// or 40 where all blocks are resident at once, four to an SM (with 16 columns per tile a page takes twice as long: 16, or 32 where the tiles alone are more
// than four to an SM); a share is a page per warp at least.  Both sides, us: one sequence of 2k 6.4 in shares of 4 pages, 15.1 whole; 8 of 2k 10.0 in 8, 15.8 whole; 32 of 1.5k to 2.2k 24.9
// in 36, 29.9 in 24; 32 of 8k 66.2 in 32, 67.2 in 40, 73.1 in 48; three of 9k to 131k 59.4 in 32, 64.6 in 40; 48 of 200 to 4000 40.0 in 32, 43.2 in 40,
// 53.9 whole (8 kv heads of 128 entries).  Over 28 shapes of 64 and 128 entries, even and uneven, 32 takes 2 % less than 40; 24 takes less yet where
// the lengths are uneven and more where they are even.
// Tiles of 128 columns: as many shares as keep all blocks resident, two to an SM, of 64 pages at most (every share of a column costs its sums a way to memory and
// back): 512 rows of one sequence of 4096 97 us in 32, 107 in 16, 192 in 4.  128 columns per tile from 256 columns on: see the kernel.
// No more shares than keep the workspace of T rows within 2^28 floats (one, and no workspace, where two would not; so many rows fill the machine many times over): 8192
// rows of 131072 positions 30.9 ms in 7 shares with 1 GB, 37.1 in 32 with 4.4; 32768 rows of 32768 15.7 in one, 17.6 in 8 with 4.4 GB.
Plan plan_of(int B, long long T, int max_q_len, int max_kv_len, int Hq, int Hkv, int window, int split_pages, int sms) {
  constexpr long long kMostFloats = 1ll << 28;
  Plan p;
  const long long G = Hq / Hkv, most = G * max_q_len;
  p.cols = most >= 2 * kWideCols ? kWideCols : most > 8 ? 16 : 8;
  p.tiles = (int)((most + p.cols - 1) / p.cols);
  long long pages = ((long long)max_kv_len + PAGE - 1) / PAGE;
  const long long rows = std::min<long long>((p.cols + G - 2) / G + 1, max_q_len);  // rows that a tile's columns may touch
  long long seen = pages;
  if (window > 0) seen = std::min(pages, ((long long)window + rows - 1 + PAGE - 2) / PAGE + 1);
  if (split_pages <= 0) {
    const long long items = (long long)B * Hkv * p.tiles;
    long long shares;
    if (p.cols == kWideCols) {
      shares = std::max(2LL * sms / items, (seen + 63) / 64);
    } else {
      const long long most_pages = p.cols == 16 ? (items > 4LL * sms ? 32 : 16) : items * ((seen + 39) / 40) <= 4LL * sms ? 40 : 32;
      shares = std::max((5LL * sms / 3 + items - 1) / items, (seen + most_pages - 1) / most_pages);
    }
    shares = std::min(shares, std::max(kMostFloats / std::max(T * Hq * (128 + 4), 1ll), 1ll));
    split_pages = (int)std::max<long long>((seen + shares - 1) / std::max(shares, 1LL), kWarps);
  }
  p.split_pages = split_pages;
  p.max_splits = (int)std::max<long long>(1, (seen + split_pages - 1) / split_pages);
  return p;
}
int device_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return effective_sms(sms);
}
bool sizes_ok(int B, int T, int max_q_len, int max_kv_len, int Hq, int Hkv, int D, int split_pages, int window) {
  return B >= 1 && B <= 65535 && T >= 0 && max_q_len >= 1 && max_kv_len >= 0 && max_kv_len <= INT32_MAX - 2 * PAGE && Hkv >= 1 && Hkv <= kMostGridY && Hq >= Hkv && Hq % Hkv == 0 &&
         (long long)max_q_len * Hq <= INT32_MAX / 2 && (D == 64 || D == 128) && (long long)Hq * D <= INT32_MAX && Hq / Hkv <= 4096 && split_pages >= 0 && split_pages <= 1 << 24 && window >= 0;
}

// more than 48 KB of shared memory wants to be asked for once per device
template <auto kernel>
cudaError_t allow_smem(int bytes) {
  static std::atomic<uint64_t> asked{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e != cudaSuccess || (asked.load(std::memory_order_relaxed) & bit)) return e;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return e;
}
template <auto kernel, int D>
cudaError_t launch(cudaStream_t stream, AttnQ4Args& a, const Plan& p, int smem, int threads = kThreads) {
  cudaError_t e = allow_smem<kernel>(smem);
  const int tiles = kMostGridY / a.Hkv;  // of a launch
  for (a.tile0 = 0; e == cudaSuccess && a.tile0 < p.tiles; a.tile0 += tiles)
    e = launch_k(kernel, dim3(p.max_splits, std::min(tiles, p.tiles - a.tile0) * a.Hkv, a.B), dim3(threads), smem, stream, true, a);
  if (e != cudaSuccess || p.max_splits == 1) return e;
  const long long at_most = (long long)a.max_q_len * a.Hq;  // rows and heads of a sequence
  if (at_most * a.B >= 4096)
    return launch_k(attn_q4_join_kernel<D, 1>, dim3((unsigned)((at_most + kWarps - 1) / kWarps), a.B), dim3(kThreads), 0, stream, true, a, p.cols);
  return launch_k(attn_q4_join_kernel<D, kWarps>, dim3((unsigned)at_most, a.B), dim3(kThreads), 0, stream, true, a, p.cols);
}
template <int D, bool CAP>
cudaError_t launch(cudaStream_t stream, AttnQ4Args& a, const Plan& p) {
  if (p.cols == kWideCols) return launch<attn_q4_wide_kernel<D, CAP>, D>(stream, a, p, Wide<D>::SMEM, Wide<D>::THREADS);
  if (p.cols == 16) return launch<attn_q4_kernel<D, 2, CAP>, D>(stream, a, p, Cfg<D, 2>::SMEM);
  return launch<attn_q4_kernel<D, 1, CAP>, D>(stream, a, p, Cfg<D, 1>::SMEM);
}
template <int D>
cudaError_t launch(cudaStream_t stream, AttnQ4Args& a, const Plan& p) {
  return a.softcap > 0.f ? launch<D, true>(stream, a, p) : launch<D, false>(stream, a, p);
}

}  // namespace

int attn_q4_split(int B, int max_q_len, int max_kv_len, int Hq, int Hkv, int window, int sms) {
  if (!sizes_ok(B, 0, max_q_len, max_kv_len, Hq, Hkv, 128, 0, window) || sms < 0) return -1;
  if (sms == 0) sms = device_sms();
  return sms > 0 ? plan_of(B, (long long)B * max_q_len, max_q_len, max_kv_len, Hq, Hkv, window, 0, sms).split_pages : -1;
}
size_t attn_q4_workspace_floats(int B, int T, int max_q_len, int max_kv_len, int Hq, int Hkv, int D, int split_pages, int window) {
  if (!sizes_ok(B, T, max_q_len, max_kv_len, Hq, Hkv, D, split_pages, window)) return 0;
  const int sms = split_pages > 0 ? 1 : device_sms();
  if (sms <= 0) return 0;
  const Plan p = plan_of(B, T, max_q_len, max_kv_len, Hq, Hkv, window, split_pages, sms);
  return p.max_splits > 1 ? (size_t)T * Hq * p.max_splits * (D + 4) : 0;
}

namespace {
std::atomic<long long> wait_limit{HB_WAIT_TIMEOUT_CYCLES};
}
long long attn_q4_wait_cycles(long long cycles) { return wait_limit.exchange(cycles); }
cudaError_t attn_q4_status() {
  unsigned ran_out = 0;
  cudaError_t e = cudaMemcpyFromSymbol(&ran_out, wait_ran_out, sizeof ran_out);
  if (e != cudaSuccess || !ran_out) return e;
  const unsigned none = 0;
  e = cudaMemcpyToSymbol(wait_ran_out, &none, sizeof none);
  return e == cudaSuccess ? cudaErrorLaunchTimeout : e;
}

cudaError_t attn_q4(cudaStream_t stream, AttnQ4Args a) {
  if (!sizes_ok(a.B, a.T, a.max_q_len, a.max_kv_len, a.Hq, a.Hkv, a.D, a.split_pages, a.window)) return cudaErrorInvalidValue;
  if (a.page_size != PAGE || a.num_pages < 1 || a.num_pages > INT32_MAX / PAGE || a.max_pages < 0 || !(a.softcap >= 0.f) || !(a.softcap < INFINITY) || !(fabsf(a.scale) < INFINITY))
    return cudaErrorInvalidValue;
  if (a.T == 0) return cudaSuccess;
  if (!a.q || !a.k_cache || !a.v_cache || !a.kv_lens || !a.out || (a.max_pages > 0 && !a.page_table)) return cudaErrorInvalidValue;
  if (!a.cu_seqlens && (a.T < a.B || a.max_q_len != 1)) return cudaErrorInvalidValue;
  const int need = a.Hq * a.D;
  if (((uintptr_t)a.q & 15) || a.ldq < need || a.ldq % 8 || a.ldo < need || ((uintptr_t)a.out & 1) || ((uintptr_t)a.k_cache & 15) || ((uintptr_t)a.v_cache & 15))
    return cudaErrorInvalidValue;
  const int sms = a.split_pages > 0 ? 1 : device_sms();
  if (sms <= 0) return cudaErrorNoDevice;
  const Plan p = plan_of(a.B, a.T, a.max_q_len, a.max_kv_len, a.Hq, a.Hkv, a.window, a.split_pages, sms);
  if (p.max_splits > 1 && (!a.workspace || ((uintptr_t)a.workspace & 15))) return cudaErrorInvalidValue;
  a.split_pages = p.split_pages;
  a.max_splits = p.max_splits;
  if (a.window >= a.max_kv_len) a.window = 0;  // every position is in it
  a.wait_cycles = wait_limit.load(std::memory_order_relaxed);
  a.group = a.Hq / a.Hkv;
  a.inv_group = ((1ull << 32) + a.group - 1) / a.group;  // x inv >> 32 = x / group for x < 2^32 / group: columns of a tile and the rest before them
  a.kv_bound = (int)std::min<long long>((long long)a.max_pages * PAGE, a.max_kv_len);
  return a.D == 128 ? launch<128>(stream, a, p) : launch<64>(stream, a, p);
}

}  // namespace hb

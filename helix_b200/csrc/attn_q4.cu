// Attention of the last rows of each sequence over a 4-bit paged cache (layout: quant4.cuh): single tokens, and portions of several rows.
//
//   o = sum_j p_j v_j,  p = softmax over the visible j of s_j,  s = scale q.k (capped: cap tanh(s / cap)),  a sink adds exp(sink) to the denominator
//
// The columns of a block are (row, query head) pairs of one kv head, eight per product: S^T[16 positions x 8 columns] = K q^T and
// O^T[16 entries x 8 columns] += V^T P^T as warp-wide 16 x 8 x 16 products.  Both operands that come from the cache are then the 16-row one, the
// codes go straight from their words to its registers, and no cached byte passes through shared memory twice.  The tensor-memory path would need
// the widened entries in shared memory: four times the cache's bytes written there and read again.
// Instructions bound it (HBM gives a position of a kv head of 128 entries 25 issue slots), the products least of all.
//   c - 8 is exact in fp16.  (Codes as they are, numbers below fp16's smallest normal one, with the 8 taken off by a further product, save four
//      of nine instructions per word, but such products are summed to some 14 bits only: results whose codes are near 8 were off by 2^-15 of a group's weight.)
//   S: the products of a group of 32 entries are summed by themselves, then times the key group's scale in fp32.
//   O: the value group's scale depends on the position, which is summed over: it goes into P^T, one operand per group, fp16 (bf16 would add as much
//      error as the output's own rounding; here two roundings of at most 2^-11 each, and 2^-35 of the largest weight for weights far below it).  A
//      group's scales are brought near 1 by a power of two that follows their largest finite one so far, as the running maximum does for the
//      scores; scales below 2^-18 of that largest lose bits.
//   q: fp16 after a power of two per column (bf16 has fewer bits; entries 2^-27 of the column's largest and below lose some).
// Softmax statistics and sums are fp32.  A warp takes every fourth page of the block's share by itself; the four meet at the end.
//
// A sequence of more than `split` pages is cut into as few even shares as none is larger, so a row's bits depend on its own sequence and
// `split`, not on who shares the launch.
// Sequences of more than one share leave (O, m, l) per share in the workspace, which a second kernel joins in order.
//
// Measured (8 kv heads of 128 entries, 32 query heads): 32 sequences of 1.5k to 2.2k positions 25 us (68 MB, 41 % of the copy rate: two blocks on most SMs
// and one on the others, some 5 us of launch, first loads and last sums), 74 of 8k 140 us (700 MB, 76 %: 18.5 instructions per position and kv head at 65 %
// of the issue slots; at 2k each, 41.5 us, the kernel takes 7 % less without its loads, 12 % less without the 8 taken off the codes, 2 % less without V's
// products), three of 9k to 131k 65 us (242 MB, 56 %).  Also tried: scores in shared memory and rolled loops (a fifth more instructions), e4m3 products (widened to fp16 by
// further instructions on this chip: 41 -> 52), pages dealt evenly over all blocks by the launch's lengths (two runs of pages per block: 26 -> 37), clusters
// that join their sums through distributed shared memory (26 -> 29 for 32 sequences in pairs).
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
constexpr int SLOTS = 3;  // halves (K or V) of pages that a warp has in shared memory
constexpr float kLog2e = 1.4426950408889634f;

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

// the 16 (D = 128) or 8 (D = 64) bytes that a lane takes of a row or pair
template <int D>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[D / 32]) {
  if constexpr (D == 128) {
    const uint4 u = *reinterpret_cast<const uint4*>(p);
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else {
    const uint2 u = *reinterpret_cast<const uint2*>(p);
    w[0] = u.x; w[1] = u.y;
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

template <int D, int NT, bool CAP>
__global__ void __launch_bounds__(kThreads, Cfg<D, NT>::BLOCKS) attn_q4_kernel(const AttnQ4Args a) {
  using C = Cfg<D, NT>;
  constexpr int J = C::J;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int G = a.group;
  const int b = blockIdx.z, ct = blockIdx.y / a.Hkv, kvh = blockIdx.y - ct * a.Hkv;
  const Tile tile = tile_of(a, b, ct, C::COLS);
  if (tile.cols <= 0) return;
  auto row_of = [&](int c) { return div_g(a, tile.rest + c); };  // row of column c
  const int shares = tile.splits;
  if (tile.pages == 0) {  // nothing to see
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < tile.cols * D; i += kThreads) {
        const int c = i / D, r = row_of(c);
        a.out[(size_t)(tile.row0 + r) * a.ldo + (size_t)(kvh * G + tile.rest + c - r * G) * D + i % D] = __float2bfloat16(0.f);
      }
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
      for (int i = 0; i < 4; ++i) {
        const uint32_t lo = w[i] & 0x7fffu, hi = (w[i] >> 16) & 0x7fffu;
        if (lo < 0x7f80u) mag = max(mag, lo);
        if (hi < 0x7f80u) mag = max(mag, hi);
      }
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
#pragma unroll
  for (int j = 0; j < J; ++j) {
    ex[j] = 12;
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
    if constexpr (CAP) {  // cap tanh(x / cap) as log2 of a weight, tanh(y) = 1 - 2 / (e^2y + 1)
      const float in = 2.f * kLog2e / a.softcap, out = a.softcap * kLog2e;
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int h = 0; h < 4; ++h) s[blk][n][h] = fmaf(-2.f * out, __fdividef(1.f, exp2_fast(s[blk][n][h] * mul[n][h & 1] * in) + 1.f), out);
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
  __syncthreads();

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

// One block per (row, head): what more than one block has worked on is joined, a warp taking every fourth share
template <int D>
__global__ void __launch_bounds__(kThreads) attn_q4_join_kernel(const AttnQ4Args a, int cols_per_tile) {
  constexpr int V = D / 32;
  __shared__ float s_part[kWarps][D + 2];
  const int b = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int i = blockIdx.x / a.Hq, head = blockIdx.x - i * a.Hq;
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
  // up to eight of the warp's shares at a time
  float m = -INFINITY, sum = 0.f, acc[V] = {};
  for (int s0 = warp; s0 < shares; s0 += 8 * kWarps) {
    float x[8][V];
    float2 ml[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      ml[k] = make_float2(-INFINITY, 0.f);
      if (s0 + k * kWarps < shares) {
        const float* p = src + (size_t)(s0 + k * kWarps) * (D + 4);
        ml[k] = *reinterpret_cast<const float2*>(p + D);
#pragma unroll
        for (int v = 0; v < V; ++v) x[k][v] = p[lane + 32 * v];
      } else {
#pragma unroll
        for (int v = 0; v < V; ++v) x[k][v] = 0.f;
      }
    }
    float top = m;
#pragma unroll
    for (int k = 0; k < 8; ++k) top = fmaxf(top, ml[k].x);
    const float ref = top == -INFINITY ? 0.f : top, old = exp2_fast(m - ref);
    m = top;
    sum *= old;
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] *= old;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const float f = exp2_fast(ml[k].x - ref);
      sum = fmaf(ml[k].y, f, sum);
#pragma unroll
      for (int v = 0; v < V; ++v) acc[v] = fmaf(x[k][v], f, acc[v]);
    }
  }
#pragma unroll
  for (int v = 0; v < V; ++v) s_part[warp][lane + 32 * v] = acc[v];
  if (lane == 0) {
    s_part[warp][D] = m;
    s_part[warp][D + 1] = sum;
  }
  __syncthreads();
  if (threadIdx.x < D) {
    float top = sink;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, s_part[w][D]);
    const float ref = top == -INFINITY ? 0.f : top;
    float y = 0.f, all = exp2_fast(sink - ref);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = exp2_fast(s_part[w][D] - ref);
      y = fmaf(s_part[w][threadIdx.x], f, y);
      all = fmaf(s_part[w][D + 1], f, all);
    }
    a.out[(size_t)row * a.ldo + (size_t)head * D + threadIdx.x] = __float2bfloat16(all == 0.f ? 0.f : y / all);
  }
}

struct Plan {
  int split_pages, max_splits, tiles, cols;
};
// By the rule (split_pages 0) a tile's pages are cut into so many shares that there are some 1.67 blocks per SM, and that none has more than 32 pages,
// or 40 where all blocks are resident at once, four to an SM (16 where a tile has 16 columns: a page takes twice as long there); a share is a page
// per warp at least.  Both sides, us: one sequence of 2k 6.4 in shares of 4 pages, 15.1 whole; 8 of 2k 10.0 in 8, 15.8 whole; 32 of 1.5k to 2.2k 24.9
// in 36, 29.9 in 24; 32 of 8k 66.2 in 32, 67.2 in 40, 73.1 in 48; three of 9k to 131k 59.4 in 32, 64.6 in 40; 48 of 200 to 4000 40.0 in 32, 43.2 in 40,
// 53.9 whole (8 kv heads of 128 entries).  Over 28 shapes of 64 and 128 entries, even and uneven, 32 takes 2 % less than 40; 24 takes less yet where
// the lengths are uneven and more where they are even.
Plan plan_of(int B, int max_q_len, int max_kv_len, int Hq, int Hkv, int window, int split_pages, int sms) {
  Plan p;
  const long long G = Hq / Hkv, most = G * max_q_len;
  p.cols = most > 8 ? 16 : 8;
  p.tiles = (int)((most + p.cols - 1) / p.cols);
  long long pages = ((long long)max_kv_len + PAGE - 1) / PAGE;
  const long long rows = std::min<long long>((p.cols + G - 2) / G + 1, max_q_len);  // rows that a tile's columns may touch
  long long seen = pages;
  if (window > 0) seen = std::min(pages, ((long long)window + rows - 1 + PAGE - 2) / PAGE + 1);
  if (split_pages <= 0) {
    const long long items = (long long)B * Hkv * p.tiles;
    const long long most_pages = p.cols == 16 ? 16 : items * ((seen + 39) / 40) <= 4LL * sms ? 40 : 32;
    const long long shares = std::max((5LL * sms / 3 + items - 1) / items, (seen + most_pages - 1) / most_pages);
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
  return B >= 1 && B <= 65535 && T >= 0 && max_q_len >= 1 && max_kv_len >= 0 && max_kv_len <= INT32_MAX - 2 * PAGE && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 &&
         (long long)max_q_len * Hq <= INT32_MAX / 2 && (D == 64 || D == 128) && (long long)Hq * D <= INT32_MAX && Hq / Hkv <= 4096 && split_pages >= 0 && split_pages <= 1 << 24 && window >= 0;
}

// more than 48 KB of shared memory wants to be asked for once per device
template <int D, int NT, bool CAP>
cudaError_t allow_smem() {
  static std::atomic<uint64_t> asked{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e != cudaSuccess || (asked.load(std::memory_order_relaxed) & bit)) return e;
  e = cudaFuncSetAttribute(attn_q4_kernel<D, NT, CAP>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, NT>::SMEM);
  if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return e;
}
template <int D, int NT, bool CAP>
cudaError_t launch(cudaStream_t stream, const AttnQ4Args& a, const Plan& p) {
  cudaError_t e = allow_smem<D, NT, CAP>();
  if (e != cudaSuccess) return e;
  e = launch_k(attn_q4_kernel<D, NT, CAP>, dim3(p.max_splits, p.tiles * a.Hkv, a.B), dim3(kThreads), Cfg<D, NT>::SMEM, stream, true, a);
  if (e != cudaSuccess || p.max_splits == 1) return e;
  return launch_k(attn_q4_join_kernel<D>, dim3(a.max_q_len * a.Hq, a.B), dim3(kThreads), 0, stream, true, a, p.cols);
}
template <int D, int NT>
cudaError_t launch(cudaStream_t stream, const AttnQ4Args& a, const Plan& p) {
  return a.softcap > 0.f ? launch<D, NT, true>(stream, a, p) : launch<D, NT, false>(stream, a, p);
}

}  // namespace

int attn_q4_split(int B, int max_q_len, int max_kv_len, int Hq, int Hkv, int window, int sms) {
  if (!sizes_ok(B, 0, max_q_len, max_kv_len, Hq, Hkv, 128, 0, window) || sms < 0) return -1;
  if (sms == 0) sms = device_sms();
  return sms > 0 ? plan_of(B, max_q_len, max_kv_len, Hq, Hkv, window, 0, sms).split_pages : -1;
}
size_t attn_q4_workspace_floats(int B, int T, int max_q_len, int max_kv_len, int Hq, int Hkv, int D, int split_pages, int window) {
  if (!sizes_ok(B, T, max_q_len, max_kv_len, Hq, Hkv, D, split_pages, window)) return 0;
  const int sms = split_pages > 0 ? 1 : device_sms();
  if (sms <= 0) return 0;
  const Plan p = plan_of(B, max_q_len, max_kv_len, Hq, Hkv, window, split_pages, sms);
  return p.max_splits > 1 ? (size_t)T * Hq * p.max_splits * (D + 4) : 0;
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
  const Plan p = plan_of(a.B, a.max_q_len, a.max_kv_len, a.Hq, a.Hkv, a.window, a.split_pages, sms);
  if (p.max_splits > 1 && (!a.workspace || ((uintptr_t)a.workspace & 15))) return cudaErrorInvalidValue;
  if ((long long)p.tiles * a.Hkv > 65535) return cudaErrorInvalidValue;
  a.split_pages = p.split_pages;
  a.max_splits = p.max_splits;
  if (a.window >= a.max_kv_len) a.window = 0;  // every position is in it
  a.group = a.Hq / a.Hkv;
  a.inv_group = ((1ull << 32) + a.group - 1) / a.group;  // x inv >> 32 = x / group for x < 2^32 / group: columns of a tile and the rest before them
  a.kv_bound = (int)std::min<long long>((long long)a.max_pages * PAGE, a.max_kv_len);
  if (a.D == 128) return p.cols == 16 ? launch<128, 2>(stream, a, p) : launch<128, 1>(stream, a, p);
  return p.cols == 16 ? launch<64, 2>(stream, a, p) : launch<64, 1>(stream, a, p);
}

}  // namespace hb

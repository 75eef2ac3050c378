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
//      error as the output's own rounding; here two roundings of at most 2^-11 each).  A group's scales are brought near 1 by a power of two that
//      follows their largest finite one so far, as the running maximum does for the scores: what falls below 2^-36 of a sequence's
//      largest weight of that group is lost, and only there fp16's range is felt.
//   q: fp16 after a power of two per column (bf16 has fewer bits; entries 2^-27 of the column's largest and below lose some).
// Softmax statistics and sums are fp32.  A warp takes every fourth page of the block's share by itself; the four meet at the end.
//
// Shares are `split` pages, counted from position 0, so a row's bits depend on its own sequence and `split`, not on who shares the launch.
// Sequences of more than one share leave (O, m, l) per share in the workspace, which a second kernel joins in order.
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
constexpr int STAGES = 2;  // pages of a warp in shared memory: one in use, one under way
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
  int row0, rows;      // packed rows of the sequence
  int kv, pos0;        // its length, the position of its first row
  int col0, cols;      // columns of the tile
  int lo, hi;          // positions that some column sees
  int split0, splits;  // shares
};
__device__ __forceinline__ Tile tile_of(const AttnQ4Args& a, int b, int ct, int cols_per_tile) {
  Tile t;
  const int G = a.Hq / a.Hkv;
  t.row0 = a.cu_seqlens ? min(max(a.cu_seqlens[b], 0), a.T) : b;
  t.rows = a.cu_seqlens ? min(min(max(a.cu_seqlens[b + 1], 0), a.T) - t.row0, a.max_q_len) : 1;
  t.kv = min(max(a.kv_lens[b], 0), a.kv_bound);
  t.pos0 = t.kv - t.rows;
  t.col0 = ct * cols_per_tile;
  t.cols = min(max(t.rows, 0) * G - t.col0, cols_per_tile);
  const int last = (t.col0 + max(t.cols, 1) - 1) / G;
  t.hi = min(max(t.pos0 + last + 1, 0), t.kv);
  t.lo = a.window > 0 ? max(t.pos0 + t.col0 / G - a.window + 1, 0) : 0;
  const int p0 = t.lo / PAGE, p1 = (t.hi + PAGE - 1) / PAGE;
  t.split0 = p0 / a.split_pages;
  t.splits = t.hi > t.lo ? (p1 + a.split_pages - 1) / a.split_pages - t.split0 : 0;
  return t;
}

template <int D, int NT>
struct Cfg {
  static constexpr int J = D / q4::kGroup;
  static constexpr int BLOCK = q4::block_bytes(D);
  static constexpr int COLS = 8 * NT;
  static constexpr int RING = kWarps * STAGES * 2 * BLOCK;
  static constexpr int MERGE = kWarps * COLS * (D + 2) * 4;
  static constexpr int SMEM = RING > MERGE ? RING : MERGE;
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

template <int D, int NT>
__global__ void __launch_bounds__(kThreads, NT == 1 ? 3 : 2) attn_q4_kernel(const AttnQ4Args a) {
  using C = Cfg<D, NT>;
  constexpr int J = C::J;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.z, kvh = blockIdx.y % a.Hkv, ct = blockIdx.y / a.Hkv;
  const int G = a.Hq / a.Hkv;
  const Tile tile = tile_of(a, b, ct, C::COLS);
  if (tile.cols <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  if (tile.splits == 0) {  // nothing to see
    if (blockIdx.x == 0)
      for (int i = threadIdx.x; i < tile.cols * D; i += kThreads) {
        const int c = tile.col0 + i / D;
        a.out[(size_t)(tile.row0 + c / G) * a.ldo + (size_t)(kvh * G + c % G) * D + i % D] = __float2bfloat16(0.f);
      }
    return;
  }
  if ((int)blockIdx.x >= tile.splits) return;
  const int split = tile.split0 + blockIdx.x;
  const int p_begin = max(split * a.split_pages, tile.lo / PAGE), p_end = min((split + 1) * a.split_pages, (tile.hi + PAGE - 1) / PAGE);

  uint8_t* ring = smem + warp * (STAGES * 2 * C::BLOCK);
  const int32_t* table = a.page_table + (size_t)b * a.max_pages;
  const size_t block0 = (size_t)kvh * C::BLOCK + lane * 16, page_stride = (size_t)a.Hkv * C::BLOCK;
  // the warp's pages are p_begin + warp + 4 i; lane i % 32 holds the number of page i, -1 for one that is none: its positions are not seen
  const int n_mine = (p_end - p_begin - warp + kWarps - 1) / kWarps;
  int ids = -1;
  auto look_up = [&](int i) {
    ids = -1;
    if (i + lane < n_mine) {
      const int id = table[p_begin + warp + kWarps * (i + lane)];
      if (id >= 0 && id < a.num_pages) ids = id;
    }
  };
  auto fetch = [&](int i, int stage) {  // all lanes; returns the page's number
    if ((i & 31) == 0) look_up(i);
    const int id = __shfl_sync(0xffffffffu, ids, i & 31);
    if (i < n_mine && id >= 0) {
      const uint8_t *k = a.k_cache + (size_t)id * page_stride + block0, *v = a.v_cache + (size_t)id * page_stride + block0;
      uint8_t* dst = ring + stage * 2 * C::BLOCK + lane * 16;
#pragma unroll
      for (int c = 0; c < C::BLOCK; c += 512)
        if (c + 512 <= C::BLOCK || c + lane * 16 < C::BLOCK) copy16(dst + c, k + c);
      copy_commit();
#pragma unroll
      for (int c = 0; c < C::BLOCK; c += 512)
        if (c + 512 <= C::BLOCK || c + lane * 16 < C::BLOCK) copy16(dst + C::BLOCK + c, v + c);
    } else {
      copy_commit();
    }
    copy_commit();
    return i < n_mine ? id : -1;
  };
  int id = fetch(0, 0);

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
      const int col = tile.col0 + c;
      const bf16* src = a.q + (size_t)(tile.row0 + col / G) * a.ldq + (size_t)(kvh * G + col % G) * D + t * 8;
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
    const float scale = a.softcap > 0.f ? fabsf(a.scale) : fabsf(a.scale) * kLog2e;
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
  auto last_of = [&](int c) { return c < tile.cols ? tile.pos0 + (tile.col0 + c) / G : -1; };  // positions a column sees: first_of <= j <= last_of
  auto first_of = [&](int last) { return a.window > 0 ? last - a.window + 1 : 0; };
  // every column sees a page whole that lies in [all_lo, all_hi]
  const int all_hi = tile.pos0 + tile.col0 / G;
  const int all_lo = a.window > 0 ? tile.pos0 + (tile.col0 + tile.cols - 1) / G - a.window + 1 : 0;

  float o[J][2][NT][4];
  float m[NT][2], l[NT][2];  // running maximum (log2 of a weight) and sum of weights times 16
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

  // One page; `whole`: every column sees all of it
  auto page = [&](uint8_t* kb, const int pos, auto whole_t) {
    constexpr bool whole = decltype(whole_t)::value;
    uint8_t* vb = kb + C::BLOCK;
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
          for (int i = 0; i < 4; ++i) s[blk][n][i] = j == 0 ? (i < 2 ? d0 : d1)[j] * c[i] : fmaf((i < 2 ? d0 : d1)[j], c[i], s[blk][n][i]);
        }
      }
    }
    if (a.softcap > 0.f) {  // cap tanh(x / cap) as log2 of a weight, tanh(y) = 1 - 2 / (e^2y + 1)
      const float in = 2.f * kLog2e / a.softcap, out = a.softcap * kLog2e;
#pragma unroll
      for (int blk = 0; blk < 4; ++blk)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            s[blk][n][i] = fmaf(-2.f * out, __fdividef(1.f, exp2_fast(s[blk][n][i] * mul[n][i & 1] * in) + 1.f), out);
    }
    if constexpr (!whole) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int hi = last_of(n * 8 + 2 * t + i), lo = first_of(hi);
#pragma unroll
          for (int blk = 0; blk < 4; ++blk)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int at = pos + blk * 16 + g + 8 * h;
              if (at > hi || at < lo) s[blk][n][i + 2 * h] = -INFINITY;
            }
        }
    }
    // running maximum
    bool moved = false;
    float keep[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float x = fmaxf(s[0][n][i], s[0][n][i + 2]);
#pragma unroll
        for (int blk = 1; blk < 4; ++blk) x = fmaxf(x, fmaxf(s[blk][n][i], s[blk][n][i + 2]));
#pragma unroll
        for (int w = 4; w < 32; w <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, w));
        if (!(a.softcap > 0.f)) x *= mul[n][i];
        keep[n][i] = x > m[n][i] ? exp2_fast(m[n][i] - x) : 1.f;  // (-inf before: 0)
        moved |= x > m[n][i];
        m[n][i] = fmaxf(m[n][i], x);
      }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          l[n][i] *= keep[n][i];
#pragma unroll
          for (int j = 0; j < J; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              o[j][h][n][i] *= keep[n][i];
              o[j][h][n][i + 2] *= keep[n][i];
            }
        }
    }
    // value scales: a lane takes those of positions 2 lane and 2 lane + 1, follows each group's largest exponent, and puts them back as
    // fp16 pairs of the two positions with the largest in [2^10, 2^11)
    {
      uint32_t w[J];
      uint8_t* mine = vb + q4::code_bytes(D) + lane * (J * 4);
      load_words<D>(mine, w);
      const int at = pos + 2 * lane;
      auto finite = [](uint32_t x) {  // halves that are infinities or NaN: 0 (they reach their columns through the weights)
        return (x & 0xffffu) < 0x7f80u ? ((x >> 16) < 0x7f80u ? x : x & 0xffffu) : ((x >> 16) < 0x7f80u ? x & 0xffff0000u : 0u);
      };
      uint32_t pair[J];
#pragma unroll
      for (int i = 0; i < J / 2; ++i) {
        uint32_t x = 0, y = 0;
        if (whole || (at >= tile.lo && at < tile.hi)) x = w[i] & 0x7fff7fffu;
        if (whole || (at + 1 >= tile.lo && at + 1 < tile.hi)) y = w[J / 2 + i] & 0x7fff7fffu;
        const uint32_t both = __vmaxu2(x, y);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int j = 2 * i + h;
          uint32_t most = __reduce_max_sync(0xffffffffu, h ? both >> 16 : both & 0xffffu);
          if (most >= 0x7f80u) {
            const uint32_t z = __vmaxu2(finite(x), finite(y));
            most = __reduce_max_sync(0xffffffffu, h ? z >> 16 : z & 0xffffu);
          }
          const int e = (int)(most >> 7);
          if (e > ex[j]) {
            const float less = exp2f((float)(ex[j] - e));
            ex[j] = e;
#pragma unroll
            for (int q = 0; q < 2; ++q)
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int k = 0; k < 4; ++k) o[j][q][n][k] *= less;
          }
          const float near1 = __uint_as_float((uint32_t)(264 - ex[j]) << 23);  // 2^(137 - ex)
          pair[j] = q4::pack_f16x2((h ? q4::bf16_hi(w[i]) : q4::bf16_lo(w[i])) * near1, (h ? q4::bf16_hi(w[J / 2 + i]) : q4::bf16_lo(w[J / 2 + i])) * near1);
        }
      }
      if constexpr (J == 4) *reinterpret_cast<uint4*>(mine) = make_uint4(pair[0], pair[1], pair[2], pair[3]);
      else *reinterpret_cast<uint2*>(mine) = make_uint2(pair[0], pair[1]);
      __syncwarp();
    }
#pragma unroll
    for (int blk = 0; blk < 4; ++blk) {
      const int p0 = blk * 8 + t;
      uint32_t v0[J], v1[J], s0[J], s1[J], b0[NT], b1[NT];
      load_words<D>(vb + p0 * D + (g ^ q4::place_xor(D, p0)) * (D / 8), v0);
      load_words<D>(vb + (p0 + 4) * D + (g ^ q4::place_xor(D, p0 + 4)) * (D / 8), v1);
      load_words<D>(vb + q4::code_bytes(D) + p0 * (J * 4), s0);
      load_words<D>(vb + q4::code_bytes(D) + (p0 + 4) * (J * 4), s1);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float base = 4.f - (m[n][i & 1] == -INFINITY ? 0.f : m[n][i & 1]);  // weights times 16: fp16 holds them better
          w[i] = exp2_fast(a.softcap > 0.f ? s[blk][n][i] + base : fmaf(s[blk][n][i], mul[n][i & 1], base));
          l[n][i & 1] += w[i];
        }
        b0[n] = q4::transpose8(q4::pack_f16x2(w[0], w[1]));
        b1[n] = q4::transpose8(q4::pack_f16x2(w[2], w[3]));
      }
      uint32_t see0[NT], see1[NT];  // what a column does not see has no part in it, whatever its bytes say
      if constexpr (!whole) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
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

  for (int i = 0; i < n_mine; ++i) {
    const int next = fetch(i + 1, (i + 1) & 1);
    copy_wait<2>();
    __syncwarp();
    if (id >= 0) {
      uint8_t* kb = ring + (i & 1) * 2 * C::BLOCK;
      const int pos = (p_begin + warp + kWarps * i) * PAGE;
      if (pos >= all_lo && pos + PAGE - 1 <= all_hi) page(kb, pos, std::true_type{});
      else page(kb, pos, std::false_type{});
    }
    __syncwarp();  // the stage is free for the fetch after next
    id = next;
  }
  copy_wait<0>();
  __syncthreads();

  // the four warps meet: [warp][column][D + 2]
  float* sm = reinterpret_cast<float*>(smem);
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int c = n * 8 + 2 * t + i;
      float* dst = sm + (size_t)(warp * C::COLS + c) * (D + 2);
      float sum = l[n][i];
#pragma unroll
      for (int w = 4; w < 32; w <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
#pragma unroll
      for (int j = 0; j < J; ++j) {
        const float back = __uint_as_float((uint32_t)(ex[j] - 10) << 23);  // 2^(ex - 137)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          dst[32 * j + 4 * g + 2 * h] = o[j][h][n][i] * back;
          dst[32 * j + 4 * g + 2 * h + 1] = o[j][h][n][i + 2] * back;
        }
      }
      if (g == 0) {
        dst[D] = m[n][i];
        dst[D + 1] = sum;
      }
    }
  __syncthreads();
  for (int i = threadIdx.x; i < tile.cols * D; i += kThreads) {
    const int c = i / D, d = i % D;
    const int col = tile.col0 + c, row = tile.row0 + col / G, head = kvh * G + col % G;
    float mt = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mt = fmaxf(mt, sm[(size_t)(w * C::COLS + c) * (D + 2) + D]);
    float sink = -INFINITY;
    if (tile.splits == 1 && a.sink) sink = __bfloat162float(a.sink[head]) * kLog2e;
    const float mm = fmaxf(mt, sink), ref = mm == -INFINITY ? 0.f : mm;
    float acc = 0.f, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* src = sm + (size_t)(w * C::COLS + c) * (D + 2);
      const float f = exp2_fast(src[D] - ref - 4.f);  // (sums are 16 times what they stand for)
      acc = fmaf(src[d], f, acc);
      sum = fmaf(src[D + 1], f, sum);
    }
    if (tile.splits == 1) {
      sum += exp2_fast(sink - ref);
      a.out[(size_t)row * a.ldo + (size_t)head * D + d] = __float2bfloat16(sum == 0.f ? 0.f : acc / sum);
    } else {
      float* dst = a.workspace + (((size_t)row * a.Hq + head) * a.max_splits + blockIdx.x) * (D + 2);
      dst[d] = acc;
      if (d == 0) {
        dst[D] = mt;
        dst[D + 1] = sum;
      }
    }
  }
}

// One warp per (row, head) of sequences that more than one block has worked on
template <int D>
__global__ void __launch_bounds__(128) attn_q4_join_kernel(const AttnQ4Args a, int cols_per_tile) {
  constexpr int V = D / 32;
  pdl_wait();
  pdl_launch_dependents();
  const int b = blockIdx.y, lane = threadIdx.x & 31;
  const int at = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (at >= a.max_q_len * a.Hq) return;
  const int i = at / a.Hq, head = at % a.Hq, G = a.Hq / a.Hkv;
  const Tile tile = tile_of(a, b, (i * G + head % G) / cols_per_tile, cols_per_tile);
  if (i >= tile.rows || tile.splits <= 1) return;
  const int row = tile.row0 + i;
  const float* src = a.workspace + ((size_t)row * a.Hq + head) * a.max_splits * (D + 2);
  const float sink = a.sink ? __bfloat162float(a.sink[head]) * kLog2e : -INFINITY;
  float m = sink;
  for (int s = lane; s < tile.splits; s += 32) m = fmaxf(m, src[(size_t)s * (D + 2) + D]);
#pragma unroll
  for (int w = 16; w > 0; w >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
  const float ref = m == -INFINITY ? 0.f : m;
  float acc[V] = {}, sum = exp2_fast(sink - ref);
  for (int s = 0; s < tile.splits; ++s) {
    const float* p = src + (size_t)s * (D + 2);
    const float f = exp2_fast(p[D] - ref);
    sum = fmaf(p[D + 1], f, sum);
#pragma unroll
    for (int v = 0; v < V; ++v) acc[v] = fmaf(p[lane + 32 * v], f, acc[v]);
  }
#pragma unroll
  for (int v = 0; v < V; ++v)
    a.out[(size_t)row * a.ldo + (size_t)head * D + lane + 32 * v] = __float2bfloat16(sum == 0.f ? 0.f : acc[v] / sum);
}

struct Plan {
  int split_pages, max_splits, tiles, cols;
};
// Shares: with few (sequence, kv head, tile) items the cache is cut so that there are blocks for every SM's places; never below four
// pages, one per warp.
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
    const long long items = (long long)B * Hkv * p.tiles, places = 3LL * sms;
    const long long want = std::max<long long>(1, places / items);
    split_pages = (int)std::min<long long>(std::max<long long>((seen + want - 1) / want, 4), 1 << 24);
    split_pages = (split_pages + kWarps - 1) / kWarps * kWarps;
  }
  p.split_pages = split_pages;
  const long long all = (pages + split_pages - 1) / split_pages;
  p.max_splits = (int)std::max<long long>(1, window > 0 ? std::min(all, (seen + split_pages - 2) / split_pages + 1) : all);
  return p;
}
int device_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return effective_sms(sms);
}
bool sizes_ok(int B, int T, int max_q_len, int max_kv_len, int Hq, int Hkv, int D, int split_pages, int window) {
  return B >= 1 && B <= 65535 && T >= 0 && max_q_len >= 1 && max_kv_len >= 0 && max_kv_len <= INT32_MAX - 2 * PAGE && Hkv >= 1 && Hq >= Hkv && Hq % Hkv == 0 &&
         (long long)max_q_len * Hq <= INT32_MAX / 2 && (D == 64 || D == 128) && (long long)Hq * D <= INT32_MAX && split_pages >= 0 && split_pages <= 1 << 24 && window >= 0;
}

// more than 48 KB of shared memory wants to be asked for once per device
template <int D, int NT>
cudaError_t allow_smem() {
  static std::atomic<uint64_t> asked{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e != cudaSuccess || (asked.load(std::memory_order_relaxed) & bit)) return e;
  e = cudaFuncSetAttribute(attn_q4_kernel<D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D, NT>::SMEM);
  if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return e;
}
template <int D, int NT>
cudaError_t launch(cudaStream_t stream, const AttnQ4Args& a, const Plan& p) {
  cudaError_t e = allow_smem<D, NT>();
  if (e != cudaSuccess) return e;
  e = launch_k(attn_q4_kernel<D, NT>, dim3(p.max_splits, p.tiles * a.Hkv, a.B), dim3(kThreads), Cfg<D, NT>::SMEM, stream, true, a);
  if (e != cudaSuccess || p.max_splits == 1) return e;
  return launch_k(attn_q4_join_kernel<D>, dim3((a.max_q_len * a.Hq + 3) / 4, a.B), dim3(128), 0, stream, true, a, p.cols);
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
  return p.max_splits > 1 ? (size_t)T * Hq * p.max_splits * (D + 2) : 0;
}

cudaError_t attn_q4(cudaStream_t stream, AttnQ4Args a) {
  if (!sizes_ok(a.B, a.T, a.max_q_len, a.max_kv_len, a.Hq, a.Hkv, a.D, a.split_pages, a.window)) return cudaErrorInvalidValue;
  if (a.page_size != PAGE || a.num_pages < 1 || a.num_pages > INT32_MAX / PAGE || a.max_pages < 0 || !(a.softcap >= 0.f) || !(a.scale == a.scale))
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
  if (p.max_splits > 1 && !a.workspace) return cudaErrorInvalidValue;
  if ((long long)p.tiles * a.Hkv > 65535) return cudaErrorInvalidValue;
  a.split_pages = p.split_pages;
  a.max_splits = p.max_splits;
  a.kv_bound = (int)std::min<long long>((long long)a.max_pages * PAGE, a.max_kv_len);
  if (a.D == 128) return p.cols == 16 ? launch<128, 2>(stream, a, p) : launch<128, 1>(stream, a, p);
  return p.cols == 16 ? launch<64, 2>(stream, a, p) : launch<64, 1>(stream, a, p);
}

}  // namespace hb

// Rows of a step written into a 4-bit paged cache (layout: quant4.cuh).
//
// A group of 32 entries: m = the entry of largest magnitude (the first of equals), d = bf16(m / -8), c = clamp(floor(x / d + 1/2) + 8, 0, 15), so that m
// itself gets code 0 and is kept to bf16's rounding; d = 0 gives code 8, and a group with an infinity or a NaN gets d = NaN: it reads as NaN.
// The scale is rounded before the codes are chosen, so they are the nearest ones for the scale that is stored.
//
// Eight entries per thread (one 16-byte load), four threads per group.  Their codes fill one word of the key layout and two half words of the
// value layout; no byte is shared by two positions, so rows of one page may be written by any threads in any order.
//
// Instructions bound it: 16,001 rows of 8 heads of 128 entries with the rows written back (149 MB) 30.2 us, 76 % of the copy rate (one key per entry that
// orders magnitude, place and sign, and half words stored singly: 38; packed maxima: 33).
#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "quant4.cuh"

namespace hb {
namespace {

constexpr int kThreads = 256;

// Eight entries and their group's scale: the eight codes as bytes of two words (entry i in byte i), the scale, and the entries as the cache stands for them
struct Coded {
  uint32_t lo, hi;
  bf16 scale;
};

__device__ __forceinline__ uint32_t max_bf16x2(uint32_t a, uint32_t b) {  // NaN if either is
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2_down(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// All four lanes of a group call it with their eight entries
template <bool SEEN>
__device__ __forceinline__ Coded encode(const uint4 raw, int quarter, uint4& seen) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  // the largest of the entries and of their negatives, as two halves
  const uint32_t p = max_bf16x2(max_bf16x2(w[0], w[1]), max_bf16x2(w[2], w[3]));
  const uint32_t q = max_bf16x2(max_bf16x2(w[0] ^ 0x80008000u, w[1] ^ 0x80008000u), max_bf16x2(w[2] ^ 0x80008000u, w[3] ^ 0x80008000u));
  uint32_t pq = max_bf16x2(__byte_perm(p, q, 0x5410), __byte_perm(p, q, 0x7632));
  pq = max_bf16x2(pq, __shfl_xor_sync(0xffffffffu, pq, 1));
  pq = max_bf16x2(pq, __shfl_xor_sync(0xffffffffu, pq, 2));
  const float up = __uint_as_float(pq << 16), dn = __uint_as_float(pq & 0xffff0000u);
  float m = up > dn ? up : -dn;
  if (up == dn) {  // both signs reach it (or all is zero): the first entry says which; the other lanes of the group are here too
    uint32_t key = 0;  // 31 - place | sign
#pragma unroll
    for (int i = 7; i >= 0; --i) {
      const uint32_t u = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
      if ((u & 0x7fffu) == (pq & 0x7fffu)) key = (uint32_t)(31 - 8 * quarter - i) << 1 | u >> 15;
    }
    const uint32_t four = 0xfu << (threadIdx.x & 28);
    key = max(key, __shfl_xor_sync(four, key, 1));
    key = max(key, __shfl_xor_sync(four, key, 2));
    m = key & 1 ? -up : up;
  }
  Coded c;
  c.scale = __float2bfloat16(m * -0.125f);
  const float d = __bfloat162float(c.scale);
  // x / d as x (1 / d).  With eight bits each, a quotient that is no half integer is at least 2^-9 from one, while product and sum are off by less
  // than 2^-18: 2^-16 more puts every half integer itself on its upper side and moves nothing else.  1 / d of a tiny d would overflow: both are
  // raised first.  x / d + 8.5 is above 0 where the scale is rounded by 2^-8 at most, so that only subnormal ones need the lower end; adding 2^23
  // towards zero leaves the whole part in the low bits.
  constexpr float kHalf = 8.5f + 1.52587890625e-5f, kWhole = 8388608.f;
  uint32_t b[8];
  uint64_t y[4];
  if (fabsf(d) < 1e-30f) {
    const float raise = 1.8446744e19f, inv = 1.f / (d * raise);  // 2^64
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f[2];
#pragma unroll
      for (int o = 0; o < 2; ++o) {
        const float x = __uint_as_float(o ? w[i] & 0xffff0000u : w[i] << 16) * raise;
        f[o] = fmaxf(fminf(fmaf(x, inv, kHalf), 15.5f), 0.f);
      }
      y[i] = add2_down(f2_pack(f[0], f[1]), f2_pack(kWhole, kWhole));
    }
  } else {
    const float inv = 1.f / d;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f0, f1;
      f2_unpack(f2_fma(f2_pack(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u)), f2_pack(inv, inv), f2_pack(kHalf, kHalf)), f0, f1);
      y[i] = add2_down(f2_pack(fminf(f0, 15.5f), fminf(f1, 15.5f)), f2_pack(kWhole, kWhole));
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float f0, f1;
    f2_unpack(y[i], f0, f1);
    b[2 * i] = __float_as_uint(f0);
    b[2 * i + 1] = __float_as_uint(f1);
  }
  c.lo = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  c.hi = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  if (SEEN) {
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float f0, f1;
      f2_unpack(f2_mul(f2_add(y[i], f2_pack(-kWhole - 8.f, -kWhole - 8.f)), f2_pack(d, d)), f0, f1);
      u[i] = pack_bf16x2(f0, f1);
    }
    seen = make_uint4(u[0], u[1], u[2], u[3]);
  }
  const bool none = !(fabsf(m) < INFINITY);
  if (d == 0.f || none) {
    c.lo = c.hi = 0x08080808u;
    if (SEEN) seen = none ? make_uint4(0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu) : make_uint4(0, 0, 0, 0);
    if (none) c.scale = __ushort_as_bfloat16(0x7fffu);
  }
  return c;
}

template <int D, bool SEEN>
__global__ void __launch_bounds__(kThreads) kv_write_q4_kernel(const CacheWriteQ4Args a) {
  constexpr int LANES = D / 8, J = D / q4::kGroup, PART = D / 8;  // threads per row, groups, bytes of a quarter or chunk
  pdl_wait();
  pdl_launch_dependents();
  // A block takes tokens of one head in a row, pairs shifted by the first slot's parity: two tokens that share the words of values are then usually
  // neighbours in a warp and put their half words together
  const int lane = threadIdx.x % LANES, j = lane >> 2, quarter = lane & 3, h = blockIdx.y;
  const long long token = (long long)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES - (a.slots[0] & 1);
  const bool live = token >= 0 && token < a.T;
  const int t = (int)min(max(token, 0ll), (long long)a.T - 1);  // (threads without a row repeat one without storing: the exchange wants whole warps)
  const size_t col = (size_t)h * D + lane * 8;
  const uint4 kraw = *reinterpret_cast<const uint4*>(a.k + (size_t)t * a.ldk + col);
  const uint4 vraw = *reinterpret_cast<const uint4*>(a.v + (size_t)t * a.ldv + col);
  const int slot = a.slots[t];
  uint4 k_seen, v_seen;
  const Coded k = encode<SEEN>(kraw, quarter, k_seen), v = encode<SEEN>(vraw, quarter, v_seen);
  // values: entries 4 c + r in nibble r of a half word, c = 0, 1
  const uint32_t v2 = v.lo | v.lo >> 4, v3 = v.hi | v.hi >> 4;
  const uint32_t halves = __byte_perm(v2, v3, 0x6420);
  const bool stored = live && slot >= 0 && slot < a.num_pages * q4::kPage;
  const uint32_t theirs = __shfl_xor_sync(0xffffffffu, halves, LANES);
  const int their_slot = __shfl_xor_sync(0xffffffffu, stored ? slot : -2, LANES);
  if (!live) return;
  if (stored) {
    const int page = (int)((unsigned)slot / q4::kPage), pos = slot & (q4::kPage - 1);
    const size_t block = ((size_t)page * a.Hkv + h) * q4::block_bytes(D);
    // keys: even entries in nibbles 0..3, odd ones in 4..7
    const uint32_t even = __byte_perm(k.lo, k.hi, 0x6420), odd = __byte_perm(k.lo, k.hi, 0x7531);
    const uint32_t e2 = even | even >> 4, o2 = odd | odd >> 4;  // bytes 0 and 2: two codes each
    *reinterpret_cast<uint32_t*>(a.k_cache + block + pos * (D / 2) + quarter * PART + j * 4) = __byte_perm(e2, o2, 0x6420);
    const int pair = pos >> 1, x = q4::place_xor(D, pair);
    uint8_t* words = a.v_cache + block + pair * D + j * 4;
    if (their_slot == (slot ^ 1) && (slot & 1) == (int)(threadIdx.x / LANES & 1)) {  // a word each
      const uint32_t odd = slot & 1, even_half = odd ? theirs >> 16 : halves & 0xffffu, odd_half = odd ? halves & 0xffff0000u : theirs << 16;
      *reinterpret_cast<uint32_t*>(words + ((2 * quarter + odd) ^ x) * PART) = even_half | odd_half;
    } else {
      uint8_t* mine = words + (pos & 1) * 2;
      *reinterpret_cast<uint16_t*>(mine + ((2 * quarter) ^ x) * PART) = (uint16_t)halves;
      *reinterpret_cast<uint16_t*>(mine + ((2 * quarter + 1) ^ x) * PART) = (uint16_t)(halves >> 16);
    }
    if (quarter == 0) {
      const size_t at = block + q4::code_bytes(D) + (pos * J + j) * 2;
      *reinterpret_cast<bf16*>(a.k_cache + at) = k.scale;
      *reinterpret_cast<bf16*>(a.v_cache + at) = v.scale;
    }
  }
  if (SEEN) {
    if (a.k_seen) *reinterpret_cast<uint4*>(a.k_seen + (size_t)t * a.ldks + col) = k_seen;
    if (a.v_seen) *reinterpret_cast<uint4*>(a.v_seen + (size_t)t * a.ldvs + col) = v_seen;
  }
}

bool rows_ok(const void* p, int ld, int need) { return ((uintptr_t)p & 15) == 0 && ld >= need && ld % 8 == 0; }

}  // namespace

size_t kv_q4_plane_bytes(int num_pages, int Hkv, int D) {
  return num_pages > 0 && Hkv > 0 && (D == 64 || D == 128) ? (size_t)num_pages * Hkv * q4::block_bytes(D) : 0;
}

cudaError_t kv_write_q4(cudaStream_t stream, const CacheWriteQ4Args& a) {
  if (a.T < 0 || a.Hkv < 1 || (a.D != 64 && a.D != 128) || a.page_size != q4::kPage || a.num_pages < 1 || a.num_pages > INT32_MAX / q4::kPage)
    return cudaErrorInvalidValue;
  if (a.T == 0) return cudaSuccess;
  if (a.Hkv > 65535 || !a.k || !a.v || !a.slots || !a.k_cache || !a.v_cache || ((uintptr_t)a.k_cache & 15) || ((uintptr_t)a.v_cache & 15)) return cudaErrorInvalidValue;
  const int need = a.Hkv * a.D;
  if (!rows_ok(a.k, a.ldk, need) || !rows_ok(a.v, a.ldv, need) || (a.k_seen && !rows_ok(a.k_seen, a.ldks, need)) || (a.v_seen && !rows_ok(a.v_seen, a.ldvs, need)))
    return cudaErrorInvalidValue;
  const int rows = kThreads / (a.D / 8);  // of a block; one token more, where pairs are shifted
  const unsigned blocks = (unsigned)(((long long)a.T + 1 + rows - 1) / rows);
  const bool seen = a.k_seen || a.v_seen;
  return launch_k(a.D == 128 ? seen ? kv_write_q4_kernel<128, true> : kv_write_q4_kernel<128, false> : seen ? kv_write_q4_kernel<64, true> : kv_write_q4_kernel<64, false>,
                  dim3(blocks, a.Hkv), dim3(kThreads), 0, stream, true, a);
}

}  // namespace hb

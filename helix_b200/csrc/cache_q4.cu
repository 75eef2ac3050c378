// Rows of a step written into a 4-bit paged cache (layout: quant4.cuh).
//
// A group of 32 entries: m = the entry of largest magnitude (the first of equals), d = bf16(m / -8), c = clamp(floor(x / d + 1/2) + 8, 0, 15), so that m
// itself gets code 0 and is kept to bf16's rounding; d = 0 gives code 8, and a group with an infinity or a NaN gets d = NaN: it reads as NaN.
// The scale is rounded before the codes are chosen, so they are the nearest ones for the scale that is stored.
//
// Eight entries per thread (one 16-byte load), four threads per group.  Their codes fill one word of the key layout and two half words of the
// value layout, so no thread needs another's codes and no byte is shared by two positions: rows of one page may be written by any threads in any order.
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
__device__ __forceinline__ float add_down(float a, float b) {
  float r;
  asm("add.rz.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
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
  const bool tiny = fabsf(d) < 1e-30f;
  const float raise = tiny ? 1.8446744e19f : 1.f;  // 2^64
  const float inv = 1.f / (d * raise);
  uint32_t b[8];
  float y[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float x = __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
    if (tiny) x *= raise;
    float f = fminf(fmaf(x, inv, 8.5f + 1.52587890625e-5f), 15.5f);
    if (tiny) f = fmaxf(f, 0.f);
    f = add_down(f, 8388608.f);
    b[i] = __float_as_uint(f);
    if (SEEN) y[i] = (f - 8388616.f) * d;
  }
  c.lo = __byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410);
  c.hi = __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410);
  if (SEEN) seen = make_uint4(pack_bf16x2(y[0], y[1]), pack_bf16x2(y[2], y[3]), pack_bf16x2(y[4], y[5]), pack_bf16x2(y[6], y[7]));
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
  const size_t id = (size_t)blockIdx.x * kThreads + threadIdx.x;
  const size_t rows = (size_t)a.T * a.Hkv;
  const size_t row = min(id / LANES, rows - 1);  // (threads behind the last row repeat it without storing: the exchange wants whole warps)
  const bool live = id / LANES < rows;
  const int lane = (int)(id % LANES), j = lane >> 2, quarter = lane & 3;
  const int t = (int)(row / a.Hkv), h = (int)(row % a.Hkv);
  const size_t col = (size_t)h * D + lane * 8;
  const uint4 kraw = *reinterpret_cast<const uint4*>(a.k + (size_t)t * a.ldk + col);
  const uint4 vraw = *reinterpret_cast<const uint4*>(a.v + (size_t)t * a.ldv + col);
  const int slot = a.slots[t];
  uint4 k_seen, v_seen;
  const Coded k = encode<SEEN>(kraw, quarter, k_seen), v = encode<SEEN>(vraw, quarter, v_seen);
  if (!live) return;
  if (slot >= 0 && slot < a.num_pages * q4::kPage) {
    const int page = slot / q4::kPage, pos = slot % q4::kPage;
    const size_t block = ((size_t)page * a.Hkv + h) * q4::block_bytes(D);
    // keys: even entries in nibbles 0..3, odd ones in 4..7
    const uint32_t even = __byte_perm(k.lo, k.hi, 0x6420), odd = __byte_perm(k.lo, k.hi, 0x7531);
    const uint32_t e2 = even | even >> 4, o2 = odd | odd >> 4;  // bytes 0 and 2: two codes each
    *reinterpret_cast<uint32_t*>(a.k_cache + block + pos * (D / 2) + quarter * PART + j * 4) = __byte_perm(e2, o2, 0x6420);
    // values: entries 4 c + r in nibble r
    const uint32_t v2 = v.lo | v.lo >> 4, v3 = v.hi | v.hi >> 4;
    const int pair = pos >> 1;
    uint8_t* row = a.v_cache + block + pair * D + j * 4 + (pos & 1) * 2;
    const int x = q4::place_xor(D, pair);
    *reinterpret_cast<uint16_t*>(row + ((2 * quarter) ^ x) * PART) = (uint16_t)__byte_perm(v2, 0, 0x4420);
    *reinterpret_cast<uint16_t*>(row + ((2 * quarter + 1) ^ x) * PART) = (uint16_t)__byte_perm(v3, 0, 0x4420);
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
  if ((long long)a.Hkv * a.D > INT32_MAX || !a.k || !a.v || !a.slots || !a.k_cache || !a.v_cache || ((uintptr_t)a.k_cache & 15) || ((uintptr_t)a.v_cache & 15)) return cudaErrorInvalidValue;
  const int need = a.Hkv * a.D;
  if (!rows_ok(a.k, a.ldk, need) || !rows_ok(a.v, a.ldv, need) || (a.k_seen && !rows_ok(a.k_seen, a.ldks, need)) || (a.v_seen && !rows_ok(a.v_seen, a.ldvs, need)))
    return cudaErrorInvalidValue;
  const size_t blocks = ((size_t)a.T * a.Hkv * (a.D / 8) + kThreads - 1) / kThreads;
  if (blocks > INT32_MAX) return cudaErrorInvalidValue;
  const bool seen = a.k_seen || a.v_seen;
  return launch_k(a.D == 128 ? seen ? kv_write_q4_kernel<128, true> : kv_write_q4_kernel<128, false> : seen ? kv_write_q4_kernel<64, true> : kv_write_q4_kernel<64, false>,
                  dim3((unsigned)blocks), dim3(kThreads), 0, stream, true, a);
}

}  // namespace hb

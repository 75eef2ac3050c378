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

struct Coded {
  uint32_t code[8];
  bf16 scale;
};

// All four lanes of a group call it with their eight entries
__device__ __forceinline__ Coded encode(const uint4 raw, int quarter) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  // magnitude | 31 - place | sign: the largest key names the first entry of largest magnitude (an entry's 15 magnitude bits order as integers)
  uint32_t key = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = (w[i >> 1] >> (16 * (i & 1))) & 0xffffu;
    key = max(key, (u & 0x7fffu) << 6 | (uint32_t)(31 - 8 * quarter - i) << 1 | u >> 15);
  }
  key = max(key, __shfl_xor_sync(0xffffffffu, key, 1));
  key = max(key, __shfl_xor_sync(0xffffffffu, key, 2));
  const uint32_t mag = key >> 6;
  const float m = __uint_as_float(mag << 16 | (key & 1u) << 31);
  Coded c;
  c.scale = __float2bfloat16(m * -0.125f);
  const float d = __bfloat162float(c.scale);
  // x / d as x (1 / d).  With eight bits each, a quotient that is no half integer is at least 2^-9 from one, while product and sum are off by less
  // than 2^-18: 2^-16 more puts every half integer itself on its upper side and moves nothing else.  1 / d of a tiny d would overflow: both are raised first.
  const float up = fabsf(d) < 1e-30f ? 1.8446744e19f : 1.f;  // 2^64
  const float inv = 1.f / (d * up);
  const bool zero = d == 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t u = (w[i >> 1] >> (16 * (i & 1))) << 16;
    const float x = __uint_as_float(u) * up;
    const float f = fminf(fmaxf(floorf(fmaf(x, inv, 8.5f + 1.52587890625e-5f)), 0.f), 15.f);
    c.code[i] = zero ? 8u : (uint32_t)f;
  }
  if (mag >= 0x7f80u) c.scale = __ushort_as_bfloat16(0x7fffu);
  return c;
}
__device__ __forceinline__ uint4 decoded(const Coded& c) {
  const float d = __bfloat162float(c.scale);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(d * (float)((int)c.code[2 * i] - 8), d * (float)((int)c.code[2 * i + 1] - 8));
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int D>
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
  const Coded k = encode(kraw, quarter), v = encode(vraw, quarter);
  if (!live) return;
  if (slot >= 0 && slot < a.num_pages * q4::kPage) {
    const int page = slot / q4::kPage, pos = slot % q4::kPage;
    const size_t block = ((size_t)page * a.Hkv + h) * q4::block_bytes(D);
    uint32_t kw = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) kw |= k.code[i] << (4 * (i / 2 + 4 * (i & 1)));
    *reinterpret_cast<uint32_t*>(a.k_cache + block + pos * (D / 2) + quarter * PART + j * 4) = kw;
    const int pair = pos >> 1;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int place = (2 * quarter + c) ^ q4::place_xor(D, pair);
      const uint32_t hw = v.code[4 * c] | v.code[4 * c + 1] << 4 | v.code[4 * c + 2] << 8 | v.code[4 * c + 3] << 12;
      *reinterpret_cast<uint16_t*>(a.v_cache + block + pair * D + place * PART + j * 4 + (pos & 1) * 2) = (uint16_t)hw;
    }
    if (quarter == 0) {
      const size_t at = block + q4::code_bytes(D) + (pos * J + j) * 2;
      *reinterpret_cast<bf16*>(a.k_cache + at) = k.scale;
      *reinterpret_cast<bf16*>(a.v_cache + at) = v.scale;
    }
  }
  if (a.k_seen) *reinterpret_cast<uint4*>(a.k_seen + (size_t)t * a.ldks + col) = decoded(k);
  if (a.v_seen) *reinterpret_cast<uint4*>(a.v_seen + (size_t)t * a.ldvs + col) = decoded(v);
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
  return launch_k(a.D == 128 ? kv_write_q4_kernel<128> : kv_write_q4_kernel<64>, dim3((unsigned)blocks), dim3(kThreads), 0, stream, true, a);
}

}  // namespace hb

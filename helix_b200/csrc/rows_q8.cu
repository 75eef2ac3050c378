// Rows of bf16 or fp32 to 8-bit codes with a scale each: s = max |x| / 127, c = the whole number nearest to x / s.
//
// One pass: a row stays in its threads' registers between the maximum and the codes (rows longer than that are read again from L2).  Bytes bound it: 2 or 4 in, 1 out,
// 2 more where the rows are wanted as the codes stand for them.
#include <algorithm>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace hb {
namespace {

constexpr int E = 8;  // neighbouring entries of a thread: 16 bytes of bf16, 8 of codes

template <bool F32>
__device__ __forceinline__ void load_entries(const void* row, int i, int K, float (&f)[E]) {
  if (i + E <= K) {
    if constexpr (F32) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(row) + i)), b = __ldg(reinterpret_cast<const float4*>(static_cast<const float*>(row) + i) + 1);
      f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
    } else {
      unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const bf16*>(row) + i), f);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      f[e] = i + e < K ? (F32 ? static_cast<const float*>(row)[i + e] : __bfloat162float(static_cast<const bf16*>(row)[i + e])) : 0.f;
  }
}

// c for one entry.  x times the rounded 1 / s is off by at most 127 * 2^-23 < 2^-16: only quotients that lie within that of the middle of two codes need more, and there the
// products in 64 bits are exact (8 + 24 bits).  Nearly no entry goes there.
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  const float q = x * inv, r = rintf(q);
  int c = (int)r;
  if (fabsf(q - r) > 0.5f - 0x1p-15f) {
    const float lower = floorf(fabsf(q));  // (the middle is lower + 1/2: no quotient this near to it has another whole part)
    const double d = (double)fabsf(x) - ((double)lower + 0.5) * (double)s;
    const int n = (int)lower;
    const int m = d > 0.0 ? n + 1 : d < 0.0 ? n : n + (n & 1);
    c = x < 0.f ? -m : m;
  }
  return max(-127, min(127, c));
}
// where 1 / s has no normal fp32 value: the quotient in 64 bits (24 + 24 bits: what is not the middle is 2^-48 from it at least)
__device__ __noinline__ int code_of_small(float x, float s) { return max(-127, min(127, (int)rint((double)x / (double)s))); }

template <bool F32, int WARPS, int CH>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) rows_q8_kernel(const RowsQ8Args a) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int STEP = WARPS * 32 * E;  // entries of a row that its threads take at a time
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = WARPS == 1 ? blockIdx.x * 4 + warp : blockIdx.x;
  const int at = (WARPS == 1 ? lane : (int)threadIdx.x) * E;
  if (t >= a.T) return;  // (whole warps where a row has one, else nobody)
  const void* row = static_cast<const uint8_t*>(a.x) + (size_t)t * a.ldx * (F32 ? 4 : 2);
  float f[CH][E];
  uint32_t top = 0;  // of the magnitudes' bits, which are ordered as the magnitudes are, infinities and NaN above all
  auto look = [&](const float(&v)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
  };
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    load_entries<F32>(row, min(c * STEP + at, a.K), a.K, f[c]);
  }
#pragma unroll
  for (int c = 0; c < CH; ++c) look(f[c]);
  for (int i = CH * STEP + at; i < a.K; i += STEP) {
    float v[E];
    load_entries<F32>(row, i, a.K, v);
    look(v);
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (WARPS > 1) {
    __shared__ uint32_t tops[WARPS];
    if (lane == 0) tops[warp] = top;
    __syncthreads();
    top = __reduce_max_sync(0xffffffffu, lane < WARPS ? tops[lane] : 0u);
  }
  const float s = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7fffffffu);
  const bool live = s > 0.f, small = s < 0x1p-100f;
  const float inv = live ? __frcp_rn(s) : 0.f;
  if (at == 0) a.scales[t] = s;
  int8_t* codes = a.codes + (size_t)t * a.ldc;
  bf16* seen = a.seen ? a.seen + (size_t)t * a.lds : nullptr;
  auto write = [&](int i, const float(&v)[E]) {
    if (i >= a.K) return;
    int c[E];
    if (!live) {
#pragma unroll
      for (int e = 0; e < E; ++e) c[e] = 0;
    } else if (small) {
#pragma unroll
      for (int e = 0; e < E; ++e) c[e] = code_of_small(v[e], s);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) c[e] = code_of(v[e], s, inv);
    }
    if (i + E <= a.K) {
      uint2 o;
      o.x = (c[0] & 255) | (c[1] & 255) << 8 | (c[2] & 255) << 16 | (uint32_t)c[3] << 24;
      o.y = (c[4] & 255) | (c[5] & 255) << 8 | (c[6] & 255) << 16 | (uint32_t)c[7] << 24;
      *reinterpret_cast<uint2*>(codes + i) = o;
      if (seen) {
        uint4 w;
        w.x = pack_bf16x2(s * (float)c[0], s * (float)c[1]);
        w.y = pack_bf16x2(s * (float)c[2], s * (float)c[3]);
        w.z = pack_bf16x2(s * (float)c[4], s * (float)c[5]);
        w.w = pack_bf16x2(s * (float)c[6], s * (float)c[7]);
        *reinterpret_cast<uint4*>(seen + i) = w;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < a.K) {
          codes[i + e] = (int8_t)c[e];
          if (seen) seen[i + e] = __float2bfloat16(s * (float)c[e]);
        }
    }
  };
#pragma unroll
  for (int c = 0; c < CH; ++c) write(c * STEP + at, f[c]);
  for (int i = CH * STEP + at; i < a.K; i += STEP) {
    float v[E];
    load_entries<F32>(row, i, a.K, v);
    write(i, v);
  }
}

template <bool F32>
cudaError_t launch_rows(cudaStream_t stream, const RowsQ8Args& a) {
  if (a.K <= 1024) return launch_k(rows_q8_kernel<F32, 1, 4>, dim3((a.T + 3) / 4), dim3(128), 0, stream, true, a);
  if (a.K <= 4096) return launch_k(rows_q8_kernel<F32, 4, 4>, dim3(a.T), dim3(128), 0, stream, true, a);
  if (a.K <= 8192) return launch_k(rows_q8_kernel<F32, 8, 4>, dim3(a.T), dim3(256), 0, stream, true, a);
  return launch_k(rows_q8_kernel<F32, 16, 4>, dim3(a.T), dim3(512), 0, stream, true, a);
}

}  // namespace

cudaError_t rows_q8(cudaStream_t stream, const RowsQ8Args& a) {
  if (a.T < 0 || a.K < 1 || a.K > INT32_MAX - 65536) return cudaErrorInvalidValue;  // (steps past the last entry stay within 32 bits)
  if (a.T == 0) return cudaSuccess;
  if (!a.x || ((uintptr_t)a.x & 15) || a.ldx < a.K || a.ldx % 8 || !a.codes || ((uintptr_t)a.codes & 15) || a.ldc < a.K || a.ldc % 16 || !a.scales || ((uintptr_t)a.scales & 3) ||
      (a.seen && (((uintptr_t)a.seen & 15) || a.lds < a.K || a.lds % 8)))
    return cudaErrorInvalidValue;
  return a.x_f32 ? launch_rows<true>(stream, a) : launch_rows<false>(stream, a);
}

}  // namespace hb

// Rows of bf16 or fp32 to 8-bit codes with a scale each: s = max |x| / 127, c = the whole number nearest to x / s.
//
// One pass: a row stays in its threads' registers between the maximum and the codes (rows longer than that are read again from L2).  Bytes bound it: 2 or 4 in, 1 out,
// 2 more where the rows are wanted as the codes stand for them.
#include <algorithm>
#include <atomic>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace hb {
namespace {

template <bool F32>
constexpr int kPiece = F32 ? 4 : 8;  // neighbouring entries of a thread: 16 bytes

// A piece as it lies in memory, zeros behind the last entry
template <bool F32>
__device__ __forceinline__ uint4 load_piece(const void* row, int i, int K) {
  constexpr int E = kPiece<F32>;
  if (i + E <= K) return *reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(row) + (size_t)i * (F32 ? 4 : 2));
  uint32_t u[4] = {0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (i + e < K) {
      if constexpr (F32) u[e] = static_cast<const uint32_t*>(row)[i + e];
      else u[e / 2] |= (uint32_t) static_cast<const uint16_t*>(row)[i + e] << (16 * (e & 1));
    }
  return make_uint4(u[0], u[1], u[2], u[3]);
}
template <bool F32, int E = kPiece<F32>>
__device__ __forceinline__ void entries_of(const uint4& u, float (&f)[E]) {
  if constexpr (F32) {
    f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
  } else {
    unpack_bf16x8(u, f);
  }
}
__device__ __forceinline__ float max3_nan(float a, float b, float c) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The whole number nearest to x / s where x times the rounded 1 / s lies within 2^-15 of the middle of two (that product is off by 127 * 2^-24 at most: elsewhere it decides
// alone).  The products in 64 bits are exact (8 + 24 bits).  Nearly no entry comes here.
__device__ __noinline__ float near_middle(float x, float s, float inv) {
  const float lower = floorf(fabsf(x * inv));  // (no quotient this near to the middle has another whole part)
  const double d = (double)fabsf(x) - ((double)lower + 0.5) * (double)s;
  const int n = (int)lower;
  const int m = d > 0.0 ? n + 1 : d < 0.0 ? n : n + (n & 1);
  return x < 0.f ? -(float)m : (float)m;
}
// where 1 / s has no normal fp32 value: the quotient in 64 bits (24 + 24 bits: what is not the middle is 2^-48 from it at least)
__device__ __noinline__ float of_small(float x, float s) { return (float)fmax(-127.0, fmin(127.0, rint((double)x / (double)s))); }

// The largest magnitude of a thread's entries, NaN if one is
template <bool F32>
struct Top {
  float top = 0.f;
  uint32_t two = 0;
  __device__ __forceinline__ void look(const uint4& u) {
    if constexpr (F32) {
      top = max3_nan(top, fabsf(__uint_as_float(u.x)), fabsf(__uint_as_float(u.y)));
      top = max3_nan(top, fabsf(__uint_as_float(u.z)), fabsf(__uint_as_float(u.w)));
    } else {
      constexpr uint32_t kAbs = 0x7fff7fffu;
      two = max_nan_bf16x2(max_nan_bf16x2(max_nan_bf16x2(two, u.x & kAbs), max_nan_bf16x2(u.y & kAbs, u.z & kAbs)), u.w & kAbs);
    }
  }
  // of the row's WARPS warps (magnitudes are ordered as their bits are, NaN above all)
  template <int WARPS>
  __device__ __forceinline__ uint32_t of_row(uint32_t* tops) {
    if constexpr (!F32) {
      const float2 f = unpack_bf16x2(two);
      top = max3_nan(top, f.x, f.y);
    }
    uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if constexpr (WARPS > 1) {
      const int lane = threadIdx.x & 31;
      if (lane == 0) tops[threadIdx.x >> 5] = bits;
      __syncthreads();
      bits = __reduce_max_sync(0xffffffffu, lane < WARPS ? tops[lane] : 0u);
    }
    return bits;
  }
};

struct Row {
  float s, inv;
  bool live, small;
  int8_t* codes;
  bf16* seen;
  __device__ __forceinline__ Row(const RowsQ8Args& a, int t, uint32_t top) {
    s = top < 0x7f800000u ? __fdiv_rn(__uint_as_float(top), 127.f) : __uint_as_float(0x7fffffffu);
    live = s > 0.f;
    small = s < 0x1p-100f;
    inv = live && !small ? __frcp_rn(s) : 0.f;
    codes = a.codes + (size_t)t * a.ldc;
    seen = a.seen ? a.seen + (size_t)t * a.lds : nullptr;
  }
};

// Codes, and what they stand for, of the piece from entry i on
template <bool F32>
__device__ __forceinline__ void write_piece(const Row& r, int i, int K, const uint4& u) {
  constexpr int E = kPiece<F32>;
  int8_t* codes = r.codes;
  bf16* seen = r.seen;
  float v[E];
  entries_of<F32>(u, v);
  // adding 3 * 2^22 rounds to a whole number, whose low byte is the code
  constexpr float kWhole = 12582912.f;
  const uint64_t inv2 = f2_pack(r.inv, r.inv), up = f2_pack(kWhole, kWhole), down = f2_pack(-kWhole, -kWhole), minus = f2_pack(-1.f, -1.f);
  float w[E], far = 0.f;  // the code with its 3 * 2^22
#pragma unroll
  for (int e = 0; e < E; e += 2) {
    const uint64_t x = f2_pack(v[e], v[e + 1]), y = f2_fma(x, inv2, up), whole = f2_add(y, down), off = f2_fma(x, inv2, f2_mul(whole, minus));
    float o0, o1;
    f2_unpack(off, o0, o1);
    f2_unpack(y, w[e], w[e + 1]);
    far = max3_nan(far, fabsf(o0), fabsf(o1));
  }
  if (!r.live || r.small || !(far <= 0.5f - 0x1p-15f)) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (!r.live) w[e] = kWhole;
      else if (r.small) w[e] = kWhole + of_small(v[e], r.s);
      else if (fabsf(fmaf(v[e], r.inv, kWhole - w[e])) > 0.5f - 0x1p-15f) w[e] = kWhole + near_middle(v[e], r.s, r.inv);
    }
  }
  if (i + E <= K) {
    uint32_t o[E / 4];
#pragma unroll
    for (int e = 0; e < E; e += 4)
      o[e / 4] = __byte_perm(__byte_perm(__float_as_uint(w[e]), __float_as_uint(w[e + 1]), 0x0040), __byte_perm(__float_as_uint(w[e + 2]), __float_as_uint(w[e + 3]), 0x0040), 0x5410);
    if constexpr (E == 8) *reinterpret_cast<uint2*>(codes + i) = make_uint2(o[0], o[1]);
    else *reinterpret_cast<uint32_t*>(codes + i) = o[0];
    if (seen) {
      uint32_t u[E / 2];
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        float x0, x1;
        f2_unpack(f2_mul(f2_add(f2_pack(w[e], w[e + 1]), down), f2_pack(r.s, r.s)), x0, x1);
        u[e / 2] = pack_bf16x2(x0, x1);
      }
      if constexpr (E == 8) *reinterpret_cast<uint4*>(seen + i) = make_uint4(u[0], u[1], u[2], u[3]);
      else *reinterpret_cast<uint2*>(seen + i) = make_uint2(u[0], u[1]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (i + e < K) {
        codes[i + e] = (int8_t)__float_as_uint(w[e]);
        if (seen) seen[i + e] = __float2bfloat16(r.s * (w[e] - kWhole));
      }
  }
}

template <bool F32, int WARPS, int CH>
__global__ void __launch_bounds__(WARPS == 1 ? 128 : WARPS * 32) rows_q8_kernel(const RowsQ8Args a) {
  pdl_wait();
  pdl_launch_dependents();
  constexpr int STEP = WARPS * 32 * kPiece<F32>;  // entries of a row that its threads take at a time
  __shared__ uint32_t tops[WARPS];
  const int t = WARPS == 1 ? blockIdx.x * 4 + (threadIdx.x >> 5) : blockIdx.x;
  const int at = (WARPS == 1 ? (int)threadIdx.x & 31 : (int)threadIdx.x) * kPiece<F32>;
  if (t >= a.T) return;  // (whole warps where a row has one, else nobody)
  const void* row = static_cast<const uint8_t*>(a.x) + (size_t)t * a.ldx * (F32 ? 4 : 2);
  uint4 x[CH];
  Top<F32> top;
#pragma unroll
  for (int c = 0; c < CH; ++c) x[c] = load_piece<F32>(row, min(c * STEP + at, a.K), a.K);
#pragma unroll
  for (int c = 0; c < CH; ++c) top.look(x[c]);
  for (int i = CH * STEP + at; i < a.K; i += STEP) top.look(load_piece<F32>(row, i, a.K));
  const Row r(a, t, top.template of_row<WARPS>(tops));
  if (at == 0) a.scales[t] = r.s;
#pragma unroll
  for (int c = 0; c < CH; ++c)
    if (c * STEP + at < a.K) write_piece<F32>(r, c * STEP + at, a.K, x[c]);
  for (int i = CH * STEP + at; i < a.K; i += STEP) write_piece<F32>(r, i, a.K, load_piece<F32>(row, i, a.K));
}

// Long rows, one after the other: few blocks find room on an SM, so each has its next row on the way (into its threads' own places in shared memory) while it works on one
template <bool F32, int WARPS, int CH>
__global__ void __launch_bounds__(WARPS * 32) rows_q8_ring_kernel(const RowsQ8Args a) {
  constexpr int E = kPiece<F32>, THREADS = WARPS * 32, STEP = THREADS * E;
  extern __shared__ uint4 ring[];  // [2][CH][THREADS]
  __shared__ uint32_t tops[2][WARPS];
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, at = tid * E;
  auto row_of = [&](int t) { return static_cast<const uint8_t*>(a.x) + (size_t)t * a.ldx * (F32 ? 4 : 2); };
  auto fetch = [&](long long t, int half) {
    if (t < a.T) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (c * STEP + at + E <= a.K)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(ring + (half * CH + c) * THREADS + tid)), "l"(row_of((int)t) + (size_t)(c * STEP + at) * (F32 ? 4 : 2))
                       : "memory");
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  fetch(blockIdx.x, 0);
  int half = 0;
  for (long long t = blockIdx.x; t < a.T; t += gridDim.x, half ^= 1) {
    fetch(t + gridDim.x, half ^ 1);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    const void* row = row_of((int)t);
    auto piece = [&](int c) {
      const int i = c * STEP + at;
      return i + E <= a.K ? ring[(half * CH + c) * THREADS + tid] : load_piece<F32>(row, min(i, a.K), a.K);
    };
    Top<F32> top;
#pragma unroll
    for (int c = 0; c < CH; ++c) top.look(piece(c));
    const Row r(a, (int)t, top.template of_row<WARPS>(tops[half]));
    if (tid == 0) a.scales[t] = r.s;
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (c * STEP + at < a.K) write_piece<F32>(r, c * STEP + at, a.K, piece(c));
  }
}

template <bool F32, int WARPS, int CH>
cudaError_t launch_ring(cudaStream_t stream, const RowsQ8Args& a, int sms) {
  constexpr int kRing = 2 * CH * WARPS * 32 * 16;
  static std::atomic<uint64_t> asked{0};  // more than 48 KB of shared memory wants to be asked for once per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(asked.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(rows_q8_ring_kernel<F32, WARPS, CH>, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing);
    if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  return launch_k(rows_q8_ring_kernel<F32, WARPS, CH>, dim3((unsigned)std::min<long long>(a.T, (long long)sms * std::max(1, 226 * 1024 / (kRing + 1024)))), dim3(WARPS * 32), kRing,
                  stream, true, a);
}

// A row's threads: as few warps as hold it in registers, 1024 entries each.  fp32 rows of more than 8192 entries, where there are more than the SMs take at a time: one after the
// other (4096 x 14336 91 -> 69 us; bf16 rows, half as long in bytes, 55 -> 63)
template <bool F32, int WARPS>
cudaError_t launch_rows(cudaStream_t stream, const RowsQ8Args& a, int sms) {
  if constexpr (WARPS < 16) {
    if (a.K > WARPS * 1024) return launch_rows<F32, (WARPS < 4 ? WARPS + 1 : WARPS + 2)>(stream, a, sms);
  }
  constexpr int CH = 1024 / (32 * kPiece<F32>);
  if constexpr (F32 && WARPS > 8) {
    if (a.K <= WARPS * 1024 && a.T > 4 * sms) return launch_ring<F32, WARPS, CH>(stream, a, sms);
  }
  return launch_k(rows_q8_kernel<F32, WARPS, CH>, dim3(WARPS == 1 ? (a.T + 3) / 4 : a.T), dim3(WARPS == 1 ? 128 : WARPS * 32), 0, stream, true, a);
}

}  // namespace

cudaError_t rows_q8(cudaStream_t stream, const RowsQ8Args& a) {
  if (a.T < 0 || a.T > (1 << 30) || a.K < 1 || a.K > (1 << 30)) return cudaErrorInvalidValue;
  if (a.T == 0) return cudaSuccess;
  if (!a.x || ((uintptr_t)a.x & 15) || a.ldx < a.K || a.ldx % 8 || !a.codes || ((uintptr_t)a.codes & 15) || a.ldc < a.K || a.ldc % 16 || !a.scales || ((uintptr_t)a.scales & 3) ||
      (a.seen && (((uintptr_t)a.seen & 15) || a.lds < a.K || a.lds % 8)))
    return cudaErrorInvalidValue;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return cudaErrorNoDevice;
  sms = effective_sms(sms);
  return a.x_f32 ? launch_rows<true, 1>(stream, a, sms) : launch_rows<false, 1>(stream, a, sms);
}

}  // namespace hb

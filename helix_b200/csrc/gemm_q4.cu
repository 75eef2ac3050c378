// Products of few rows with 4-bit weights: out[M, N] = x[M, K] W[N, K]^T, W in groups of 32 along K (code c stands for d (c - 8), d fp16).
//
// The bytes of the weights bound it (0.5625 per weight), so each is read once and goes straight from its load to a product's registers: a tile of
// 16 rows x 128 columns lies in memory as the 32 lanes take it (quant4.cuh, key-like rows), the 16-row operand of a warp-wide 16 x 8 x 16
// product is W, x the 8-column one.  c - 8 is exact in bf16; a group's products are summed by themselves and multiplied by d in fp32.
#include <algorithm>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "quant4.cuh"

namespace hb {
namespace {

constexpr int TN = 16, TK = 128;                       // a tile of weights
constexpr int TILE = TN * TK / 2 + TN * (TK / 32) * 2;  // its bytes: codes, then fp16 scales [row][group]
constexpr int kWarps = 8, kThreads = kWarps * 32;

// One block per 16 rows of W: its warps share the tiles along K
template <int NT>
__global__ void __launch_bounds__(kThreads) gemm_q4_kernel(const GemmQ4Args a) {
  constexpr int COLS = 8 * NT;
  __shared__ float s_sum[kWarps][TN][COLS + 1];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * TN, m0 = blockIdx.y * COLS;
  const int kt_all = (a.K + TK - 1) / TK;
  const uint8_t* w = a.w + (size_t)blockIdx.x * kt_all * TILE;
  float acc[NT][4] = {};
  for (int kt = warp; kt < kt_all; kt += kWarps) {
    const uint8_t* tile = w + (size_t)kt * TILE;
    const uint4 c0 = __ldg(reinterpret_cast<const uint4*>(tile + lane * 16)), c1 = __ldg(reinterpret_cast<const uint4*>(tile + 512 + lane * 16));
    const uint2 d0 = __ldg(reinterpret_cast<const uint2*>(tile + 1024 + g * 8)), d1 = __ldg(reinterpret_cast<const uint2*>(tile + 1024 + 64 + g * 8));
    const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int k = kt * TK + j * 32 + t * 8;
      const uint32_t u0 = j < 2 ? d0.x : d0.y, u1 = j < 2 ? d1.x : d1.y;
      const float s0 = __half2float(__ushort_as_half((unsigned short)(j & 1 ? u0 >> 16 : u0 & 0xffffu)));
      const float s1 = __half2float(__ushort_as_half((unsigned short)(j & 1 ? u1 >> 16 : u1 & 0xffffu)));
      uint32_t a0[4], a1[4];
      q4::codes_bf16(w0[j], a0);
      q4::codes_bf16(w1[j], a1);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int m = m0 + n * 8 + g;
        uint4 x = make_uint4(0, 0, 0, 0);
        if (m < a.M && k < a.K) x = *reinterpret_cast<const uint4*>(a.x + (size_t)m * a.ldx + k);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        q4::mma_bf16(c, a0[0], a1[0], a0[1], a1[1], x.x, x.y);
        q4::mma_bf16(c, a0[2], a1[2], a0[3], a1[3], x.z, x.w);
        acc[n][0] = fmaf(s0, c[0], acc[n][0]);
        acc[n][1] = fmaf(s0, c[1], acc[n][1]);
        acc[n][2] = fmaf(s1, c[2], acc[n][2]);
        acc[n][3] = fmaf(s1, c[3], acc[n][3]);
      }
    }
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) s_sum[warp][g + 8 * (i >> 1)][n * 8 + 2 * t + (i & 1)] = acc[n][i];
  __syncthreads();
  for (int i = threadIdx.x; i < TN * COLS; i += kThreads) {
    const int r = i % TN, c = i / TN, n = n0 + r, m = m0 + c;
    if (n >= a.N || m >= a.M) continue;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < kWarps; ++q) v += s_sum[q][r][c];
    if (a.bias) v += __bfloat162float(a.bias[n]);
    if (a.r) v += __bfloat162float(a.r[(size_t)m * a.ldr + n]);
    if (a.out_f32) reinterpret_cast<float*>(a.out)[(size_t)m * a.ldo + n] = v;
    else reinterpret_cast<bf16*>(a.out)[(size_t)m * a.ldo + n] = __float2bfloat16(v);
  }
}

// Blocks of a file ({fp16 d; 16 bytes}, byte i holding entries i and i + 16) to tiles: one thread per 16-byte quarter of a tile's row
__global__ void __launch_bounds__(256) gemm_q4_pack_kernel(const uint8_t* __restrict__ blocks, uint8_t* __restrict__ out, int N, int K, size_t total) {
  const size_t id = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= total) return;
  const int kt_all = (K + TK - 1) / TK, groups = K / 32;
  const int t = (int)(id & 3), r = (int)(id >> 2) & 15;
  const size_t tile = id >> 6;
  const int kt = (int)(tile % kt_all);
  const size_t n = tile / kt_all * TN + r;
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int grp = kt * 4 + j;
    const bool live = n < (size_t)N && grp < groups;
    const uint8_t* b = blocks + (n * groups + grp) * 18;
    w[j] = 0x88888888u;  // nothing there: codes of 0, and a scale of 0
    if (live) {
      w[j] = 0;
      for (int i = 0; i < 8; ++i) {
        const int e = 8 * t + i;
        const uint32_t c = e < 16 ? b[2 + e] & 15u : b[2 + e - 16] >> 4;
        w[j] |= c << (4 * (i / 2 + 4 * (i & 1)));
      }
    }
    if (t == j) *reinterpret_cast<uint16_t*>(out + tile * TILE + TN * TK / 2 + r * 8 + j * 2) = live ? (uint16_t)(b[0] | b[1] << 8) : (uint16_t)0;
  }
  *reinterpret_cast<uint4*>(out + tile * TILE + r * 64 + t * 16) = make_uint4(w[0], w[1], w[2], w[3]);
}

size_t tiles_of(int N, int K) { return (size_t)((N + TN - 1) / TN) * ((K + TK - 1) / TK); }
bool weights_ok(int N, int K) { return N >= 1 && K >= 32 && K % 32 == 0 && N <= INT32_MAX - TN && K <= INT32_MAX - TK; }

}  // namespace

size_t gemm_q4_bytes(int N, int K) { return weights_ok(N, K) ? tiles_of(N, K) * TILE : 0; }

cudaError_t gemm_q4_pack(cudaStream_t stream, const void* blocks, void* out, int N, int K) {
  if (!weights_ok(N, K) || !blocks || !out || ((uintptr_t)out & 15)) return cudaErrorInvalidValue;
  const size_t total = tiles_of(N, K) * TN * 4, grid = (total + 255) / 256;
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  gemm_q4_pack_kernel<<<(unsigned)grid, 256, 0, stream>>>(static_cast<const uint8_t*>(blocks), static_cast<uint8_t*>(out), N, K, total);
  return cudaGetLastError();
}

cudaError_t gemm_q4(cudaStream_t stream, const GemmQ4Args& a) {
  if (a.M < 0 || a.M > 256 || !weights_ok(a.N, a.K)) return cudaErrorInvalidValue;
  if (a.M == 0) return cudaSuccess;
  if (!a.x || !a.w || !a.out || ((uintptr_t)a.x & 15) || a.ldx < a.K || a.ldx % 8 || ((uintptr_t)a.w & 15) || a.ldo < a.N || ((uintptr_t)a.out & (a.out_f32 ? 3 : 1)) ||
      (a.r && (a.ldr < a.N || ((uintptr_t)a.r & 1))) || ((uintptr_t)a.bias & 1))
    return cudaErrorInvalidValue;
  const int nt = a.M <= 8 ? 1 : a.M <= 16 ? 2 : 4;
  const dim3 grid((a.N + TN - 1) / TN, (a.M + 8 * nt - 1) / (8 * nt));
  switch (nt) {
    case 1: return launch_k(gemm_q4_kernel<1>, grid, dim3(kThreads), 0, stream, true, a);
    case 2: return launch_k(gemm_q4_kernel<2>, grid, dim3(kThreads), 0, stream, true, a);
    default: return launch_k(gemm_q4_kernel<4>, grid, dim3(kThreads), 0, stream, true, a);
  }
}

}  // namespace hb

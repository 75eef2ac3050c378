// Products of few rows with 4-bit weights: out[M, N] = x[M, K] W[N, K]^T, W in groups of 32 along K (code c stands for d (c - 8), d fp16).
//
// The bytes of the weights bound it (0.5625 per weight).  A tile of 16 rows x 128 columns lies in memory as the 32 lanes take it (quant4.cuh, key-like
// rows); the 16-row operand of a warp-wide 16 x 8 x 16 product is W, x the 8-column one.  c - 8 is exact in bf16; a group's products are summed by
// themselves and multiplied by d in fp32.  16 rows x 32 columns for eight rows of x are some 32 instructions, where HBM gives an SM 50.
//
// A block owns 16 rows per warp; x passes through shared memory once for all its warps.  The blocks of a cluster share K and add their sums through
// distributed shared memory, in order: few rows of W still keep every SM reading, without a workspace or a second launch.
//
// Measured: 1 x 28672 x 4096 19 us (66 MB, 53 % of the copy rate; the same loads without the arithmetic 13), 8 x 4096 x 14336 13.7, 13 x 4096 x 14336 17,
// 32 x 28672 x 4096 41 (448 blocks on 148 SMs: four places carry 3.03; a third of that is the tail; half the products, no scales or no codes
// taken apart change it by less than a tenth each).  Also tried: eight warps along K per 16 rows (x read eight times: 85), x staged whole (58), shares of
// 5 to 8 warps (within 5 %), two tiles of rows per warp (47).
#include <algorithm>
#include <atomic>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"
#include "quant4.cuh"

namespace hb {
namespace {

constexpr int TN = 16, TK = 128;                       // a tile of weights
constexpr int TILE = TN * TK / 2 + TN * (TK / 32) * 2;  // its bytes: codes, then fp16 scales [row][group]
constexpr int STAGES = 4;                               // tiles of W in a warp's ring

__device__ __forceinline__ void copy16(void* dst, const void* src, int bytes) {  // the rest of the 16 is zero
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int ROWS = kWarps * TN;                       // rows of W per block
constexpr int RING = kWarps * STAGES * TILE;
template <int NT>
struct Cfg {
  static constexpr int COLS = 8 * NT;
  static constexpr int XK = NT == 1 ? 4 : 2;        // tiles along K whose columns of x are staged at a time, once for the block
  static constexpr int XROW = XK * TK * 2 + 64;     // bytes of a row of x: two rows of a load's phase meet different banks
  static constexpr int X = COLS * XROW;             // two of them
  static constexpr int SUMS = COLS * (ROWS + 4) * 4;
  static constexpr int SMEM = RING + 2 * X > SUMS ? RING + 2 * X : SUMS;
  static constexpr int BLOCKS = NT == 1 ? 6 : NT == 2 ? 5 : 4;  // per SM, by registers and shared memory
};

template <int NT>
__global__ void __launch_bounds__(kThreads, Cfg<NT>::BLOCKS) gemm_q4_kernel(const GemmQ4Args a) {
  using C = Cfg<NT>;
  constexpr int XK = C::XK, XROW = C::XROW;
  extern __shared__ __align__(128) uint8_t smem[];
  pdl_wait();
  pdl_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int m0 = blockIdx.z * C::COLS, rows = min(a.M - m0, C::COLS);
  const int kt_all = (a.K + TK - 1) / TK, n_tiles = (a.N + TN - 1) / TN;
  const int parts = gridDim.x, part = blockIdx.x;  // the cluster's blocks, along K
  const int kt0 = (int)((long long)kt_all * part / parts), kt1 = (int)((long long)kt_all * (part + 1) / parts);
  const bf16* x0 = a.x + (size_t)m0 * a.ldx;
  uint8_t* ring = smem + warp * (STAGES * TILE) + lane * 16;
  // what is fetched next (past the last rows: any tile, its sums go nowhere)
  const uint8_t* next = a.w + ((size_t)min((int)blockIdx.y * kWarps + warp, n_tiles - 1) * kt_all + kt0) * TILE + lane * 16;
  auto fetch = [&](int kt, int stage) {
    if (kt < kt1) {
#pragma unroll
      for (int c = 0; c < TILE; c += 512)
        if (c + 512 <= TILE || c + lane * 16 < TILE) copy16(ring + stage * TILE + c, next + c, 16);
      next += TILE;
    }
    copy_commit();
  };
  // A warp copies every warps-th row of x, a lane 16 bytes at a time; belongs to the copies of the tile that is fetched next
  auto fetch_x = [&](int kt, int half) {
    if (kt < kt1) {
      const uint8_t* src = reinterpret_cast<const uint8_t*>(x0 + (size_t)warp * a.ldx + kt * TK) + lane * 16;
      uint8_t* dst = smem + RING + half * C::X + warp * XROW + lane * 16;
      const int left = (a.K - kt * TK) * 2 - lane * 16;  // bytes of a row from the lane's place on (K is a multiple of 16 bytes)
      for (int m = warp; m < rows; m += kWarps, src += (size_t)kWarps * a.ldx * 2, dst += kWarps * XROW)
#pragma unroll
        for (int c = 0; c < XK * TK * 2; c += 512) copy16(dst + c, c < left ? src + c : reinterpret_cast<const uint8_t*>(a.x), c < left ? 16 : 0);
    }
  };
  fetch_x(kt0, 0);
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) fetch(kt0 + i, i);

  float acc[NT][4] = {};
  auto tile = [&](const uint8_t* w, const uint8_t* xs) {
    const uint4 c0 = *reinterpret_cast<const uint4*>(w), c1 = *reinterpret_cast<const uint4*>(w + 512);
    const uint2 d0 = *reinterpret_cast<const uint2*>(w + 1024 + g * 8 - lane * 16), d1 = *reinterpret_cast<const uint2*>(w + 1024 + 64 + g * 8 - lane * 16);
    const uint32_t w0[4] = {c0.x, c0.y, c0.z, c0.w}, w1[4] = {c1.x, c1.y, c1.z, c1.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t u0 = j < 2 ? d0.x : d0.y, u1 = j < 2 ? d1.x : d1.y;
      const float s0 = __half2float(__ushort_as_half((unsigned short)(j & 1 ? u0 >> 16 : u0 & 0xffffu)));
      const float s1 = __half2float(__ushort_as_half((unsigned short)(j & 1 ? u1 >> 16 : u1 & 0xffffu)));
      uint32_t a0[4], a1[4];
      q4::codes_bf16(w0[j], a0);
      q4::codes_bf16(w1[j], a1);
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const uint4 x = *reinterpret_cast<const uint4*>(xs + min(n * 8 + g, rows - 1) * XROW + j * 64);
        float c[4] = {0.f, 0.f, 0.f, 0.f};
        q4::mma_bf16(c, a0[0], a1[0], a0[1], a1[1], x.x, x.y);
        q4::mma_bf16(c, a0[2], a1[2], a0[3], a1[3], x.z, x.w);
        acc[n][0] = fmaf(s0, c[0], acc[n][0]);
        acc[n][1] = fmaf(s0, c[1], acc[n][1]);
        acc[n][2] = fmaf(s1, c[2], acc[n][2]);
        acc[n][3] = fmaf(s1, c[3], acc[n][3]);
      }
    }
  };
  const uint8_t* xs = smem + RING + t * 16;
  for (int kt = kt0; kt < kt1; kt += STAGES) {
#pragma unroll
    for (int u = 0; u < STAGES; ++u) {
      constexpr int kSwap = STAGES / XK;  // (even or one: which of the two places of x is in use follows from u, or from kt)
      const int half = kSwap == 1 ? (kt - kt0) / STAGES & 1 : u / XK & 1;
      // W's tile of this round is STAGES - 2 groups back; x of a new chunk, copied with the tile fetched XK rounds ago, XK - 1
      if (u % XK == 0) copy_wait<(XK - 1 < STAGES - 2 ? XK - 1 : STAGES - 2)>();
      else copy_wait<STAGES - 2>();
      __syncwarp();
      if (u % XK == 0) {
        __syncthreads();  // the columns of x are there for all, and the ones before are free
        fetch_x(kt + u + XK, half ^ 1);
      }
      fetch(kt + u + STAGES - 1, (u + STAGES - 1) % STAGES);
      if (kt + u < kt1) tile(ring + u * TILE, xs + half * C::X + u % XK * (TK * 2));
    }
  }
  copy_wait<0>();
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem);  // [column][ROWS + 4]
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int i = 0; i < 4; ++i) sums[(n * 8 + 2 * t + (i & 1)) * (ROWS + 4) + warp * TN + g + 8 * (i >> 1)] = acc[n][i];
  if (parts > 1) {
    __syncwarp();
    cluster_sync_all();
  } else {
    __syncthreads();
  }
  const int r = threadIdx.x % ROWS, n = blockIdx.y * ROWS + r;  // (two threads per row of W)
  if (n < a.N) {
    const float bias = a.bias ? __bfloat162float(a.bias[n]) : 0.f;
    for (int c = part * 2 + threadIdx.x / ROWS; c < rows; c += parts * 2) {
      float* at = sums + c * (ROWS + 4) + r;
      float v = 0.f;
      if (parts == 1) v = *at;
      else
        for (int q = 0; q < parts; ++q) v += *cluster_ptr<2>(at, q);
      const int m = m0 + c;
      v += bias;
      if (a.r) v += __bfloat162float(a.r[(size_t)m * a.ldr + n]);
      if (a.out_f32) reinterpret_cast<float*>(a.out)[(size_t)m * a.ldo + n] = v;
      else reinterpret_cast<bf16*>(a.out)[(size_t)m * a.ldo + n] = __float2bfloat16(v);
    }
  }
  if (parts > 1) {
    __syncwarp();
    cluster_sync_all();  // others may still read this block's sums
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

int device_sms() {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return effective_sms(sms);
}
template <int NT>
cudaError_t launch_q4(cudaStream_t stream, const GemmQ4Args& a, int sms) {
  using C = Cfg<NT>;
  static std::atomic<uint64_t> asked{0};  // more than 48 KB of shared memory wants to be asked for once per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  const uint64_t bit = dev < 64 ? 1ull << dev : 0;
  if (e == cudaSuccess && !(asked.load(std::memory_order_relaxed) & bit)) {
    e = cudaFuncSetAttribute(gemm_q4_kernel<NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
    if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  }
  if (e != cudaSuccess) return e;
  const int blocks_n = (a.N + ROWS - 1) / ROWS, tiles_m = (a.M + C::COLS - 1) / C::COLS, kt_all = (a.K + TK - 1) / TK;
  // Parts of K: twice as many while that leaves no more than some seven blocks per SM and four tiles per part.  Eight blocks join their sums slowly: only
  // where few blocks run, or where the tiles of 16 and more rows of x are slower still.  us: 1 x 4096 x 4096 12.8 in one part, 7.3 in 2, 5.9 in 4, 6.6 in 8;
  // 8 x 4096 x 14336 13.3 in 4, 15.4 in 8; 32 x 4096 x 14336 24.2 in 4, 22.2 in 8; 1 x 28672 x 4096 26.5 in one, 19.1 in 2, 19.8 in 4.
  const long long blocks = (long long)blocks_n * tiles_m;
  const int most = NT > 1 || blocks * 8 <= sms ? 8 : 4;
  int parts = 1;
  while (parts < most && blocks * parts * 2 <= 7LL * sms && kt_all >= parts * 2 * 4) parts *= 2;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(parts, blocks_n, tiles_m);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (parts > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = parts;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, gemm_q4_kernel<NT>, a);
}

size_t tiles_of(int N, int K) { return (size_t)((N + TN - 1) / TN) * ((K + TK - 1) / TK); }
bool weights_ok(int N, int K) { return N >= 1 && K >= 32 && K % 32 == 0 && N <= 65535 * ROWS && K <= (1 << 30) - TK; }  // (blocks of a grid; bytes of a row of x in 32 bits)

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
  const int sms = device_sms();
  if (sms <= 0) return cudaErrorNoDevice;
  if (a.M <= 8) return launch_q4<1>(stream, a, sms);
  if (a.M <= 16) return launch_q4<2>(stream, a, sms);
  return launch_q4<4>(stream, a, sms);
}

}  // namespace hb

// Page tables, slot maps and packed-row indices of a step, made on the GPU from the requests' lengths (the engine makes its own on the host: its
// scheduler has the lengths there; a step captured in a graph, or lengths that a kernel decided, cannot go through the host).
//
// Request b holds own = ceil(ctx / 64) pages.  new < 0: it ended, its pages go on top of the free stack in request order.  Otherwise it has `new`
// more tokens at rows [cu[b], cu[b + 1]) and takes need = ceil((ctx + new) / 64) - own pages from the top of the stack, in request order.  Which pages:
// an exclusive sum of need over the requests, which every block makes for itself (sums over at most 2048 requests in shared memory); rows,
// taken pages and returned pages are then independent, each finding its request by bisection of such a sum.  Nothing one block writes is read by
// another but the lengths and the stack height, where outputs are to overwrite them: then the blocks are one cluster, with its barrier between.
// Latency bounds it: 48 requests of one token each 3.6 us, a few sums and dependent loads; 700 requests with 56,000 rows 22 us in a cluster, 8.0 on all SMs.
#include <algorithm>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace hb {
namespace {

constexpr int kMaxReqs = 2048, kPer = 2;  // requests in all, and per thread
constexpr int kPage = 64;

// inclusive sums over the block's kPer consecutive values per thread, N sums at once, in place
template <int THREADS, int N>
__device__ __forceinline__ void block_scan(long long (&v)[N][kPer], long long (*s_warp)[32]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  long long sum[N];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int i = 1; i < kPer; ++i) v[n][i] += v[n][i - 1];
    sum[n] = v[n][kPer - 1];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, sum[n], o);
      if (lane >= o) sum[n] += x;
    }
    if (lane == 31) s_warp[n][warp] = sum[n];
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    long long w = lane < THREADS / 32 && lane < warp ? s_warp[n][lane] : 0;  // every warp adds up those before it
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
    const long long before = w + sum[n] - v[n][kPer - 1];
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[n][i] += before;
  }
  __syncthreads();  // s_warp is used again
}

// first of n ascending values that is above x
__device__ __forceinline__ int above(const int* v, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (v[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

template <int THREADS>
__global__ void __launch_bounds__(THREADS) page_tables_kernel(const PageTableArgs a, int clustered) {
  constexpr int REQS = THREADS * kPer;
  __shared__ int s_row[REQS], s_back[REQS], s_take[REQS], s_ctx[REQS];  // inclusive sums; lengths (-1 - length: refused)
  __shared__ long long s_warp[2][32];
  const int tid = threadIdx.x, B = a.B, T = a.T;
  long long ctx[kPer], sums[2][kPer], take[1][kPer];  // sums: of rows and of returned pages
  int fresh[kPer];
  const int count = min(max(*a.free_count, 0), a.num_pages);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    ctx[i] = b < B ? max(a.ctx_lens[b], 0) : 0;
    fresh[i] = b < B ? a.new_lens[b] : 0;
    sums[0][i] = max(fresh[i], 0);
    sums[1][i] = fresh[i] < 0 ? min((ctx[i] + kPage - 1) / kPage, (long long)a.max_pages) : 0;
  }
  block_scan<THREADS>(sums, s_warp);
  bool fits[kPer];
  long long need[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const long long after = (ctx[i] + max(fresh[i], 0) + kPage - 1) / kPage;
    fits[i] = after <= a.max_pages && sums[0][i] <= T;
    need[i] = fits[i] && fresh[i] >= 0 ? after - (ctx[i] + kPage - 1) / kPage : 0;
    take[0][i] = need[i];
  }
  if (tid == THREADS - 1) s_warp[1][0] = sums[1][kPer - 1];
  block_scan<THREADS>(take, s_warp);
  const int top = (int)min((long long)count + s_warp[1][0], (long long)a.num_pages);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    const bool ok = fits[i] && (need[i] == 0 || take[0][i] <= top);
    s_row[b] = (int)min(sums[0][i], (long long)T);
    s_back[b] = (int)min(sums[1][i], (long long)INT32_MAX);
    s_take[b] = (int)min(take[0][i], (long long)INT32_MAX);
    s_ctx[b] = ok ? (int)ctx[i] : -1 - (int)ctx[i];
  }
  // pages taken in all: the sum up to the last request that gets some
  long long best = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (need[i] > 0 && take[0][i] <= top) best = max(best, take[0][i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) s_warp[0][tid >> 5] = best;
  __syncthreads();
  best = (tid & 31) < THREADS / 32 ? s_warp[0][tid & 31] : 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  const int taken = (int)best, left = top - taken;
  if (clustered) cluster_sync_all();  // every block has read what the outputs may overwrite

  auto on_stack = [&](int i) {  // entry i of the stack with the returned pages on it
    if (i < count) return a.free_pages[i];
    const int j = i - count, b = above(s_back, B, j);
    return a.page_table[(size_t)b * a.max_pages + j - (b > 0 ? s_back[b - 1] : 0)];
  };
  const int first = blockIdx.x * THREADS + tid, step = gridDim.x * THREADS;
  for (int t = first; t < T; t += step) {
    const int b = above(s_row, B, t);
    int pos = 0, slot = -1;
    if (b < B) {
      const bool ok = s_ctx[b] >= 0;
      const int c = ok ? s_ctx[b] : -1 - s_ctx[b];
      pos = (int)min((long long)c + t - (b > 0 ? s_row[b - 1] : 0), (long long)INT32_MAX);
      if (ok) {
        const int at = pos / kPage - (c + kPage - 1) / kPage;
        const int page = at < 0 ? a.page_table[(size_t)b * a.max_pages + pos / kPage] : on_stack(top - 1 - ((b > 0 ? s_take[b - 1] : 0) + at));
        if (page >= 0 && page < a.num_pages) slot = page * kPage + pos % kPage;
      }
    }
    a.positions[t] = pos;
    a.slot_mapping[t] = slot;
  }
  for (int k = first; k < taken; k += step) {
    const int b = above(s_take, B, k);
    const int c = s_ctx[b] >= 0 ? s_ctx[b] : -1 - s_ctx[b];
    a.page_table[(size_t)b * a.max_pages + (c + kPage - 1) / kPage + k - (b > 0 ? s_take[b - 1] : 0)] = on_stack(top - 1 - k);
  }
  for (int i = count + first; i < left; i += step) a.free_pages[i] = on_stack(i);
  for (int b = first; b < B; b += step) {
    const bool ok = s_ctx[b] >= 0;
    const int c = ok ? s_ctx[b] : -1 - s_ctx[b], n = s_row[b] - (b > 0 ? s_row[b - 1] : 0);
    const bool ended = s_back[b] > (b > 0 ? s_back[b - 1] : 0);
    a.cu_seqlens[b + 1] = s_row[b];
    a.kv_lens[b] = ended ? 0 : ok ? c + n : c;
    if (b == 0) {
      a.cu_seqlens[0] = 0;
      *a.free_left = left;
    }
  }
}

}  // namespace

cudaError_t page_tables(cudaStream_t stream, const PageTableArgs& a) {
  if (!a.ctx_lens || !a.new_lens || !a.page_table || !a.free_pages || !a.free_count || !a.free_left || !a.cu_seqlens || !a.kv_lens || !a.positions ||
      !a.slot_mapping)
    return cudaErrorInvalidValue;
  if (a.B < 1 || a.B > kMaxReqs || a.T < 0 || a.T > 1 << 30 || a.max_pages < 1 || a.max_pages > INT32_MAX / kPage || a.num_pages < 1 || a.num_pages > INT32_MAX / kPage || a.page_size != kPage)
    return cudaErrorInvalidValue;
  // few rows: one block; many: blocks of a row per thread, or a cluster where the lengths or the stack's height are overwritten
  const bool small = a.B <= 256 * kPer && a.T <= 1024, over = a.kv_lens == a.ctx_lens || a.free_left == a.free_count;
  const int threads = small ? 256 : 1024, most = (std::max(a.T, a.B) + 1023) / 1024;
  const int blocks = small || most <= 2 ? 1 : over ? 8 : std::min(most, 128);
  const int clustered = over && blocks > 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(blocks);
  cfg.blockDim = dim3(threads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = blocks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = clustered ? 1 : 0;
  return small ? cudaLaunchKernelEx(&cfg, page_tables_kernel<256>, a, clustered) : cudaLaunchKernelEx(&cfg, page_tables_kernel<1024>, a, clustered);
}

}  // namespace hb

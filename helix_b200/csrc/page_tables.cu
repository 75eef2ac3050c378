// Page tables, slot maps and packed-row indices of a step, made on the GPU from the requests' lengths (the engine makes its own on the host: its
// scheduler has the lengths there; a step captured in a graph, or lengths that a kernel decided, cannot go through the host).
//
// Request b holds own = ceil(ctx / 64) pages.  new < 0: it ended, its pages go on top of the free stack in request order.  Otherwise it has `new`
// more tokens at rows [cu[b], cu[b + 1]) and takes need = ceil((ctx + new) / 64) - own pages from the top of the stack, in request order.  Which pages:
// an exclusive sum of need over the requests, which every block of the one cluster makes for itself (two sums over at most 2048 requests in
// shared memory); rows, taken pages and returned pages are then independent, each finding its request by bisection of such a sum.  Nothing
// one block writes is read by another but the lengths and the stack height, which outputs may overwrite: the cluster barrier lies between.
#include <algorithm>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace hb {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kMaxReqs = 2048, kPer = kMaxReqs / kThreads;
constexpr int kPage = 64;

// inclusive sum over the block's kPer consecutive values per thread, in place
__device__ __forceinline__ void block_scan(long long (&v)[kPer], long long* s_warp) {
#pragma unroll
  for (int i = 1; i < kPer; ++i) v[i] += v[i - 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long mine = v[kPer - 1];
  long long sum = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long x = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31) s_warp[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    long long w = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += x;
    }
    s_warp[lane] = w;
  }
  __syncthreads();
  const long long before = sum - mine + (warp > 0 ? s_warp[warp - 1] : 0);
#pragma unroll
  for (int i = 0; i < kPer; ++i) v[i] += before;
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

__global__ void __launch_bounds__(kThreads) page_tables_kernel(const PageTableArgs a) {
  __shared__ int s_row[kMaxReqs], s_back[kMaxReqs], s_take[kMaxReqs], s_ctx[kMaxReqs];  // inclusive sums; lengths (-1 - length: refused)
  __shared__ long long s_warp[kWarps];
  const int tid = threadIdx.x, B = a.B, T = a.T;
  const int rank = blockIdx.x, blocks = gridDim.x;
  long long ctx[kPer], row[kPer], back[kPer], take[kPer];
  int fresh[kPer];
  const int count = min(max(*a.free_count, 0), a.num_pages);
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    ctx[i] = b < B ? max(a.ctx_lens[b], 0) : 0;
    fresh[i] = b < B ? a.new_lens[b] : 0;
    row[i] = max(fresh[i], 0);
    back[i] = fresh[i] < 0 ? min((ctx[i] + kPage - 1) / kPage, (long long)a.max_pages) : 0;
  }
  block_scan(row, s_warp);
  block_scan(back, s_warp);
  bool fits[kPer];
  long long need[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const long long after = (ctx[i] + max(fresh[i], 0) + kPage - 1) / kPage;
    fits[i] = after <= a.max_pages && row[i] <= T;
    need[i] = fits[i] && fresh[i] >= 0 ? after - (ctx[i] + kPage - 1) / kPage : 0;
    take[i] = need[i];
  }
  block_scan(take, s_warp);
  if (tid == kThreads - 1) s_warp[0] = back[kPer - 1];
  __syncthreads();
  const int top = (int)min((long long)count + s_warp[0], (long long)a.num_pages);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int b = tid * kPer + i;
    const bool ok = fits[i] && (need[i] == 0 || take[i] <= top);
    s_row[b] = (int)min(row[i], (long long)T);
    s_back[b] = (int)min(back[i], (long long)INT32_MAX);
    s_take[b] = (int)min(take[i], (long long)INT32_MAX);
    s_ctx[b] = ok ? (int)ctx[i] : -1 - (int)ctx[i];
  }
  // pages taken in all: the sum up to the last request that gets some
  long long best = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (need[i] > 0 && take[i] <= top) best = max(best, take[i]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) best = max(best, __shfl_xor_sync(0xffffffffu, best, o));
  if ((tid & 31) == 0) s_warp[tid >> 5] = best;
  __syncthreads();
  best = 0;
  for (int i = 0; i < kWarps; ++i) best = max(best, s_warp[i]);
  const int taken = (int)best, left = top - taken;
  cluster_sync_all();  // every block has read what the outputs may overwrite

  auto on_stack = [&](int i) {  // entry i of the stack with the returned pages on it
    if (i < count) return a.free_pages[i];
    const int j = i - count, b = above(s_back, B, j);
    return a.page_table[(size_t)b * a.max_pages + j - (b > 0 ? s_back[b - 1] : 0)];
  };
  const int first = rank * kThreads + tid, step = blocks * kThreads;
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
  if (a.B < 1 || a.B > kMaxReqs || a.T < 0 || a.max_pages < 1 || a.max_pages > INT32_MAX / kPage || a.num_pages < 1 || a.num_pages > INT32_MAX / kPage || a.page_size != kPage)
    return cudaErrorInvalidValue;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(std::max(a.T, a.B) <= 2 * kThreads ? 1 : 8);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cfg.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, page_tables_kernel, a);
}

}  // namespace hb

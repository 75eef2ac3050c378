// Scores of given tokens from logits: log softmax of a token, its rank, the entropy of the row and the first tokens of the order (logit descending, id ascending).
//
// One pass over a row, read once: every thread keeps the running maximum m of its entries, S = sum e^(x - m) and U = sum (x - m) e^(x - m), so that at the end
//   log softmax(x_t) = x_t - m - log S,   entropy = log S - U / S.
// The first tokens pass through a list in shared memory: an entry goes there only if it is not behind a bound, the n-th best of what was seen up to some step before.  The bound
// is drawn anew after 1, 2, 4, 8.. steps, so that some n entries are listed between two of these whatever the row's length, and the threads run freely in between.  Rows in which
// more are listed than there is room for (rising ones, say) have those steps looked through again step by step.  Places in the order are compared as one whole number of 64
// bits (value bits made ordered, then the id complemented): no two are alike, ties go to the lower id, and the result does not depend on who came first.
//
// Bytes bound it: 4 or 2 per logit.  A row belongs to a cluster of 1 to 8 blocks, so that few rows still keep all SMs reading.
#include <algorithm>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace hb {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int E = 8;                    // neighbouring entries of a thread
constexpr int kStep = kThreads * E;     // entries that a block takes at a time
constexpr int kMost = 64;               // n_top at most
constexpr int kList = 1024;             // places of the list: what is kept (kMost) and what one step may add (kMost * E) fit
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ uint32_t ordered(float x) {  // 0 for a NaN, which comes last; zeros tie
  const float y = x + 0.f;
  const uint32_t u = __float_as_uint(y);
  return y == y ? (u & 0x80000000u ? ~u : u | 0x80000000u) : 0u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
__device__ __forceinline__ u64 place_of(float x, int id) {  // the larger, the earlier; 0: never
  const uint32_t k = ordered(x);
  return k ? (u64)k << 32 | (uint32_t)~id : 0ull;
}
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

struct Sums {
  float m, s, u;
};
// S and U of two parts brought to the larger maximum
__device__ __forceinline__ Sums join(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  Sums r{m, 0.f, 0.f};
  auto add = [&](const Sums& p) {
    const float d = p.m == m ? 0.f : p.m - m;
    const float w = d < -200.f ? 0.f : exp2_fast(d * kLog2e);  // (nothing is left of it below e^-200: and no infinity times 0)
    if (w > 0.f || p.s != p.s) {
      r.s = fmaf(w, p.s, r.s);
      r.u += w * fmaf(d < -200.f ? 0.f : d, p.s, p.u);
    }
  };
  add(a);
  add(b);
  if (a.s != a.s || b.s != b.s) r.s = __uint_as_float(0x7fffffffu);
  return r;
}

struct Shared {
  u64 list[kList];
  u64 best[kMost];   // a block's first tokens
  Sums warp_sums[kWarps];
  int warp_before[kWarps];
  Sums sums;
  int before;
  int count;
};

// The list becomes its n largest (n at most kMost), in order; returns the n-th, 0 where there are fewer.  All threads come here.
__device__ __forceinline__ u64 thin_out(Shared& sh, int n) {
  __syncthreads();
  const int count = min(sh.count, kList);
  u64 mine[kList / kThreads];
  int ahead[kList / kThreads];
#pragma unroll
  for (int k = 0; k < kList / kThreads; ++k) {
    mine[k] = k * kThreads + (int)threadIdx.x < count ? sh.list[k * kThreads + threadIdx.x] : 0ull;
    ahead[k] = 0;
    if (mine[k])
      for (int j = 0; j < count; ++j) ahead[k] += sh.list[j] > mine[k];
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < kList / kThreads; ++k)
    if (mine[k] && ahead[k] < n) sh.list[ahead[k]] = mine[k];
  if (threadIdx.x == 0) sh.count = min(count, n);
  __syncthreads();
  return count >= n ? sh.list[n - 1] : 0ull;
}

template <bool F32>
__device__ __forceinline__ float logit_at(const void* row, int i) {
  return F32 ? __ldg(static_cast<const float*>(row) + i) : __bfloat162float(static_cast<const bf16*>(row)[i]);
}
// A thread's entries travel to its own places in shared memory some steps ahead of it: nobody else reads them, so there is nothing to wait for but its own copies
template <bool F32>
struct Ring {
  static constexpr int WIDE = F32 ? 2 : 1;   // 16 bytes of a thread's entries
  static constexpr int AHEAD = F32 ? 2 : 4;  // steps
  uint4 v[AHEAD][WIDE][kThreads];
};
__device__ __forceinline__ void copy16(void* dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool F32, int NC, bool TOP>
__global__ void __launch_bounds__(kThreads, 3) token_scores_kernel(const TokenScoresArgs a) {
  __shared__ Shared sh;
  __shared__ Ring<F32> ring;
  constexpr int AHEAD = Ring<F32>::AHEAD, WIDE = Ring<F32>::WIDE;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = NC == 1 ? 0 : (int)(blockIdx.x % NC), t = blockIdx.x / NC;
  const void* row = static_cast<const uint8_t*>(a.logits) + (size_t)t * a.ldl * (F32 ? 4 : 2);
  // this block's entries: a share of whole eights
  const int eights = (a.V + E - 1) / E;
  const int begin = (int)((long long)eights * part / NC) * E, end = min(a.V, (int)((long long)eights * (part + 1) / NC) * E);
  const int target = a.targets ? a.targets[t] : -1;
  const bool has = target >= 0 && target < a.V;
  const float xt = has ? logit_at<F32>(row, target) : 0.f;
  if (tid == 0) sh.count = 0;
  __syncthreads();

  Sums my{-INFINITY, 0.f, 0.f};
  int before = 0;
  u64 bound = 0;  // an entry that is listed is not behind it
  auto entries_at = [&](int i, float (&f)[E]) {
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = i + e < end ? logit_at<F32>(row, i + e) : -INFINITY;
  };
  auto list = [&](const float(&f)[E], int i) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const u64 place = i + e < end ? place_of(f[e], i + e) : 0ull;
      if (place > bound) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kList) sh.list[at] = place;
      }
    }
  };
  // One step, its entries seen as they are: the n-th best of the threads' first places bounds what may be among the row's first n, so that no more than n threads list theirs
  auto careful = [&](int i0) {
    const int i = i0 + tid * E;
    float f[E];
    entries_at(i, f);
    u64 first = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const u64 place = i + e < end ? place_of(f[e], i + e) : 0ull;
      first = place > first ? place : first;
    }
    if (first <= bound) first = 0;
    const int hits = __syncthreads_count(first != 0);
    if (hits == 0) return;
    if (hits > a.n_top) {
      u64 at = 0;
      for (int bit = 63; bit >= 0; --bit) {
        const u64 trial = at | 1ull << bit;
        const int c = __syncthreads_count(first >= trial);
        if (c >= a.n_top) {
          at = trial;
          if (c == a.n_top) break;
        }
      }
      bound = at - 1 > bound ? at - 1 : bound;
    }
    if (first > bound) list(f, i);
    const u64 nth = thin_out(sh, a.n_top);
    if (nth > bound) bound = nth;
  };
  int seen = begin, draw = begin;  // where the steps begin that the list has not been thinned out behind, and behind the last of them
  auto settle = [&](int behind) {  // the list is thinned out behind the steps before `behind`
    __syncthreads();
    if (sh.count > kList) {
      if (tid == 0) sh.count = min(seen > begin ? a.n_top : 0, kList);  // what was kept lies in front
      __syncthreads();
      for (int s = seen; s < behind; s += kStep) careful(s);
    } else {
      const u64 nth = thin_out(sh, a.n_top);
      if (nth > bound) bound = nth;
    }
    seen = behind;
  };
  auto whole = [&](int i) { return i + E <= end; };
  auto fetch = [&](int i, int place) {
    if (whole(i)) {
#pragma unroll
      for (int k = 0; k < WIDE; ++k) copy16(&ring.v[place][k][tid], static_cast<const uint8_t*>(row) + (size_t)i * (F32 ? 4 : 2) + 16 * k);
    }
    copy_commit();
  };
#pragma unroll
  for (int k = 0; k < AHEAD; ++k) fetch(begin + k * kStep + tid * E, k);
  int place = 0;
  if constexpr (TOP) {
    if (begin < end) careful(begin);
    seen = begin + kStep;
    draw = begin + 2 * kStep;
  }
  for (int i0 = begin; i0 < end; i0 += kStep) {
    const int i = i0 + tid * E;
    float f[E];
    copy_wait<AHEAD - 1>();
    if (whole(i)) {
      const uint4 u = ring.v[place][0][tid];
      if constexpr (F32) {
        const uint4 v = ring.v[place][WIDE - 1][tid];
        f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
        f[4] = __uint_as_float(v.x); f[5] = __uint_as_float(v.y); f[6] = __uint_as_float(v.z); f[7] = __uint_as_float(v.w);
      } else {
        unpack_bf16x8(u, f);
      }
    } else {
      entries_at(i, f);
    }
    fetch(i + AHEAD * kStep, place);
    place = place + 1 == AHEAD ? 0 : place + 1;
    const float top = fmaxf(fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])), fmaxf(fmaxf(f[4], f[5]), fmaxf(f[6], f[7])));
    if (top > my.m) {
      if (my.m > -INFINITY) {
        const float d = my.m - top, w = exp2_fast(d * kLog2e);
        my.u = w > 0.f ? w * fmaf(d, my.s, my.u) : 0.f;
        my.s *= w;
      }
      my.m = top;
    }
    const float m = my.m > -INFINITY ? my.m : 0.f;
    const uint64_t off = f2_pack(-m, -m), log2e = f2_pack(kLog2e, kLog2e);
    uint64_t s2 = f2_pack(0.f, 0.f), u2 = s2;  // two at a time
#pragma unroll
    for (int e = 0; e < E; e += 2) {
      const uint64_t d = f2_add(f2_pack(f[e], f[e + 1]), off);
      float d0, d1, x0, x1;
      f2_unpack(d, d0, d1);
      f2_unpack(f2_mul(d, log2e), x0, x1);
      const uint64_t w = f2_pack(exp2_fast(x0), exp2_fast(x1));
      s2 = f2_add(s2, w);
      u2 = f2_fma(w, f2_pack(fmaxf(d0, -1e4f), fmaxf(d1, -1e4f)), u2);  // (a masked entry: 0 times what is no infinity)
    }
    float lo, hi;
    f2_unpack(s2, lo, hi);
    my.s += lo + hi;
    f2_unpack(u2, lo, hi);
    my.u += lo + hi;
    if (i >= end) {  // (nothing: the -inf in its place is no token)
    } else if (i + E <= target) {
#pragma unroll
      for (int e = 0; e < E; ++e) before += f[e] >= xt;
    } else if (i > target) {
#pragma unroll
      for (int e = 0; e < E; ++e) before += f[e] > xt && i + e < end;
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) before += i + e < end && (f[e] > xt || (f[e] == xt && i + e < target));
    }
    if constexpr (TOP) {
      if (i0 > begin) {  // (the first step has been seen)
        if (ordered(top) >= (uint32_t)(bound >> 32)) list(f, i);
        if (i0 + kStep >= draw && i0 + kStep < end) {
          settle(i0 + kStep);
          draw = i0 + kStep + (i0 + kStep - begin);
        }
      }
    }
  }
  if constexpr (TOP) {
    if (seen < end) settle(end);
  }

  // the block's sums
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const Sums other{__shfl_xor_sync(0xffffffffu, my.m, o), __shfl_xor_sync(0xffffffffu, my.s, o), __shfl_xor_sync(0xffffffffu, my.u, o)};
    my = lane & o ? join(other, my) : join(my, other);
  }
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) {
    sh.warp_sums[warp] = my;
    sh.warp_before[warp] = before;
  }
  __syncthreads();
  if (tid == 0) {
    Sums all = sh.warp_sums[0];
    int n = sh.warp_before[0];
    for (int w = 1; w < kWarps; ++w) {
      all = join(all, sh.warp_sums[w]);
      n += sh.warp_before[w];
    }
    sh.sums = all;
    sh.before = n;
  }
  if constexpr (TOP) {
    if (NC > 1 && tid < kMost) sh.best[tid] = tid < sh.count ? sh.list[tid] : 0ull;  // (the list is in order)
  }
  __syncthreads();
  Sums all = sh.sums;
  int n_before = sh.before;
  if constexpr (NC > 1) {
    __syncwarp();
    cluster_sync_all();
    if (part == 0) {
      for (int c = 1; c < NC; ++c) {
        all = join(all, *cluster_ptr<NC>(&sh.sums, c));
        n_before += *cluster_ptr<NC>(&sh.before, c);
      }
      if constexpr (TOP) {
        // (no more than 8 x 64 places: one per thread)
        const int c = tid / kMost, j = tid % kMost;
        const u64 p = c < NC && j < a.n_top ? *cluster_ptr<NC>(&sh.best[j], c) : 0ull;
        if (tid == 0) sh.count = 0;
        __syncthreads();
        if (p) sh.list[atomicAdd(&sh.count, 1)] = p;
        __syncthreads();
      }
    }
    __syncwarp();
    cluster_sync_all();  // the others may leave
    if (part != 0) return;
    if constexpr (TOP) thin_out(sh, a.n_top);
  }
  const bool none = all.s == 0.f;  // nothing but -inf
  const float log_s = logf(all.s), lse = none ? INFINITY : all.m + log_s;
  if (tid == 0) {
    if (a.lp) a.lp[t] = has ? xt - lse : -INFINITY;
    if (a.rank) a.rank[t] = has && xt == xt ? n_before : -1;
    if (a.entropy) a.entropy[t] = none ? 0.f : log_s - all.u / all.s;
  }
  if constexpr (TOP) {
    for (int j = tid; j < a.n_top; j += kThreads) {
      const u64 p = j < sh.count ? sh.list[j] : 0ull;
      a.top_ids[(size_t)t * a.n_top + j] = p ? (int)~(uint32_t)p : -1;
      if (a.top_lp) a.top_lp[(size_t)t * a.n_top + j] = p ? value_of((uint32_t)(p >> 32)) - lse : __uint_as_float(0x7fffffffu);
    }
  }
}

template <bool F32, int NC, bool TOP>
cudaError_t launch_nc(cudaStream_t stream, const TokenScoresArgs& a) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.T * NC);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (NC > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = NC;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, token_scores_kernel<F32, NC, TOP>, a);
}
template <bool F32, bool TOP>
cudaError_t launch_top(cudaStream_t stream, const TokenScoresArgs& a, int sms) {
  // blocks per row: twice as many while not all SMs have one of their three and a block keeps some steps
  int nc = 1;
  while (nc < 8 && (long long)a.T * nc * 2 <= 3LL * sms && a.V >= nc * 2 * kStep) nc *= 2;
  switch (nc) {
    case 1: return launch_nc<F32, 1, TOP>(stream, a);
    case 2: return launch_nc<F32, 2, TOP>(stream, a);
    case 4: return launch_nc<F32, 4, TOP>(stream, a);
    default: return launch_nc<F32, 8, TOP>(stream, a);
  }
}

}  // namespace

cudaError_t token_scores(cudaStream_t stream, const TokenScoresArgs& a) {
  if (a.T < 0 || a.T > (1 << 28) || a.V < 1 || a.V > (1 << 30) || a.n_top < 0 || a.n_top > kMost || a.n_top > a.V) return cudaErrorInvalidValue;
  if (a.T == 0) return cudaSuccess;
  if (!a.logits || ((uintptr_t)a.logits & 15) || a.ldl < a.V || a.ldl % 8 || ((a.lp || a.rank) && !a.targets) || (a.n_top > 0 && !a.top_ids)) return cudaErrorInvalidValue;
  if ((((uintptr_t)a.targets | (uintptr_t)a.lp | (uintptr_t)a.rank | (uintptr_t)a.entropy | (uintptr_t)a.top_ids | (uintptr_t)a.top_lp) & 3)) return cudaErrorInvalidValue;
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return cudaErrorNoDevice;
  sms = effective_sms(sms);
  if (a.f32) return a.n_top ? launch_top<true, true>(stream, a, sms) : launch_top<true, false>(stream, a, sms);
  return a.n_top ? launch_top<false, true>(stream, a, sms) : launch_top<false, false>(stream, a, sms);
}

}  // namespace hb

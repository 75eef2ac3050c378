// Scores of given tokens from logits: log softmax of a token, its rank, the entropy of the row and the first tokens of the order (logit descending, id ascending).
//
// One pass over a row, read once: every thread keeps an m near the maximum of its entries, S = sum e^(x - m) and U = sum (x - m) e^(x - m), so that at the end
//   log softmax(x_t) = x_t - m - log S,   entropy = log S - U / S.
// A thread also remembers the step in which it met its maximum, and the largest of its other steps' maxima.  The n-th best of the threads' maxima bounds what may be among
// the row's first n: n threads have such entries, and list those of that step; the few whose other steps reach the bound too are looked through once more (from L2).  Places in the
// order are compared as one whole number of 64 bits (value bits made ordered, then the id complemented): no two are alike, ties go to the lower id, and the result does not
// depend on who came first.  Rows in which more entries are listed than there is room for (rising ones, say) are looked through step by step, the list thinned out to the first n
// between two steps.
//
// Bytes bound it: 4 or 2 per logit.  A row belongs to a cluster of 1 to 8 blocks, so that few rows still keep all SMs reading.
#include <algorithm>

#include "kernels.h"
#include "launch.h"
#include "ptx.cuh"

namespace hb {
namespace {

typedef unsigned long long u64;
constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMost = 64;               // n_top at most
constexpr int kList = 1280;             // places of the list: what is kept (kMost) and what one step may add (kMost threads' entries) fit
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

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ float at_least(float a, float b) {  // 1 or 0
  float r;
  asm("set.ge.f32.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

struct Sums {
  float m, s, u;
};
// The sums of the first `lanes` lanes (a power of two) brought to the largest m and added, known to all of these afterwards
__device__ __forceinline__ Sums join_lanes(const Sums& my, int lanes) {
  const float m = value_of(__reduce_max_sync(0xffffffffu, ordered(my.m)));
  const float d = my.m == m ? 0.f : my.m - m;  // (no infinity less itself)
  const float w = exp2_fast(d * kLog2e);
  Sums r{m, w * my.s, w > 0.f ? w * fmaf(d, my.s, my.u) : 0.f};
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    if (o < lanes) {
      r.s += __shfl_xor_sync(0xffffffffu, r.s, o);
      r.u += __shfl_xor_sync(0xffffffffu, r.u, o);
    }
  return r;
}

struct Shared {
  u64 list[kList];
  u64 best[kThreads];  // the threads' earliest places; a block's first tokens
  u64 bound;
  int step[kThreads];  // with a thread's maximum
  int candidate[kMost], candidates, ahead[kMost];
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
// A thread takes two pieces of 16 bytes of each step, a warp's pieces side by side.  They travel to its own places in shared memory some steps ahead of it: nobody else reads
// them, so there is nothing to wait for but its own copies.
constexpr int kWide = 2;                // pieces of a thread's entries
constexpr int kAhead = 3;               // steps
template <bool F32>
constexpr int kEntries = F32 ? 8 : 16;
struct Ring {
  uint4 v[kAhead][kWide][kThreads];
};
__device__ __forceinline__ void copy16(void* dst, const void* src) { asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory"); }
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <bool F32, int NC, bool TOP>
__global__ void __launch_bounds__(kThreads, 4) token_scores_kernel(const TokenScoresArgs a) {
  constexpr int E = kEntries<F32>, P = E / kWide, kStep = kThreads * E;  // entries of a thread, of a piece, of a step
  __shared__ Shared sh;
  __shared__ Ring ring;
  pdl_wait();
  pdl_launch_dependents();
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int part = NC == 1 ? 0 : (int)(blockIdx.x % NC), t = blockIdx.x / NC;
  const void* row = static_cast<const uint8_t*>(a.logits) + (size_t)t * a.ldl * (F32 ? 4 : 2);
  // this block's entries: a share of whole groups of E
  const int groups = (a.V + E - 1) / E;
  const int begin = (int)((long long)groups * part / NC) * E, end = min(a.V, (int)((long long)groups * (part + 1) / NC) * E);
  auto first_of = [&](int thread) { return begin + thread / 32 * (32 * E) + thread % 32 * P; };  // its first entry of the first step
  auto id_of = [](int i, int e) { return i + e / P * (32 * P) + e % P; };                         // of entry e of a thread whose first of the step is i
  auto whole = [&](int i) { return i + 32 * P + P <= end; };
  auto piece_at = [&](int i, int k) { return static_cast<const uint8_t*>(row) + (size_t)(i + k * (32 * P)) * (F32 ? 4 : 2); };
  auto fetch = [&](int i, int place) {
    if (whole(i)) {
#pragma unroll
      for (int k = 0; k < kWide; ++k) copy16(&ring.v[place][k][tid], piece_at(i, k));
    }
    copy_commit();
  };
  const int mine = first_of(tid);
#pragma unroll
  for (int k = 0; k < kAhead; ++k) fetch(mine + k * kStep, k);
  const int target = a.targets ? a.targets[t] : -1;
  const bool has = target >= 0 && target < a.V;
  const float xt = has ? logit_at<F32>(row, target) : __uint_as_float(0x7fffffffu);
  // the next value above the target's: what is no less comes before it wherever it stands (none does where that is a NaN)
  const uint32_t bits = __float_as_uint(xt + 0.f);
  const float above = xt == 0.f ? __uint_as_float(1u) : __uint_as_float(bits & 0x80000000u ? bits - 1 : bits + 1);
  if (tid == 0) sh.count = 0;
  __syncthreads();

  Sums my{-INFINITY, 0.f, 0.f};
  int first_at = mine;  // the step with the thread's maximum
  float best = -INFINITY, second = -INFINITY;  // that, and the largest of its other steps
  uint64_t before2 = f2_pack(0.f, 0.f);  // (whole numbers below 2^24)
  int equals = 0;
  auto values_of = [&](const uint4& u, const uint4& v, float(&f)[E]) {
    if constexpr (F32) {
      f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
      f[4] = __uint_as_float(v.x); f[5] = __uint_as_float(v.y); f[6] = __uint_as_float(v.z); f[7] = __uint_as_float(v.w);
    } else {
      unpack_bf16x8(u, *reinterpret_cast<float(*)[8]>(f));
      unpack_bf16x8(v, *reinterpret_cast<float(*)[8]>(f + 8));
    }
  };
  auto entries_at = [&](int i, float(&f)[E]) {  // -inf behind the last
    if (whole(i)) {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(piece_at(i, 0))), v = __ldg(reinterpret_cast<const uint4*>(piece_at(i, 1)));
      values_of(u, v, f);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = id_of(i, e) < end ? logit_at<F32>(row, id_of(i, e)) : -INFINITY;
    }
  };
  int place = 0;
  for (int i0 = begin; i0 < end; i0 += kStep) {
    const int i = mine + (i0 - begin);
    float f[E];
    copy_wait<kAhead - 1>();
    if (whole(i)) {
      values_of(ring.v[place][0][tid], ring.v[place][1][tid], f);
    } else {
      entries_at(i, f);
    }
    fetch(i + kAhead * kStep, place);
    place = place + 1 == kAhead ? 0 : place + 1;
    float top = f[0];
#pragma unroll
    for (int e = 1; e + 1 < E; e += 2) top = max3(top, f[e], f[e + 1]);
    top = fmaxf(top, f[E - 1]);
    second = fmaxf(second, fminf(best, top));
    first_at = top > best ? i : first_at;
    best = fmaxf(best, top);
    if (best - my.m > 8.f) {  // (m need not be the maximum: it follows when it is left far behind)
      if (my.m > -INFINITY) {
        const float d = my.m - best, w = exp2_fast(d * kLog2e);
        my.u = w > 0.f ? w * fmaf(d, my.s, my.u) : 0.f;
        my.s *= w;
      }
      my.m = best;
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
#pragma unroll
    for (int k = 0; k < kWide; ++k) {
      const int j = id_of(i, k * P);
      const float line = j >= end ? __uint_as_float(0x7fffffffu) : j + P <= target ? xt : above;
#pragma unroll
      for (int e = k * P; e < (k + 1) * P; e += 2) before2 = f2_add(before2, f2_pack(at_least(f[e], line), at_least(f[e + 1], line)));
      if (j < end && j <= target && target < j + P) {
#pragma unroll
        for (int e = 0; e < P; ++e) equals += j + e < target && f[k * P + e] == xt;
      }
    }
  }
  float b0, b1;
  f2_unpack(before2, b0, b1);
  int before = (int)b0 + (int)b1 + equals;
  if constexpr (TOP) {
    const int n = a.n_top;
    u64 first = 0;  // the thread's earliest place
    float f[E];
    int i = first_at;
    for (; i < end; i += kStep) {  // (where its maximum is -inf, the first that is no NaN may lie further on)
      entries_at(i, f);
      int at = E;
#pragma unroll
      for (int e = E - 1; e >= 0; --e) at = f[e] == best ? e : at;
      if (at < E && id_of(i, at) < end) {
        first = place_of(best, id_of(i, at));
        break;
      }
    }
    sh.best[tid] = first;
    if (tid == 0) sh.candidates = 0;
    __syncthreads();
    if (warp == 0) {  // the n-th of them by value, two bits at a time
      uint32_t theirs[kThreads / 32], high = 0, low = ~0u;
      int live = 0;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) {
        theirs[k] = (uint32_t)(sh.best[k * 32 + lane] >> 32);
        high = max(high, theirs[k]);
        low = min(low, theirs[k]);
        live += theirs[k] != 0;
      }
      u64 bound = 0;
      if (__reduce_add_sync(0xffffffffu, live) > n) {
        high = __reduce_max_sync(0xffffffffu, high);
        low = __reduce_min_sync(0xffffffffu, low);
        int bit = high == low ? -2 : (31 - __clz(high ^ low)) & ~1;  // (of the upper one of a pair's two)
        uint32_t key = bit < 0 ? high : bit == 30 ? 0 : high & ~((4u << bit) - 1);
        int c = kThreads;
        for (; bit >= 0 && c != n; bit -= 2) {
          uint32_t counts = 0;  // of those at or above key + 1, 2, 3 units of the pair, ten bits each
#pragma unroll
          for (int k = 0; k < kThreads / 32; ++k)
            counts += (theirs[k] >= key + (1u << bit) ? 1u : 0u) + (theirs[k] >= key + (2u << bit) ? 1u << 10 : 0u) + (theirs[k] >= key + (3u << bit) ? 1u << 20 : 0u);
          counts = __reduce_add_sync(0xffffffffu, counts);
          const int units = (counts & 1023) >= (uint32_t)n ? (counts >> 10 & 1023) >= (uint32_t)n ? (counts >> 20) >= (uint32_t)n ? 3 : 2 : 1 : 0;
          if (units) {
            key += (uint32_t)units << bit;
            c = counts >> (10 * (units - 1)) & 1023;
          }
        }
        u64 at = (u64)key << 32;
        if (c > kMost) {  // more tie than may list theirs: the n-th by its id too
          for (bit = 31; bit >= 0; --bit) {
            const u64 trial = at | 1ull << bit;
            int above = 0;
            for (int k = 0; k < kThreads / 32; ++k) above += sh.best[k * 32 + lane] >= trial;
            above = __reduce_add_sync(0xffffffffu, above);
            if (above >= n) {
              at = trial;
              if (above == n) break;
            }
          }
        }
        bound = at - 1;
      }
      if (lane == 0) sh.bound = bound;
    }
    __syncthreads();
    u64 bound = sh.bound;  // what is listed lies above it
    const float line = value_of((uint32_t)((bound + 1) >> 32));  // (what is no less may lie above the bound; a NaN for none: so all do)
    auto list = [&](const float(&f)[E], int i) {  // those of a thread's entries of a step
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (!(f[e] < line) && id_of(i, e) < end) {
          const u64 place = place_of(f[e], id_of(i, e));
          if (place > bound) {
            const int to = atomicAdd(&sh.count, 1);
            if (to < kList) sh.list[to] = place;
          }
        }
    };
    if (first > bound) {  // (kMost threads at most)
      list(f, i);
      if (ordered(second) >= (uint32_t)(bound >> 32)) sh.candidate[atomicAdd(&sh.candidates, 1)] = tid;
    }
    sh.step[tid] = i;
    __syncthreads();
    const int candidates = sh.candidates;
    for (int k = warp; k < candidates; k += kWarps) {  // a warp looks through the other entries of one of them, a step per lane
      const int c = sh.candidate[k], done = sh.step[c];
      for (int j = first_of(c) + lane * kStep; j < end; j += 32 * kStep) {
        if (j == done) continue;
        float g[E];
        entries_at(j, g);
        float top = g[0];
#pragma unroll
        for (int e = 1; e < E; ++e) top = fmaxf(top, g[e]);
        if (ordered(top) >= (uint32_t)(bound >> 32)) list(g, j);
      }
    }
    __syncthreads();
    if (sh.count > kList) {
      __syncthreads();
      if (tid == 0) sh.count = 0;
      __syncthreads();
      for (int i0 = begin; i0 < end; i0 += kStep) {
        if (first > bound) {
          entries_at(mine + (i0 - begin), f);
          list(f, mine + (i0 - begin));
        }
        __syncthreads();
        const int count = sh.count;
        __syncthreads();
        if (count > kMost) {
          const u64 nth = thin_out(sh, n);
          bound = nth > bound + 1 ? nth - 1 : bound;
        }
      }
    }
    thin_out(sh, n);
  }

  // the block's sums
  my = join_lanes(my, 32);
  before = __reduce_add_sync(0xffffffffu, before);
  if (lane == 0) {
    sh.warp_sums[warp] = my;
    sh.warp_before[warp] = before;
  }
  __syncthreads();
  Sums all = join_lanes(sh.warp_sums[lane % kWarps], kWarps);
  int n_before = __reduce_add_sync(0xffffffffu, lane < kWarps ? sh.warp_before[lane] : 0);
  if (NC > 1 && tid == 0) {
    sh.sums = all;
    sh.before = n_before;
  }
  if constexpr (TOP) {
    if (NC > 1 && tid < kMost) sh.best[tid] = tid < sh.count ? sh.list[tid] : 0ull;  // (the list is in order)
  }
  if constexpr (NC > 1) {
    __syncthreads();
    cluster_sync_all();
    all = join_lanes(*cluster_ptr<NC>(&sh.sums, lane % NC), NC);
    n_before = __reduce_add_sync(0xffffffffu, lane < NC ? *cluster_ptr<NC>(&sh.before, lane % NC) : 0);
  }
  const bool none = all.s == 0.f;  // nothing but -inf
  const float log_s = logf(all.s), lse = none ? INFINITY : all.m + log_s;
  if (part == 0 && tid == 0) {
    if (a.lp) a.lp[t] = has ? xt - lse : -INFINITY;
    if (a.rank) a.rank[t] = has && xt == xt ? n_before : -1;
    if (a.entropy) a.entropy[t] = none ? 0.f : log_s - all.u / all.s;
  }
  if constexpr (TOP) {
    const int n = a.n_top;
    auto write = [&](int to, u64 place) {
      a.top_ids[(size_t)t * n + to] = place ? (int)~(uint32_t)place : -1;
      if (a.top_lp) a.top_lp[(size_t)t * n + to] = place ? value_of((uint32_t)(place >> 32)) - lse : __uint_as_float(0x7fffffffu);
    };
    if constexpr (NC == 1) {
      for (int j = tid; j < n; j += kThreads) write(j, j < sh.count ? sh.list[j] : 0ull);
    } else {
      // every block sees all blocks' first tokens, and writes its own to where they stand among these
      for (int k = tid; k < NC * kMost; k += kThreads) sh.list[k] = k % kMost < n ? *cluster_ptr<NC>(&sh.best[k % kMost], k / kMost) : 0ull;
      if (tid < kMost) sh.ahead[tid] = 0;
      int live = 0;
      for (int k = 0; k < NC * kMost; k += kThreads) live += __syncthreads_count(k + tid < NC * kMost && sh.list[min(k + tid, NC * kMost - 1)] != 0);
      for (int k = tid; k < n * NC; k += kThreads) {
        const u64 place = sh.best[k / NC];
        const u64* other = sh.list + k % NC * kMost;
        int ahead = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) ahead += other[j] > place;
        if (ahead) atomicAdd(&sh.ahead[k / NC], ahead);
      }
      __syncthreads();
      if (tid < n) {
        if (sh.best[tid] && sh.ahead[tid] < n) write(sh.ahead[tid], sh.best[tid]);
        if (part == 0 && tid >= live) write(tid, 0ull);
      }
    }
  }
  if constexpr (NC > 1) {
    __syncwarp();
    cluster_sync_all();  // others may still read this block's
  }
}

template <bool F32, int NC, bool TOP>
cudaError_t launch_nc(cudaStream_t stream, const TokenScoresArgs& a, int sms) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)a.T * NC);
  cfg.blockDim = dim3(kThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  // Blocks that start beside the last ones of a kernel before take what room there is, and lie unevenly: worth it only where all have room, or many rounds follow
  // (300 rows of 128256 in fp32 45.8 us that way, 37.3 without; 400 in bf16 41.3, 34.8)
  const long long blocks = (long long)a.T * NC;
  if (pdl_enabled() && (blocks <= 2 * sms || blocks > 8 * sms)) {
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
  // Blocks per row: twice as many while a block keeps seven steps and not all SMs have one (up to four per row: some three, where a row has 24 steps).  us with 1 | 2 | 4 | 8
  // blocks per row: 8 x 128256 fp32 20.0 | 14.5 | 11.1 | 10.6, 32 rows 21.3 | 16.2 | 13.3 | 14.7, 64 rows 21.7 | 16.9 | 14.9 | 20.1, 100 rows 21.9 | 19.8 | 18.6, 150 rows
  // 26.5 | 24.0 | 28.2, 250 rows 29.2 | 31.0 | 36.2; 100 x 32768 9.8 | 10.7 | 11.0 | 20.6.  Blocks of twice the threads, or that fetch eight steps ahead, where few blocks run:
  // the same within a tenth either way
  int nc = 1;
  constexpr long long kStepOf = (long long)kThreads * kEntries<F32>;
  auto more = [&](int to) { return a.V >= 7 * to * kStepOf && (long long)a.T * to <= (to <= 4 && a.V >= 24 * kStepOf ? 11LL * sms / 4 : sms); };
  while (nc < 8 && more(nc * 2)) nc *= 2;
  switch (nc) {
    case 1: return launch_nc<F32, 1, TOP>(stream, a, sms);
    case 2: return launch_nc<F32, 2, TOP>(stream, a, sms);
    case 4: return launch_nc<F32, 4, TOP>(stream, a, sms);
    default: return launch_nc<F32, 8, TOP>(stream, a, sms);
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

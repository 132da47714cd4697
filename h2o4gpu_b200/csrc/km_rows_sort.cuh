// Places of rows sorted by cluster.
// Entry i = t n + j says that row t goes to cluster ids[i] (outside [0, k): nowhere).  A stable counting sort gives every entry
// its place: groups in the clusters' order, each beginning on a multiple of `align`, entries of a group in their own order.
//   slot[i] = place of entry i (-1: none);  source[p] = entry at place p (-1: padding)
#pragma once

#include "km_rows.cuh"

namespace km {
namespace rows {

constexpr int kSortThreads = 512;
constexpr int kSortMaxK = 16384;          // three tables of k words have to fit the shared memory
constexpr size_t kSortTables = 196608;    // bytes of those tables

// How one call is cut: `blocks` CTAs of `chunk` entries each, in order; `warps` warps of a CTA keep counts of their own.
struct SortPlan {
  int blocks = 1, warps = 1;
  int chunk = 0;
};
inline SortPlan sort_plan(long long entries, int k, int sms) {
  SortPlan p;
  // One CTA, one launch, up to 2048 entries.  Else as many as there are processors, with two entries a thread or more, and so few that what
  // all of them read of each other's counts (blocks^2 x k words, from L2) stays below 64 MB.
  long long most = std::min<long long>(sms, entries / (2 * kSortThreads));
  while (most > 1 && most * most * k > (16 << 20)) --most;
  p.blocks = (int)std::max<long long>(1, most);
  p.chunk = (int)((entries + p.blocks - 1) / p.blocks);
  p.warps = kSortThreads / 32;
  while (p.warps > 1 && (size_t)(p.warps + 2) * k * 4 > kSortTables) p.warps /= 2;
  return p;
}

// Entry i's cluster; entries lie side by side (stride n) but for strided ids.
__device__ __forceinline__ int sort_id(const int* ids, long long stride, int n, int i, int k) {
  const int id = ids[stride == n ? (long long)i : (i / n) * stride + i % n];
  return id >= 0 && id < k ? id : -1;
}

// Entries of each cluster in every chunk: part[block * k + cluster].
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const int* ids, long long stride, int n, int entries, int k, int chunk, int* part) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e < k; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const int i0 = blockIdx.x * chunk, i1 = min((long long)entries, (long long)i0 + chunk);
  for (int i = i0 + threadIdx.x; i < i1; i += kSortThreads) {
    const int id = sort_id(ids, stride, n, i, k);
    if (id >= 0) atomicAdd(&hist[id], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < k; e += kSortThreads) part[(size_t)blockIdx.x * k + e] = hist[e];
}

// Exclusive prefix sum of v over the CTA's threads, and the total.
__device__ __forceinline__ int cta_scan(int v, int* red, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) red[warp] = s;
  __syncthreads();
  if (warp == 0) {
    int r = lane < kSortThreads / 32 ? red[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(0xffffffffu, r, o);
      if (lane >= o) r += u;
    }
    red[lane] = r;
  }
  __syncthreads();
  const int base = warp ? red[warp - 1] : 0;
  *total = red[kSortThreads / 32 - 1];
  __syncthreads();
  return base + s - v;
}

// Places of one chunk's entries.  131,072 entries of 64 clusters: 10 us, and 3.4 for the counts before; latency of its steps.  Integer counts only: the order of the shared-memory additions does not matter, and the
// ranks inside a warp come from the lanes' order.
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const int* ids, long long stride, int n, int entries, int k, int align, SortPlan plan, const int* part,
                  int* offsets, int* counts, int* slot, int* source, int capacity) {
  extern __shared__ int tables[];
  __shared__ int red[32];
  int* wcnt = tables;                                 // [warps][k]: entries of each cluster per warp, then the next place
  int* sum = tables + (size_t)plan.warps * k;         // [k]: entries of each cluster
  int* earlier = sum + k;                             // [k]: of those, in the chunks before this one
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x;
  for (int i = threadIdx.x; i < (plan.warps + 2) * k; i += kSortThreads) tables[i] = 0;
  __syncthreads();
  const int c0 = b * plan.chunk, c1 = (int)min((long long)entries, (long long)c0 + plan.chunk);
  const int per = ((plan.chunk + plan.warps - 1) / plan.warps + 31) / 32 * 32;
  const int w0 = (int)min((long long)c1, (long long)c0 + (long long)warp * per), w1 = (int)min((long long)c1, (long long)w0 + per);
  if (warp < plan.warps)
    for (int i = w0 + lane; i < w1; i += 32) {
      const int id = sort_id(ids, stride, n, i, k);
      if (id >= 0) atomicAdd(&wcnt[(size_t)warp * k + id], 1);
    }
  // every CTA adds up all chunks' counts, so that nothing has to wait for another CTA
  if (part) {
    wait_for_previous();
    const int words = plan.blocks * k, before = b * k;
#pragma unroll 4
    for (int i = threadIdx.x; i < words; i += kSortThreads) {
      const int v = part[i], e = i % k;
      if (v) {
        atomicAdd(&sum[e], v);
        if (i < before) atomicAdd(&earlier[e], v);
      }
    }
  }
  __syncthreads();
  int base = 0;
  for (int e0 = 0; e0 < k; e0 += kSortThreads) {
    const int e = e0 + threadIdx.x;
    int all = 0, before = 0;
    if (e < k) {
      if (part) {
        all = sum[e];
        before = earlier[e];
      } else {
        for (int w = 0; w < plan.warps; ++w) all += wcnt[(size_t)w * k + e];
      }
    }
    const int padded = (all + align - 1) / align * align;
    int total;
    const int at = base + cta_scan(e < k ? padded : 0, red, &total);
    if (e < k) {
      if (b == 0) {
        offsets[e] = at;
        counts[e] = all;
      }
      // this CTA's share of the padding behind the groups
      if (e % plan.blocks == b)
        for (int p = at + all; p < at + padded; ++p) source[p] = -1;
      int next = at + before;
      for (int w = 0; w < plan.warps; ++w) {
        const int v = wcnt[(size_t)w * k + e];
        wcnt[(size_t)w * k + e] = next;
        next += v;
      }
    }
    base += total;
  }
  if (b == 0 && threadIdx.x == 0) offsets[k] = base;
  for (long long p = base + (long long)b * kSortThreads + threadIdx.x; p < capacity; p += plan.blocks * kSortThreads) source[p] = -1;
  __syncthreads();
  if (warp < plan.warps)
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      const int id = i < w1 ? sort_id(ids, stride, n, i, k) : -1;
      const unsigned int same = __match_any_sync(0xffffffffu, id);
      int place = -1;
      if (id >= 0) place = wcnt[(size_t)warp * k + id] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (id >= 0 && lane == __ffs(same) - 1) wcnt[(size_t)warp * k + id] += __popc(same);
      __syncwarp();
      if (i < w1) {
        slot[i] = place;
        if (place >= 0) source[place] = i;
      }
    }
}

}  // namespace rows
}  // namespace km

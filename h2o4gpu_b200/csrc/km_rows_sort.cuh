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
  long long chunk = 0;
};
inline SortPlan sort_plan(long long entries, int k, int sms) {
  SortPlan p;
  // One CTA, one launch, while counting on a second one would cost more than it saves; else as many as there are
  // processors, each with enough entries that reading the others' counts (blocks x k words) stays small beside them.
  const long long per = std::max<long long>(4096, k);
  p.blocks = (int)std::min<long long>(sms, std::max<long long>(1, entries / per));
  p.chunk = (entries + p.blocks - 1) / p.blocks;
  p.warps = kSortThreads / 32;
  while (p.warps > 1 && (size_t)(p.warps + 1) * k * 4 > kSortTables) p.warps /= 2;
  return p;
}

__device__ __forceinline__ int sort_id(const int* ids, long long stride, int n, long long i, int k) {
  const int id = ids[n == 1 ? i * stride : (i / n) * stride + i % n];
  return id >= 0 && id < k ? id : -1;
}

// Entries of each cluster in every chunk: part[block * k + cluster].
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(const int* ids, long long stride, int n, long long entries, int k, long long chunk, int* part) {
  extern __shared__ int hist[];
  for (int e = threadIdx.x; e < k; e += kSortThreads) hist[e] = 0;
  __syncthreads();
  const long long i1 = min(entries, (blockIdx.x + 1) * chunk);
  for (long long i = blockIdx.x * chunk + threadIdx.x; i < i1; i += kSortThreads) {
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

// Places of one chunk's entries.  Integer counts only: the order of the shared-memory additions does not matter, and the
// ranks inside a warp come from the lanes' order.
__global__ void __launch_bounds__(kSortThreads)
sort_place_kernel(const int* ids, long long stride, int n, long long entries, int k, int align, SortPlan plan, const int* part,
                  int* offsets, int* counts, int* slot, int* source, long long capacity) {
  extern __shared__ int tables[];
  __shared__ int red[32];
  int* wcnt = tables;                       // [warps][k]: entries of each cluster per warp, then the next place
  int* start = tables + (size_t)plan.warps * k;   // [k]: where the group starts
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b = blockIdx.x;
  for (int i = threadIdx.x; i < plan.warps * k; i += kSortThreads) wcnt[i] = 0;
  __syncthreads();
  const long long c0 = b * plan.chunk, c1 = min(entries, c0 + plan.chunk);
  const long long per = (plan.chunk + plan.warps - 1) / plan.warps;
  const long long w0 = min(c1, c0 + warp * per), w1 = min(c1, w0 + per);
  if (warp < plan.warps)
    for (long long i = w0 + lane; i < w1; i += 32) {
      const int id = sort_id(ids, stride, n, i, k);
      if (id >= 0) atomicAdd(&wcnt[(size_t)warp * k + id], 1);
    }
  __syncthreads();
  // group starts: every CTA adds up all chunks' counts, so that nothing has to wait for another CTA
  int base = 0;
  for (int e0 = 0; e0 < k; e0 += kSortThreads) {
    const int e = e0 + threadIdx.x;
    int all = 0, before = 0;
    if (e < k) {
      if (part) {
        for (int c = 0; c < plan.blocks; ++c) {
          const int v = part[(size_t)c * k + e];
          all += v;
          if (c < b) before += v;
        }
      } else {
        for (int w = 0; w < plan.warps; ++w) all += wcnt[(size_t)w * k + e];
      }
    }
    const int padded = (all + align - 1) / align * align;
    int total;
    const int at = base + cta_scan(e < k ? padded : 0, red, &total);
    if (e < k) {
      start[e] = at;
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
  for (long long p = base + (long long)b * kSortThreads + threadIdx.x; p < capacity; p += (long long)plan.blocks * kSortThreads)
    source[p] = -1;
  __syncthreads();
  if (warp < plan.warps)
    for (long long i0 = w0; i0 < w1; i0 += 32) {
      const long long i = i0 + lane;
      const int id = i < w1 ? sort_id(ids, stride, n, i, k) : -1;
      const unsigned int same = __match_any_sync(0xffffffffu, id);
      int place = -1;
      if (id >= 0) place = wcnt[(size_t)warp * k + id] + __popc(same & ((1u << lane) - 1u));
      __syncwarp();
      if (id >= 0 && lane == __ffs(same) - 1) wcnt[(size_t)warp * k + id] += __popc(same);
      __syncwarp();
      if (i < w1) {
        slot[i] = place;
        if (place >= 0) source[place] = (int)i;
      }
    }
}

}  // namespace rows
}  // namespace km

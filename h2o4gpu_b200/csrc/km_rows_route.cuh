// From scores to the n best clusters of a row and their weights, and the gradient of that.
// With the score's quality q = s (scale > 0) or -s (scale < 0), the clusters are taken by descending q, ties to the lowest
// index; a NaN and an infinitely bad score are never taken, an infinitely good one counts as the largest finite number.
//   z_e = exp(|scale| (q_e - q_best)),  weight = z / total,  total = sum of z over the taken clusters, or over all
// The difference is taken before the scale: two near distances subtract exactly, their scaled values would each be rounded.
//   c = sum over the taken of weight * dweight
//   over the taken: ds = scale * weight (dweight - c) at the taken, 0 elsewhere;  over all: ds_e = scale * p_e (dweight_e - c)
#pragma once

#include "km_rows.cuh"

namespace km {
namespace rows {

constexpr int kRouteMax = 32;    // clusters a row can take
constexpr int kRouteWarps = 8;

// A score as a number that orders: larger is better, 0 = cannot be taken.  (float bits of a positive number order as
// integers, those of a negative one the other way round; the largest finite number maps below 0xffffffff.)
__device__ __forceinline__ unsigned int route_order(float q) {
  if (!(q > -INFINITY)) return 0u;                       // NaN too
  q = fminf(q, 3.402823466e38f) + 0.f;                   // -0 becomes +0: they tie
  const unsigned int u = __float_as_uint(q);
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float route_quality(unsigned int o) {
  return __uint_as_float((o & 0x80000000u) ? o & 0x7fffffffu : ~o);
}
// quality in the upper word, the complement of the index in the lower: one comparison decides, ties to the lowest index
__device__ __forceinline__ unsigned long long route_key(float q, int e) {
  const unsigned int o = route_order(q);
  return o ? ((unsigned long long)o << 32) | (unsigned int)~e : 0ULL;
}
__device__ __forceinline__ unsigned long long warp_max_key(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long u = __shfl_xor_sync(0xffffffffu, v, o);
    v = u > v ? u : v;
  }
  return v;
}

// One warp per row: n passes over the scores, each for the best key below the last one.
template <typename T>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_kernel(const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all, int* ids, float* weights,
             float* best, float* total) {
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= rows) return;
  const T* sr = s + (long long)t * rs;
  const float sign = scale > 0.f ? 1.f : -1.f, a = fabsf(scale);
  unsigned long long last = ~0ULL, mine = 0ULL;
  for (int j = 0; j < n; ++j) {
    unsigned long long m = 0ULL;
    for (int e = lane; e < k; e += 32) {
      const unsigned long long key = route_key(sign * to_f(sr[e * cs]), e);
      if (key < last && key > m) m = key;
    }
    m = warp_max_key(m);
    if (lane == j) mine = m;
    last = m;
  }
  const float q = route_quality((unsigned int)(mine >> 32));
  const float q0 = __shfl_sync(0xffffffffu, mine ? q : 0.f, 0);
  const float z = mine ? expf(a * (q - q0)) : 0.f;
  float sum = z;
  if (over_all) {
    sum = 0.f;
    for (int e = lane; e < k; e += 32) {
      const unsigned int o = route_order(sign * to_f(sr[e * cs]));
      if (o) sum += expf(a * (route_quality(o) - q0));
    }
  }
  sum = warp_sum_f(sum);
  if (lane < n) {
    ids[(long long)t * n + lane] = mine ? (int)~(unsigned int)mine : -1;
    weights[(long long)t * n + lane] = mine ? z / sum : 0.f;
  }
  if (lane == 0) {
    best[t] = sign * q0;
    total[t] = sum;
  }
}

template <typename T>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_grad_kernel(const float* dweights, const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all,
                  const int* ids, const float* weights, const float* best, const float* total, T* ds, long long drs, long long dcs) {
  const int lane = threadIdx.x & 31;
  const int t = blockIdx.x * kRouteWarps + (threadIdx.x >> 5);
  if (t >= rows) return;
  int id = -1;
  float w = 0.f, g = 0.f;
  if (lane < n) {
    id = ids[(long long)t * n + lane];
    w = weights[(long long)t * n + lane];
    g = dweights[(long long)t * n + lane];
    if (id < 0 || id >= k) { id = -1; w = 0.f; g = 0.f; }
  }
  const float c = warp_sum_f(id >= 0 ? w * g : 0.f);
  T* dr = ds + (long long)t * drs;
  const float sign = scale > 0.f ? 1.f : -1.f, a = fabsf(scale);
  const float q0 = over_all ? sign * best[t] : 0.f, sum = over_all ? total[t] : 0.f;
  for (int e0 = 0; e0 < k; e0 += 32) {
    const int e = e0 + lane;
    float ge = 0.f, we = 0.f;
    bool taken = false;
    for (int j = 0; j < n; ++j) {
      const int idj = __shfl_sync(0xffffffffu, id, j);
      const float gj = __shfl_sync(0xffffffffu, g, j), wj = __shfl_sync(0xffffffffu, w, j);
      if (idj == e) { taken = true; ge = gj; we = wj; }
    }
    if (e >= k) continue;
    float v = taken ? scale * we * (ge - c) : 0.f;
    if (over_all) {
      const unsigned int o = route_order(sign * to_f(s[(long long)t * rs + e * cs]));
      v = o && sum > 0.f ? scale * (expf(a * (route_quality(o) - q0)) / sum) * (ge - c) : 0.f;
    }
    dr[e * dcs] = from_f<T>(v);
  }
}

}  // namespace rows
}  // namespace km

// From scores to the n best clusters of a row and their weights, and the gradient of that.
// With the score's quality q = s (scale > 0) or -s (scale < 0), the clusters are taken by descending q, ties to the lowest
// index; a NaN and an infinitely bad score are never taken, an infinitely good one counts as the largest finite number.
//   z_e = exp(|scale| (q_e - q_best)),  weight = z / total,  total = sum of z over the taken clusters, or over all
// The difference is taken before the scale: two near distances subtract exactly, their scaled values would each be rounded.
//   c = sum over the taken of weight * dweight
//   over the taken: ds = scale * weight (dweight - c) at the taken, 0 elsewhere;  over all: ds_e = scale * p_e (dweight_e - c)
#pragma once

#include "km_rows_vec.cuh"

namespace km {
namespace rows {

constexpr int kRouteMax = 32;    // clusters a row can take
constexpr int kRouteMaxK = 1 << 24;

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


// A score's quality: larger is better, -inf cannot be taken.
template <typename T>
__device__ __forceinline__ float route_value(T s, float sign) {
  return fminf(fmaxf(sign * to_f(s), -INFINITY), 3.402823466e38f);      // (the maximum of NaN and a number is the number)
}

// exp(x), x <= 0, for sums of many terms: 2^(x log2 e) with the product rounded once more than in expf, which puts |x| 2^-24 of a term
// on top - at most 0.4 2^-24 of the largest one, as x e^-x is - for a third of the instructions.
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
constexpr float kLog2E = 1.44269504f;

// Both kernels find the n best of a row without sorting it: the maxima of some groups of its scores give a bound that the n best reach
// (the n-th largest of the maxima), and few scores besides them do.  Those are collected, and only they are put in order.

// ---- one lane per row: scores that lie cluster after cluster, and rows too short for a warp ---------------------------------------------
// `split` warps share the clusters of 32 rows, each a run of them.
constexpr int kRouteGroup = 8;      // scores of a group, and loads on their way together
constexpr int kRouteList = 16;      // collected scores of a lane

// Puts (q, e) into a list of N sorted by descending quality; e is above all entries' clusters, so ties stay in front.
template <int N>
__device__ __forceinline__ void route_insert(float (&v)[N], int (&id)[N], float q, int e) {
  if (!(q > v[N - 1])) return;
#pragma unroll
  for (int j = N - 1; j >= 0; --j) {
    const bool here = q > v[j], above = j > 0 && q > v[j > 0 ? j - 1 : 0];
    if (here) {      // everything from its place on moves down by one
      v[j] = above ? v[j > 0 ? j - 1 : 0] : q;
      id[j] = above ? id[j > 0 ? j - 1 : 0] : e;
    }
  }
}
// The same for values alone.
template <int N>
__device__ __forceinline__ void route_insert(float (&v)[N], float q) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const float lo = fminf(v[j], q);
    v[j] = fmaxf(v[j], q);
    q = lo;
  }
}

template <typename T, int N>
__global__ void __launch_bounds__(512)
route_lane_kernel(const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all, int split, int* ids,
                  float* weights, float* best, float* total) {
  extern __shared__ float2 shared[];       // the lanes' lists, then what the warps of a tile tell each other
  const int lane = threadIdx.x, warp = threadIdx.y, part = warp % split;
  const long long tile = (long long)blockIdx.x * (blockDim.y / split) + warp / split;
  const int t = (int)min(tile * 32 + lane, (long long)rows - 1);     // a lane behind the last row works on that row and writes nothing
  const bool valid = tile * 32 + lane < rows;
  const T* sr = s + t * rs;
  const float sign = scale > 0.f ? 1.f : -1.f, a = fabsf(scale);
  const int per = ((k + split - 1) / split + kRouteGroup - 1) / kRouteGroup * kRouteGroup;
  const int c0 = min(k, part * per), c1 = min(k, c0 + per);
  float v[N];
  int id[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    v[j] = -INFINITY;
    id[j] = -1;
  }
  float first = -INFINITY, sum = 0.f;
  // f(score, cluster) over this warp's clusters, a group's loads together; then ends() of the group
  const auto walk = [&](auto f, auto ends) {
    const T* p = sr + c0 * cs;
    for (int c = c0; c < c1; c += kRouteGroup) {
      T raw[kRouteGroup];
      if (c + kRouteGroup <= c1) {
#pragma unroll
        for (int u = 0; u < kRouteGroup; ++u, p += cs) raw[u] = *p;
#pragma unroll
        for (int u = 0; u < kRouteGroup; ++u) f(raw[u], c + u);
      } else {
#pragma unroll
        for (int u = 0; u < kRouteGroup; ++u)
          if (c + u < c1) raw[u] = p[u * cs];
#pragma unroll
        for (int u = 0; u < kRouteGroup; ++u)
          if (c + u < c1) f(raw[u], c + u);
      }
      ends();
    }
  };
  // no bound to be had from one score, nor from fewer groups than are taken: one walk
  const bool direct = N == 1 || k <= kRouteGroup * N;
  if (direct) {
    walk([&](T r, int e) { route_insert(v, id, route_value(r, sign), e); }, [] {});
    first = v[0];
  } else {
    float m[N], g = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) m[j] = -INFINITY;
    walk([&](T r, int) { g = fmaxf(g, sign * to_f(r)); },      // (which leaves NaN out)
         [&] { route_insert(m, fminf(g, 3.402823466e38f)); g = -INFINITY; });
    if (split > 1) {      // the bound of all the row's groups
      float* told = reinterpret_cast<float*>(shared);
#pragma unroll
      for (int j = 0; j < N; ++j) told[(warp * N + j) * 32 + lane] = m[j];
      __syncthreads();
      for (int w = warp - part; w < warp - part + split; ++w)
        if (w != warp)
          for (int j = 0; j < N; ++j) route_insert(m, told[(w * N + j) * 32 + lane]);
      __syncthreads();
    }
    first = m[0];
    const float bound = fmaxf(m[N - 1], -3.402823466e38f);      // anything but -inf while fewer than N groups have one
    float2* list = shared + (warp * 32 + lane);
    const int stride = blockDim.y * 32;
    int have = 0;
    const auto put = [&] {
      for (int i = 0; i < have; ++i) {
        const float2 o = list[i * stride];
        route_insert(v, id, o.x, __float_as_int(o.y));
      }
      have = 0;
    };
    walk([&](T r, int e) {
      const float q = sign * to_f(r);
      if (q >= bound) list[have++ * stride] = make_float2(fminf(q, 3.402823466e38f), __int_as_float(e));
    }, [&] { if (have > kRouteList - kRouteGroup) put(); });
    put();
  }
  if (split > 1) {       // the tile's first warp joins the others' lists, in the clusters' order
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) shared[(warp * N + j) * 32 + lane] = make_float2(v[j], __int_as_float(id[j]));
    __syncthreads();
    if (part == 0)
      for (int w = warp + 1; w < warp + split; ++w)
        for (int j = 0; j < N; ++j) {
          const float2 o = shared[(w * N + j) * 32 + lane];
          route_insert(v, id, o.x, __float_as_int(o.y));
        }
    if (direct) {       // what the sums below start from
      __syncthreads();
      if (part == 0) reinterpret_cast<float*>(shared)[warp * 32 + lane] = v[0];
      __syncthreads();
      first = reinterpret_cast<float*>(shared)[(warp - part) * 32 + lane];
    }
  }
  const float q0 = first > -INFINITY ? first : 0.f;
  if (over_all) {
    const float a2 = a * kLog2E;
    walk([&](T r, int) { sum += exp2_fast(a2 * (route_value(r, sign) - q0)); }, [] {});
    if (split > 1) {
      __syncthreads();
      reinterpret_cast<float*>(shared)[warp * 32 + lane] = sum;
      __syncthreads();
      if (part == 0)
        for (int w = warp + 1; w < warp + split; ++w) sum += reinterpret_cast<float*>(shared)[w * 32 + lane];
    }
  }
  if (part != 0 || !valid) return;
  float z[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    z[j] = id[j] >= 0 ? expf(a * (v[j] - q0)) : 0.f;
    if (!over_all && j < n) sum += z[j];
  }
#pragma unroll
  for (int j = 0; j < N; ++j)
    if (j < n) {
      ids[(long long)t * n + j] = id[j];
      weights[(long long)t * n + j] = id[j] >= 0 ? z[j] / sum : 0.f;
    }
  best[t] = sign * q0;
  total[t] = sum;
}

// ---- one warp per row: scores that lie row after row ---------------------------------------------------------------------------------
// The groups are the lanes.  HELD pieces of 16 bytes a lane stay in registers; 0: longer rows, read a second time (from L2).
constexpr int kRouteWarps = 8;

template <typename T, int HELD, bool ALIGNED>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_warp_kernel(const T* s, long long rs, Span<T> in, int rows, int k, int n, float scale, bool over_all, int* ids, float* weights,
                  float* best, float* total) {
  constexpr int V = Piece<T>::V;
  __shared__ unsigned long long lists[kRouteWarps][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x / 32;
  const int t = blockIdx.x * kRouteWarps + warp;
  if (t >= rows) return;
  unsigned long long* list = lists[warp];
  const T* sr = s + (long long)t * rs;
  const float sign = scale > 0.f ? 1.f : -1.f, a = fabsf(scale);
  const int pieces = (k + V - 1) / V;
  const int per_lane = (pieces + 31) / 32;
  const T none = from_f<T>(-sign * INFINITY);
  const auto piece = [&](int i) {      // behind the row's end: scores that cannot be taken
    Piece<T> p = load_piece<T, ALIGNED>(sr, i, k, in);
    if ((i + 1) * V > k)
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (i * V + e >= k) p.e[e] = none;
    return p;
  };
  Piece<T> held[HELD ? HELD : 1];
#pragma unroll
  for (int h = 0; h < HELD; ++h) held[h] = piece(lane + h * 32);
  // f(a piece's signed scores, piece) over the row; every lane makes the same number of calls
  const auto walk = [&](auto f) {
    const auto call = [&](const Piece<T>& p, int i) {
      float2 q[V / 2];
      unpack(p, q);
#pragma unroll
      for (int e = 0; e < V / 2; ++e) q[e] = mul2(q[e], both(sign));
      f(q, i);
    };
    if (HELD) {
#pragma unroll
      for (int h = 0; h < HELD; ++h) call(held[h], lane + h * 32);
    } else {
#pragma unroll 2
      for (int i = lane; i < per_lane * 32; i += 32) call(piece(i), i);
    }
  };
  float m = -INFINITY;
  walk([&](const float2 (&q)[V / 2], int) {
#pragma unroll
    for (int e = 0; e < V / 2; ++e) m = fmaxf(m, fmaxf(q[e].x, q[e].y));      // (which leaves NaN out)
  });
  // the n-th largest of the lanes' maxima
  const unsigned int own = route_order(m);
  unsigned int o = own, top = 0, nth = 0;
  for (int j = 0; j < n; ++j) {
    const unsigned int w = __reduce_max_sync(0xffffffffu, o);
    if (j == 0) top = w;
    nth = w;
    if (w == 0) break;
    if (lane == __ffs(__ballot_sync(0xffffffffu, o == w)) - 1) o = 0;
  }
  const float q0 = top ? route_quality(top) : 0.f;
  const float bound = nth ? route_quality(nth) : -3.402823466e38f;
  // Only lanes whose maximum reaches the bound have scores that do: n of them, but for ties.  The warp looks through one such lane's
  // scores after the other (they come from L1).
  int have = 0;
  for (unsigned int lanes = __ballot_sync(0xffffffffu, own >= max(nth, 1u)); lanes; lanes &= lanes - 1) {
    const int l = __ffs(lanes) - 1;
    for (int u0 = 0; u0 < per_lane * V; u0 += 32) {
      const int u = u0 + lane, e = (l + u / V * 32) * V + u % V;
      const float q = u < per_lane * V && e < k ? sign * to_f(sr[e]) : -INFINITY;
      const unsigned int reach = __ballot_sync(0xffffffffu, q >= bound);
      const int at = have + __popc(reach & ((1u << lane) - 1u));
      if (q >= bound && at < 32) list[at] = route_key(q, e);
      have += __popc(reach);
    }
  }
  float sum = 0.f;
  if (over_all) {
    const float2 a2 = both(a * kLog2E), off = both(-q0);
    float2 s2 = both(0.f);
    const bool huge = q0 == 3.402823466e38f;      // perhaps an infinite one, which counts as this
    walk([&](float2 (&q)[V / 2], int) {
#pragma unroll
      for (int e = 0; e < V / 2; ++e) {
        if (huge) q[e] = make_float2(fminf(fmaxf(q[e].x, -INFINITY), q0), fminf(fmaxf(q[e].y, -INFINITY), q0));
        const float2 x = mul2(a2, add2(q[e], off));
        s2 = add2(s2, make_float2(exp2_fast(fmaxf(x.x, -INFINITY)), exp2_fast(fmaxf(x.y, -INFINITY))));
      }
    });
    sum = s2.x + s2.y;
  }
  __syncwarp();
  // `mine`: this lane's score among the n best, `place` where it goes; lanes without one fill the places behind
  unsigned long long mine = 0ULL;
  int place = 0;
  if (have <= 32) {
    mine = lane < have ? list[lane] : 0ULL;
    for (int i = 0; i < have; ++i) place += list[i] > mine;
    if (lane >= have) place = lane;
    if (place >= n) mine = 0ULL;
  } else {      // more reach the bound (ties): the best one below the last, n times
    unsigned long long last = ~0ULL;
    for (int j = 0; j < n; ++j) {
      unsigned long long b = 0ULL;
      walk([&](const float2 (&q)[V / 2], int i) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const unsigned long long key = route_key(e & 1 ? q[e / 2].y : q[e / 2].x, i * V + e);
          if (key < last && key > b) b = key;
        }
      });
      last = warp_max_key(b);
      if (lane == j) mine = last;
    }
    place = lane;
  }
  const float z = mine ? expf(a * (route_quality((unsigned int)(mine >> 32)) - q0)) : 0.f;
  sum = warp_sum_f(over_all ? sum : z);
  if (place < n) {
    ids[(long long)t * n + place] = mine ? (int)~(unsigned int)mine : -1;
    weights[(long long)t * n + place] = mine ? z / sum : 0.f;
  }
  if (lane == 0) {
    best[t] = sign * q0;
    total[t] = sum;
  }
}

// ---- the gradient ----------------------------------------------------------------------------------------------------------------------
// Every score's own part first (zero over the taken alone), then the taken ones' over it.

// One warp per row, 16-byte pieces.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kRouteWarps * 32)
route_grad_warp_kernel(const float* dweights, const T* s, long long rs, Span<T> in, int rows, int k, int n, float scale, bool over_all,
                       const int* ids, const float* weights, const float* best, const float* total, T* ds, long long drs) {
  constexpr int V = Piece<T>::V, H = V / 2;
  const int lane = threadIdx.x & 31, t = blockIdx.x * kRouteWarps + threadIdx.x / 32;
  if (t >= rows) return;
  int id = -1;
  float w = 0.f, g = 0.f;
  if (lane < n) {
    id = ids[(long long)t * n + lane];
    w = weights[(long long)t * n + lane];
    g = dweights[(long long)t * n + lane];
  }
  const bool taken = id >= 0 && id < k;
  const float c = warp_sum_f(taken ? w * g : 0.f);
  T* dr = ds + (long long)t * drs;
  const T* sr = over_all ? s + (long long)t * rs : nullptr;
  const float sign = scale > 0.f ? 1.f : -1.f, a = fabsf(scale);
  const float sum = over_all ? total[t] : 0.f, q0 = over_all ? sign * best[t] : 0.f, f = sum > 0.f ? -scale * c / sum : 0.f;
  const int pieces = ((k + V - 1) / V + 31) / 32 * 32;
  for (int i = lane; i < pieces; i += 32) {
    Piece<T> p;
    p.q = make_uint4(0u, 0u, 0u, 0u);
    if (over_all) {
      p = load_piece<T, ALIGNED>(sr, i, k, in);
      float2 o[H];
#pragma unroll
      for (int e = 0; e < H; ++e) {
        const float qx = route_value(p.e[2 * e], sign), qy = route_value(p.e[2 * e + 1], sign);
        o[e] = make_float2(qx > -INFINITY ? f * expf(a * (qx - q0)) : 0.f, qy > -INFINITY ? f * expf(a * (qy - q0)) : 0.f);
      }
      p = pack<T>(o);
    }
    store_piece<T, ALIGNED>(dr, i, k, p);
  }
  __syncwarp();
  if (taken) dr[id] = from_f<T>(scale * w * (g - c));
}

// One thread per row and run of clusters: scores that lie cluster after cluster, or in other strides.
constexpr int kRouteGradThreads = 128;
template <typename T>
__global__ void __launch_bounds__(kRouteGradThreads)
route_grad_lane_kernel(const float* dweights, const T* s, long long rs, long long cs, int rows, int k, int per, int n, float scale,
                       bool over_all, const int* ids, const float* weights, const float* best, const float* total, T* ds, long long drs,
                       long long dcs) {
  const long long at = (long long)blockIdx.x * kRouteGradThreads + threadIdx.x;
  if (at >= rows) return;
  const int t = (int)at, c0 = blockIdx.y * per, c1 = min(k, c0 + per);
  float c = 0.f;
  for (int j = 0; j < n; ++j) {
    const int id = ids[(long long)t * n + j];
    if (id >= 0 && id < k) c = fmaf(weights[(long long)t * n + j], dweights[(long long)t * n + j], c);
  }
  const float sign = scale > 0.f ? 1.f : -1.f, a = fabsf(scale);
  const float sum = over_all ? total[t] : 0.f, q0 = over_all ? sign * best[t] : 0.f, f = sum > 0.f ? -scale * c / sum : 0.f;
  const T* sr = s + t * rs;
  T* dr = ds + t * drs;
#pragma unroll 8
  for (int e = c0; e < c1; ++e) {
    float v = 0.f;
    if (over_all) {
      const float q = route_value(sr[e * cs], sign);
      if (q > -INFINITY) v = f * expf(a * (q - q0));
    }
    dr[e * dcs] = from_f<T>(v);
  }
  for (int j = 0; j < n; ++j) {
    const int id = ids[(long long)t * n + j];
    if (id >= c0 && id < c1) dr[id * dcs] = from_f<T>(scale * weights[(long long)t * n + j] * (dweights[(long long)t * n + j] - c));
  }
}

// ---- launches --------------------------------------------------------------------------------------------------------------------------

template <typename T>
int route_launch(const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all, int* ids, float* weights,
                 float* best, float* total, int sms, cudaStream_t stream) {
  // a lane per row where lanes' loads lie side by side, or a row is no longer than the line that its lane's loads share
  if (cs != 1 || (size_t)k * sizeof(T) <= 128 || (rs == 1 && rows > 1)) {
    const long long tiles = ((long long)rows + 31) / 32;
    int most = 16;
    while (most * n > 128) most /= 2;       // the lists that the warps of a tile exchange: 32 KB
    int split = 1;
    while (split < most && tiles * split < (long long)sms * 16 && k / split >= 64) split *= 2;
    const int warps = std::max(4, split), per_cta = warps / split;
    const auto launch = [&](auto count) -> int {
      constexpr int N = count();
      const size_t smem = sizeof(float2) * 32 * warps * std::max(N == 1 ? 1 : kRouteList, split > 1 ? N : 1);
      const auto fn = route_lane_kernel<T, N>;
      KM_CUDA(allow_smem(fn, smem));
      fn<<<(unsigned)((tiles + per_cta - 1) / per_cta), dim3(32, warps), smem, stream>>>(s, rs, cs, rows, k, n, scale, over_all, split,
                                                                                       ids, weights, best, total);
      KM_CUDA(cudaGetLastError());
      return KM_OK;
    };
    using std::integral_constant;
    if (n == 1) return launch(integral_constant<int, 1>());
    if (n == 2) return launch(integral_constant<int, 2>());
    if (n <= 4) return launch(integral_constant<int, 4>());
    if (n <= 8) return launch(integral_constant<int, 8>());
    if (n <= 16) return launch(integral_constant<int, 16>());
    return launch(integral_constant<int, 32>());
  }
  const bool al = rows_aligned(s, rs, rows, k, sizeof(T));
  const int pieces = (k + Piece<T>::V - 1) / Piece<T>::V;
  const auto pick = [&](auto aligned_) {
    constexpr bool AL = aligned_();
    return pieces <= 32 ? route_warp_kernel<T, 1, AL> : pieces <= 64 ? route_warp_kernel<T, 2, AL>
         : pieces <= 128 ? route_warp_kernel<T, 4, AL> : route_warp_kernel<T, 0, AL>;
  };
  const auto fn = al ? pick(std::true_type()) : pick(std::false_type());
  fn<<<(rows + kRouteWarps - 1) / kRouteWarps, kRouteWarps * 32, 0, stream>>>(s, rs, span_of<T>(s, rs, rows, k), rows, k, n, scale,
                                                                            over_all, ids, weights, best, total);
  KM_CUDA(cudaGetLastError());
  return KM_OK;
}

template <typename T>
int route_grad_launch(const float* dweights, const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all,
                      const int* ids, const float* weights, const float* best, const float* total, T* ds, long long drs, long long dcs,
                      int sms, cudaStream_t stream) {
  if (dcs == 1 && (!over_all || cs == 1)) {
    const bool al = rows_aligned(ds, drs, rows, k, sizeof(T)) && (!over_all || rows_aligned(s, rs, rows, k, sizeof(T)));
    const auto fn = al ? route_grad_warp_kernel<T, true> : route_grad_warp_kernel<T, false>;
    fn<<<(rows + kRouteWarps - 1) / kRouteWarps, kRouteWarps * 32, 0, stream>>>(
        dweights, s, rs, over_all ? span_of<T>(s, rs, rows, k) : Span<T>{nullptr, nullptr}, rows, k, n, scale, over_all, ids, weights,
        best, total, ds, drs);
    KM_CUDA(cudaGetLastError());
    return KM_OK;
  }
  // runs of clusters so long that a row's own values are read rarely, and enough of them to fill the device
  const long long tiles = ((long long)rows + kRouteGradThreads - 1) / kRouteGradThreads;
  int runs = 1;
  while (runs < 1024 && tiles * runs < (long long)sms * 16 && k / runs > 16) runs *= 2;
  const int per = (k + runs - 1) / runs;
  route_grad_lane_kernel<T><<<dim3((unsigned)tiles, (k + per - 1) / per), kRouteGradThreads, 0, stream>>>(
      dweights, s, rs, cs, rows, k, per, n, scale, over_all, ids, weights, best, total, ds, drs, dcs);
  KM_CUDA(cudaGetLastError());
  return KM_OK;
}

}  // namespace rows
}  // namespace km

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

// exp(x), x = a d <= 0, for sums of many terms, for a third of expf's instructions: 2^(a2 d) with a2 = a log2 e.  log2 e as a float32 is off by 0.22
// 2^-24 of itself, a2 and a2 d are rounded: the exponent is off by 2.22 |x| 2^-24 at most (1.22 where a is 1), which puts 0.82 2^-24 of the
// largest term on a term, as |x| e^x is below 0.37, besides ex2's own error.  (a2 stops at the largest
// float32, for scales above 2.3e38.)
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

// The outputs of row t from its list, best first; a lane's n values go out together where they fill whole words.
template <int N>
__device__ __forceinline__ void route_store(long long t, int n, const float (&v)[N], const int (&id)[N], float q0, float sum,
                                            bool over_all, float a, float sign, int* ids, float* weights, float* best, float* total) {
  float z[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    z[j] = id[j] >= 0 ? expf(a * (v[j] - q0)) : 0.f;
    if (!over_all && j < n) sum += z[j];
  }
#pragma unroll
  for (int j = 0; j < N; ++j) z[j] = id[j] >= 0 ? z[j] / sum : 0.f;
  int* it = ids + t * n;
  float* wt = weights + t * n;
  const bool whole = n == N && ((reinterpret_cast<uintptr_t>(ids) | reinterpret_cast<uintptr_t>(weights)) & (N >= 4 ? 15 : 4 * N - 1)) == 0;
  if (N >= 4 && whole) {
#pragma unroll
    for (int j = 0; j + 3 < N; j += 4) {
      *reinterpret_cast<int4*>(it + j) = make_int4(id[j], id[j + 1], id[j + 2], id[j + 3]);
      *reinterpret_cast<float4*>(wt + j) = make_float4(z[j], z[j + 1], z[j + 2], z[j + 3]);
    }
  } else if (N == 2 && whole) {
    *reinterpret_cast<int2*>(it) = make_int2(id[0], id[N - 1]);
    *reinterpret_cast<float2*>(wt) = make_float2(z[0], z[N - 1]);
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < n) {
        it[j] = id[j];
        wt[j] = z[j];
      }
  }
  best[t] = sign * q0;
  total[t] = sum;
}

template <typename T, int N>
__global__ void __launch_bounds__(512)
route_lane_kernel(const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all, int split, int share,
                  int* ids, float* weights, float* best, float* total) {
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
  if (N == 1) {
    walk([&](T r, int e) { route_insert(v, id, route_value(r, sign), e); }, [] {});
    first = v[0];
  } else {
    float m[N], g = -INFINITY;
#pragma unroll
    for (int j = 0; j < N; ++j) m[j] = -INFINITY;
    const auto end_group = [&] {
      route_insert(m, fminf(g, 3.402823466e38f));
      g = -INFINITY;
    };
    walk([&](T r, int e) {
           g = fmaxf(g, sign * to_f(r));      // (which leaves NaN out)
           if ((e + 1) % share == 0 && share < kRouteGroup) end_group();
         },
         [&] { end_group(); });
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
    if (N == 1) {       // what the sums below start from
      __syncthreads();
      if (part == 0) reinterpret_cast<float*>(shared)[warp * 32 + lane] = v[0];
      __syncthreads();
      first = reinterpret_cast<float*>(shared)[(warp - part) * 32 + lane];
    }
  }
  const float q0 = first > -INFINITY ? first : 0.f;
  if (over_all) {
    const float a2 = fminf(a * kLog2E, 3.402823466e38f);
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
  route_store<N>(t, n, v, id, q0, sum, over_all, a, sign, ids, weights, best, total);
}

// ---- one warp per row: scores that lie row after row ---------------------------------------------------------------------------------
// Bound by instructions, some 1,100 a row of 1000 bfloat16 scores, eight best, softmax over all: 32,768 rows take 45 us (10.4 by the bytes).
// The groups are the lanes.  HELD pieces of 16 bytes a lane stay in registers; 0: longer rows, read a second time (from L2).
constexpr int kRouteWarps = 8;

enum RouteRows { kAligned, kUnaligned, kStrided };
template <typename T, int HELD, RouteRows LIE>
__global__ void __launch_bounds__(kRouteWarps * 32, 4)
route_warp_kernel(const T* s, long long rs, long long cs, Span<T> in, int rows, int k, int n, float scale, bool over_all, int* ids, float* weights,
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
    Piece<T> p;
    if (LIE != kStrided) p = load_piece<T, LIE == kAligned>(sr, i, k, in);
    if (LIE == kStrided || (i + 1) * V > k)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        if (i * V + e >= k) p.e[e] = none;
        else if (LIE == kStrided) p.e[e] = sr[(i * V + e) * cs];
      }
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
  const int u_end = per_lane * V;
  for (unsigned int lanes = __ballot_sync(0xffffffffu, own >= max(nth, 1u)); lanes; lanes &= lanes - 1) {
    const int base = (__ffs(lanes) - 1) * V + lane / V * (32 * V) + lane % V;
    for (int u = 0; u < u_end; u += 32) {
      const int e = base + u * 32;
      const float q = u + lane < u_end && e < k ? sign * to_f(sr[LIE == kStrided ? e * cs : e]) : -INFINITY;
      const unsigned int reach = __ballot_sync(0xffffffffu, q >= bound);
      const int at = have + __popc(reach & ((1u << lane) - 1u));
      if (q >= bound && at < 32) list[at] = ((unsigned long long)__float_as_uint(q) << 32) | (unsigned int)e;
      have += __popc(reach);
    }
  }
  float sum = 0.f;
  if (over_all) {
    const float2 a2 = both(fminf(a * kLog2E, 3.402823466e38f)), off = both(-q0);
    float2 s2 = both(0.f);
    if (q0 < 3.402823466e38f) {
      walk([&](const float2 (&q)[V / 2], int) {
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float2 x = mul2(a2, add2(q[e], off));
          s2 = add2(s2, make_float2(exp2_fast(fmaxf(x.x, -INFINITY)), exp2_fast(fmaxf(x.y, -INFINITY))));
        }
      });
      sum = s2.x + s2.y;
    } else {      // perhaps an infinite one, which counts as the largest finite number
      for (int e = lane; e < k; e += 32) sum += exp2_fast(a2.x * (route_value(sr[LIE == kStrided ? e * cs : e], sign) - q0));
    }
  }
  __syncwarp();
  // `mine`: this lane's score among the n best, `place` where it goes; lanes without one fill the places behind
  unsigned long long mine = 0ULL;
  int place = 0;
  if (have <= 32) {
    if (lane < have) {
      mine = list[lane];
      mine = route_key(__uint_as_float((unsigned int)(mine >> 32)), (int)(unsigned int)mine);
    }
    __syncwarp();
    list[lane] = mine;
    __syncwarp();
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

// ---- one lane per row, the scores of 32 rows in shared memory --------------------------------------------------------------------------
// What a row costs besides its scores is then paid once for 32 rows.  Bound by instructions, 32 a score and lane: the four nearest of 100
// float32 distances of 300,000 rows take 39.9 us (20.2 by the bytes).  `split` warps share a tile, each a run of its groups; the warps then
// tell each other a bound and join their lists.
//   BY_ROW: row r at r * stride bytes (an odd number of 16-byte words: lanes read those without bank conflicts); a group is 8 scores of it
//   else:   cluster e's 32 scores at e * 32
constexpr size_t kRouteTileBytes = 100 << 10;      // two CTAs a processor
// Rows of some 1 KB: a warp per row costs the same whatever the row's length up to 2 KB, a lane per row grows with it.  8 of 256 float32 of
// 65,536 rows 37 us with a lane per row and 63 with a warp, of 512 bfloat16 47 and 66, of 512 float32 78 and 71, of 1000 bfloat16 (32,768
// rows) 50 and 41.
constexpr size_t kRouteRowTileBytes = 40 << 10;
template <typename T>
struct RouteTile {
  static constexpr int G = kRouteGroup, WORDS = G * (int)sizeof(T) / 16;      // 16-byte words of a group
  static int groups(int k) { return (k + G - 1) / G; }
  static int stride(int k) { return (groups(k) * WORDS | 1) * 16; }
  static size_t bytes(int k, bool by_row) { return by_row ? (size_t)32 * stride(k) : (size_t)groups(k) * G * 32 * sizeof(T); }
};

template <typename T, int N, bool BY_ROW>
__global__ void __launch_bounds__(512)
route_tile_kernel(const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all, int split, int share,
                  int tile_bytes, int* ids, float* weights, float* best, float* total) {
  using Tile = RouteTile<T>;
  constexpr int G = Tile::G, WORDS = Tile::WORDS, V = Piece<T>::V;
  extern __shared__ uint4 tiles[];
  const int lane = threadIdx.x, warp = threadIdx.y, part = warp % split, per_cta = blockDim.y / split;
  const long long row0 = ((long long)blockIdx.x * per_cta + warp / split) * 32;
  unsigned char* tile = reinterpret_cast<unsigned char*>(tiles) + (size_t)(warp / split) * tile_bytes;
  float2* shared = reinterpret_cast<float2*>(reinterpret_cast<unsigned char*>(tiles) + (size_t)per_cta * tile_bytes);
  const int here = (int)max(0LL, min(32LL, rows - row0));     // rows of the tile
  const int groups = (k + G - 1) / G, stride = (groups * WORDS | 1) * 16;
  const float sign = scale > 0.f ? 1.f : -1.f, a = fabsf(scale);
  const T none = from_f<T>(-sign * INFINITY);
  T* flat = reinterpret_cast<T*>(tile);
  if (BY_ROW) {
    const int words = k / V;      // the rows are whole words
    for (int r = part; r < here; r += split) {
      const uint4* from = reinterpret_cast<const uint4*>(s + (row0 + r) * rs);
      uint4* to = reinterpret_cast<uint4*>(tile + (size_t)r * stride);
      for (int i = lane; i < words; i += 32) copy_async(to + i, from + i);
      for (int e = k + lane; e < groups * G; e += 32) reinterpret_cast<T*>(to)[e] = none;
    }
  } else {
    constexpr int PER = 32 * (int)sizeof(T) / 16, AT_ONCE = 32 / PER;      // words of a cluster's 32 scores, clusters a step
    if (here == 32) {
      const T* from = s + row0 + lane % PER * V;
      uint4* to = reinterpret_cast<uint4*>(tile) + lane;
      for (int e = part * AT_ONCE + lane / PER; e < k; e += split * AT_ONCE)
        copy_async(to + (e - lane / PER) * PER, reinterpret_cast<const uint4*>(from + e * cs));
    } else if (lane < here) {
      for (int e = part; e < k; e += split) flat[e * 32 + lane] = s[row0 + lane + e * cs];
    }
    for (int e = k + part; e < groups * G; e += split) flat[e * 32 + lane] = none;
  }
  copies_commit();
  copies_wait<0>();
  __syncthreads();

  // the signed scores of a group
  const auto group = [&](int g, float2 (&q)[G / 2]) {
    if (BY_ROW) {
      const uint4* w = reinterpret_cast<const uint4*>(tile + (size_t)lane * stride) + g * WORDS;
#pragma unroll
      for (int i = 0; i < WORDS; ++i) {
        Piece<T> p;
        p.q = w[i];
        float2 f[V / 2];
        unpack(p, f);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) q[i * (V / 2) + e] = f[e];
      }
    } else {
      const T* w = flat + g * (G * 32) + lane;
#pragma unroll
      for (int e = 0; e < G / 2; ++e) q[e] = make_float2(to_f(w[2 * e * 32]), to_f(w[(2 * e + 1) * 32]));
    }
#pragma unroll
    for (int e = 0; e < G / 2; ++e) q[e] = mul2(q[e], both(sign));
  };
  const int per = (groups + split - 1) / split, g0 = min(groups, part * per), g1 = min(groups, g0 + per);
  constexpr float kHuge = 3.402823466e38f;
  float m[N];
#pragma unroll
  for (int j = 0; j < N; ++j) m[j] = -INFINITY;
  for (int g = g0; g < g1; ++g) {
    float2 q[G / 2];
    group(g, q);
    if (share == 1) {
#pragma unroll
      for (int e = 0; e < G / 2; ++e) {
        route_insert(m, fminf(fmaxf(q[e].x, -INFINITY), kHuge));
        route_insert(m, fminf(fmaxf(q[e].y, -INFINITY), kHuge));
      }
      continue;
    }
    float x[G / 2];
#pragma unroll
    for (int e = 0; e < G / 2; ++e) x[e] = fminf(fmaxf(fmaxf(q[e].x, q[e].y), -INFINITY), kHuge);      // (which leaves NaN out)
    if (share == 2) {
#pragma unroll
      for (int e = 0; e < G / 2; ++e) route_insert(m, x[e]);
    } else if (share == 4) {
      route_insert(m, fmaxf(x[0], x[1]));
      route_insert(m, fmaxf(x[2], x[3]));
    } else {
      route_insert(m, fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])));
    }
  }
  float bound = m[N - 1], first = m[0];
  if (split > 1) {      // the N-th largest of the warps' largest maxima, some two times N of them
    const int told = min(N, max(1, 2 * N / split));
    float* out = reinterpret_cast<float*>(shared);
#pragma unroll
    for (int j = 0; j < N; ++j)
      if (j < told) out[(warp * N + j) * 32 + lane] = m[j];
    __syncthreads();
    float b[N];
#pragma unroll
    for (int j = 0; j < N; ++j) b[j] = -INFINITY;
    for (int w = warp - part; w < warp - part + split; ++w)
      for (int j = 0; j < told; ++j) route_insert(b, out[(w * N + j) * 32 + lane]);
    bound = b[N - 1];
    first = b[0];
    __syncthreads();
  }
  bound = fmaxf(bound, -kHuge);
  // the scores that reach the bound, in the clusters' order, and of them the n best
  float v[N];
  int id[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    v[j] = -INFINITY;
    id[j] = -1;
  }
  const int list_stride = blockDim.y * 32;
  unsigned short* const list = reinterpret_cast<unsigned short*>(shared) + (warp * 32 + lane);
  unsigned short* end = list;
  const auto put = [&] {
    for (const unsigned short* i = list; i != end; i += list_stride) {
      const int e = *i;
      route_insert(v, id, route_value(BY_ROW ? reinterpret_cast<const T*>(tile + (size_t)lane * stride)[e] : flat[e * 32 + lane], sign),
                   e);
    }
    end = list;
  };
  const float q0 = first > -INFINITY ? first : 0.f;
  const float2 a2 = both(fminf(a * kLog2E, 3.402823466e38f)), off = both(-q0);
  float2 s2 = both(0.f);
  for (int g = g0; g < g1; ++g) {
    float2 q[G / 2];
    group(g, q);
#pragma unroll
    for (int e = 0; e < G; ++e) {
      *end = (unsigned short)(g * G + e);      // kept if the next one does not overwrite it
      if ((e & 1 ? q[e / 2].y : q[e / 2].x) >= bound) end += list_stride;
    }
    if (end > list + (kRouteList - G - 1) * list_stride) put();
    if (over_all) {
      if (q0 == kHuge)      // perhaps an infinite score, which counts as this
#pragma unroll
        for (int e = 0; e < G / 2; ++e) q[e] = make_float2(fminf(fmaxf(q[e].x, -INFINITY), kHuge), fminf(fmaxf(q[e].y, -INFINITY), kHuge));
#pragma unroll
      for (int e = 0; e < G / 2; ++e) {
        const float2 x = mul2(a2, add2(q[e], off));
        s2 = add2(s2, make_float2(exp2_fast(fmaxf(x.x, -INFINITY)), exp2_fast(fmaxf(x.y, -INFINITY))));
      }
    }
  }
  put();
  if (split > 1) {       // the tile's first warp joins the others' lists
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) shared[(warp * N + j) * 32 + lane] = make_float2(v[j], __int_as_float(id[j]));
    __syncthreads();
    if (part == 0)
      for (int w = warp + 1; w < warp + split; ++w)
        for (int j = 0; j < N; ++j) {
          const float2 o = shared[(w * N + j) * 32 + lane];
          if (!(o.x > -INFINITY)) break;
          route_insert(v, id, o.x, __float_as_int(o.y));
        }
  }
  float sum = 0.f;
  if (over_all) {
    sum = s2.x + s2.y;
    if (split > 1) {
      __syncthreads();
      reinterpret_cast<float*>(shared)[warp * 32 + lane] = sum;
      __syncthreads();
      if (part == 0)
        for (int w = warp + 1; w < warp + split; ++w) sum += reinterpret_cast<float*>(shared)[w * 32 + lane];
    }
  }
  if (part != 0 || lane >= here) return;
  const long long t = row0 + lane;
  route_store<N>(t, n, v, id, q0, sum, over_all, a, sign, ids, weights, best, total);
}

// ---- the gradient ----------------------------------------------------------------------------------------------------------------------
// Every score's own part first (zero over the taken alone), then the taken ones' over it.

// An infinite score as the largest number of its sign; NaN stays.
__device__ __forceinline__ float route_finite(float s) {
  return s > 3.402823466e38f ? 3.402823466e38f : s < -3.402823466e38f ? -3.402823466e38f : s;
}

// One warp per row, 16-byte pieces.  65,536 x 256 float32 over all: 26.4 us, 0.80 of the copy rate, 69 % of the issue slots busy.
// CTAs a processor, as many as spill next to nothing: with six where eight fit that case takes 4 us more, 32,768 x 1001 float32 (unaligned) take 84 us
// with four and 70 with six.
template <typename T, bool ALIGNED> constexpr int route_grad_ctas() { return ALIGNED ? 8 : sizeof(T) == 4 ? 6 : 5; }
template <typename T, bool ALIGNED, bool OVER_ALL>
__global__ void __launch_bounds__(kRouteWarps * 32, route_grad_ctas<T, ALIGNED>())
route_grad_warp_kernel(const float* dweights, const T* s, long long rs, Span<T> in, int rows, int k, int n, float scale,
                       const int* ids, const float* weights, const float* best, const float* total, T* ds, long long drs) {
  constexpr int V = Piece<T>::V, H = V / 2;
  const int lane = threadIdx.x & 31, t = blockIdx.x * kRouteWarps + threadIdx.x / 32;
  if (t >= rows) return;
  int id = -1;
  float w = 0.f, g = 0.f, b = 0.f, sum = 0.f;
  if (lane < n) {
    id = ids[(long long)t * n + lane];
    w = weights[(long long)t * n + lane];
    g = dweights[(long long)t * n + lane];
  }
  if (OVER_ALL) {
    b = best[t];
    sum = total[t];
  }
  const bool taken = id >= 0 && id < k;
  const float c = warp_sum_f(taken ? w * g : 0.f);
  float f = OVER_ALL && sum > 0.f ? -scale * c / sum : 0.f;
  const bool far = !(fabsf(f) <= 3.402823466e38f);
  // perhaps an infinitely good score, which counts as this; an infinitely bad one then lies so far off that its difference is infinite again
  // (where the best score is the lowest number, closed clusters have to stay infinite)
  const bool huge = b == copysignf(3.402823466e38f, scale);
  const T* sr = s + (long long)t * rs;
  T* dr = ds + (long long)t * drs;
  const int pieces = ((k + V - 1) / V + 31) / 32 * 32;
#pragma unroll 2
  for (int i = lane; i < pieces; i += 32) {
    Piece<T> p;
    if (OVER_ALL) {
      p = load_piece<T, ALIGNED>(sr, i, k, in);
      float2 o[H];
      unpack(p, o);
      if (huge)
#pragma unroll
        for (int e = 0; e < H; ++e) o[e] = make_float2(route_finite(o[e].x), route_finite(o[e].y));
      // |scale| (q - q_best) = scale (s - best); NaN and what cannot be taken give 0
#pragma unroll
      for (int e = 0; e < H; ++e) {
        const float2 x = mul2(both(scale), add2(o[e], both(-b)));
        o[e] = mul2(both(f), make_float2(expf(fmaxf(x.x, -INFINITY)), expf(fmaxf(x.y, -INFINITY))));
      }
      p = pack<T>(o);
    } else {
      p.q = make_uint4(0u, 0u, 0u, 0u);
    }
    store_piece<T, ALIGNED>(dr, i, k, p);
  }
  __syncwarp();
  if (far) {      // the scale is applied last, so that 0 times it stays 0
    f = -c / sum;
    for (int e = lane; e < k; e += 32) {
      const float o = to_f(sr[e]), x = scale * ((huge ? route_finite(o) : o) - b);
      dr[e] = from_f<T>(scale * (f * expf(fmaxf(x, -INFINITY))));
    }
    __syncwarp();
  }
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
  const float sum = over_all ? total[t] : 0.f, q0 = over_all ? sign * best[t] : 0.f;
  float f = sum > 0.f ? -scale * c / sum : 0.f, last = 1.f;
  if (!(fabsf(f) <= 3.402823466e38f)) {      // the scale is then applied last: 0 times it stays 0
    f = -c / sum;
    last = scale;
  }
  const T* sr = s + t * rs;
  T* dr = ds + t * drs;
#pragma unroll 8
  for (int e = c0; e < c1; ++e) {
    float v = 0.f;
    if (over_all) {
      const float q = route_value(sr[e * cs], sign);
      if (q > -INFINITY) v = last * (f * expf(a * (q - q0)));
    }
    dr[e * dcs] = from_f<T>(v);
  }
  for (int j = 0; j < n; ++j) {
    const int id = ids[(long long)t * n + j];
    if (id >= c0 && id < c1) dr[id * dcs] = from_f<T>(scale * weights[(long long)t * n + j] * (dweights[(long long)t * n + j] - c));
  }
}

// ---- launches --------------------------------------------------------------------------------------------------------------------------

// f(N): the lists' length, n rounded up.  (Longer lists than 8 take more registers and code than a lane per row is worth.)
constexpr int kRouteLaneMax = 8;
template <typename F>
int with_list(int n, F&& f) {
  using std::integral_constant;
  if (n == 1) return f(integral_constant<int, 1>());
  if (n == 2) return f(integral_constant<int, 2>());
  if (n <= 4) return f(integral_constant<int, 4>());
  return f(integral_constant<int, 8>());
}
// Scores whose maximum stands for them in the first walk: so many that four times N groups remain, and the bound lets few others pass.
inline int route_share(int k, int n) {
  int share = kRouteGroup;
  while (share > 1 && k / share < 4 * n) share /= 2;
  return share;
}
// Warps that share 32 rows: as many as it takes to fill the device (16 a processor), each with `least` scores of a row or more, and lists
// that fit 32 KB together.
inline int route_split(long long tiles, int k, int n, int least, int sms) {
  int split = 1;
  while (split < 16 && split * n < 128 && tiles * split < (long long)sms * 16 && k / split >= 2 * least) split *= 2;
  return split;
}

template <typename T>
int route_launch(const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all, int* ids, float* weights,
                 float* best, float* total, int sms, cudaStream_t stream) {
  const long long tiles = ((long long)rows + 31) / 32;
  // 32 rows in shared memory, where they lie in whole words and fit
  const bool by_row = cs == 1 && rows_aligned(s, rs, rows, k, sizeof(T));
  // (the best one of scores that lie cluster after cluster needs one walk, which is as fast from memory: 65,536 x 512 float32 33 us, 48 by tiles)
  const bool by_col = !by_row && n > 1 && rs == 1 && aligned(s, 16) && (cs * sizeof(T)) % 16 == 0;
  const size_t bytes = RouteTile<T>::bytes(k, by_row);
  if (n <= kRouteLaneMax && (by_row || by_col) && bytes <= (by_row ? kRouteRowTileBytes : kRouteTileBytes)) {
    // more warps for a tile than its rows fill, so that the tiles a processor holds keep it busy (what the warps tell each other costs more
    // for longer lists)
    int split = route_split(tiles, k, n, 32, sms);
    while (split < 8 && split * n < 128 && bytes / split > (size_t)((n <= 4 ? 8 : 16) << 10)) split *= 2;
    int per_cta = 1;
    while (per_cta * split < 4 && bytes * per_cta * 2 <= kRouteTileBytes / 2 && tiles >= (long long)sms * 2 * per_cta) per_cta *= 2;
    const int warps = per_cta * split;
    return with_list(n, [&](auto count) -> int {
      constexpr int N = count();
      const size_t smem = bytes * per_cta + (size_t)32 * warps * std::max<size_t>(kRouteList * 2, split > 1 ? N * 8 : 0);
      const auto fn = by_row ? route_tile_kernel<T, N, true> : route_tile_kernel<T, N, false>;
      KM_CUDA(allow_smem(fn, smem));
      fn<<<(unsigned)((tiles + per_cta - 1) / per_cta), dim3(32, warps), smem, stream>>>(s, rs, cs, rows, k, n, scale, over_all, split,
                                                                                       route_share(k, N), (int)bytes, ids, weights,
                                                                                       best, total);
      KM_CUDA(cudaGetLastError());
      return KM_OK;
    });
  }
  // a lane per row where lanes' loads lie side by side, or a row is no longer than the line that its lane's loads share
  if (n <= kRouteLaneMax && (cs != 1 || (size_t)k * sizeof(T) <= 128 || (rs == 1 && rows > 1))) {
    const int split = route_split(tiles, k, n, 64, sms), warps = std::max(4, split), per_cta = warps / split;
    return with_list(n, [&](auto count) -> int {
      constexpr int N = count();
      const size_t smem = sizeof(float2) * 32 * warps * std::max(N == 1 ? 1 : kRouteList, split > 1 ? N : 1);
      const auto fn = route_lane_kernel<T, N>;
      KM_CUDA(allow_smem(fn, smem));
      fn<<<(unsigned)((tiles + per_cta - 1) / per_cta), dim3(32, warps), smem, stream>>>(s, rs, cs, rows, k, n, scale, over_all, split,
                                                                                       route_share(k, N), ids, weights, best, total);
      KM_CUDA(cudaGetLastError());
      return KM_OK;
    });
  }
  const int pieces = (k + Piece<T>::V - 1) / Piece<T>::V;
  const auto pick = [&](auto lie) {
    constexpr RouteRows L = lie();
    return pieces <= 32 ? route_warp_kernel<T, 1, L> : pieces <= 64 ? route_warp_kernel<T, 2, L>
         : pieces <= 128 ? route_warp_kernel<T, 4, L> : route_warp_kernel<T, 0, L>;
  };
  using std::integral_constant;
  auto fn = route_warp_kernel<T, 0, kStrided>;
  if (cs == 1) fn = rows_aligned(s, rs, rows, k, sizeof(T)) ? pick(integral_constant<RouteRows, kAligned>())
                                                            : pick(integral_constant<RouteRows, kUnaligned>());
  fn<<<(rows + kRouteWarps - 1) / kRouteWarps, kRouteWarps * 32, 0, stream>>>(
      s, rs, cs, cs == 1 ? span_of<T>(s, rs, rows, k) : Span<T>{nullptr, nullptr}, rows, k, n, scale, over_all, ids, weights, best,
      total);
  KM_CUDA(cudaGetLastError());
  return KM_OK;
}

template <typename T>
int route_grad_launch(const float* dweights, const T* s, long long rs, long long cs, int rows, int k, int n, float scale, bool over_all,
                      const int* ids, const float* weights, const float* best, const float* total, T* ds, long long drs, long long dcs,
                      int sms, cudaStream_t stream) {
  if (dcs == 1 && (!over_all || cs == 1)) {
    const bool al = rows_aligned(ds, drs, rows, k, sizeof(T)) && (!over_all || rows_aligned(s, rs, rows, k, sizeof(T)));
    const auto fn = over_all ? (al ? route_grad_warp_kernel<T, true, true> : route_grad_warp_kernel<T, false, true>)
                             : (al ? route_grad_warp_kernel<T, true, false> : route_grad_warp_kernel<T, false, false>);
    fn<<<(rows + kRouteWarps - 1) / kRouteWarps, kRouteWarps * 32, 0, stream>>>(
        dweights, s, rs, over_all ? span_of<T>(s, rs, rows, k) : Span<T>{nullptr, nullptr}, rows, k, n, scale, ids, weights, best,
        total, ds, drs);
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

// Layer norm of rows and its gradient.
//   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean g - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
// Both are bound by memory: a row is read once, kept in registers while its sums are formed, and written once.
#pragma once

#include "km_rows_vec.cuh"

namespace km {
namespace rows {

constexpr int kNormThreads = 256;   // of the kernels for wide rows

// Weights or biases of the columns of piece i (2 H of them), `none` behind the row's end.  They stay in L1 from row to row.  WHOLE: they
// start on a 16-byte boundary and the row is whole pieces; else `words` says whether they start on one.
template <typename P, int H, bool WHOLE>
__device__ __forceinline__ void load_params(const P* w, int i, int d, bool inside, bool words, float none, float2 (&f)[H]) {
  constexpr int V = 2 * H;
  const int c = i * V;
#pragma unroll
  for (int e = 0; e < H; ++e) f[e] = both(none);
  if (!inside) return;
  if (WHOLE || (words && c + V <= d)) {
    constexpr int PV = Piece<P>::V;
#pragma unroll
    for (int h = 0; h < V / PV; ++h) {
      Piece<P> p;
      p.q = __ldg(reinterpret_cast<const uint4*>(w + c + h * PV));
      float2 g[PV / 2];
      unpack(p, g);
#pragma unroll
      for (int e = 0; e < PV / 2; ++e) f[h * (PV / 2) + e] = g[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < H; ++e)
      f[e] = make_float2(c + 2 * e < d ? to_f(w[c + 2 * e]) : none, c + 2 * e + 1 < d ? to_f(w[c + 2 * e + 1]) : none);
  }
}

// Pieces of an aligned row that a lane holds: `have` of them lie in the row, the others are never loaded and stay zero (a load that
// fills in zeros, addresses that are formed for every piece and row cost more instructions than the sums).
template <typename T, int NV>
__device__ __forceinline__ void load_pieces(const T* row, int first, int have, Piece<T> (&p)[NV]) {
  const uint4* q = reinterpret_cast<const uint4*>(row) + first;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (i < have) p[i].q = q[i * 32];
}

// An unaligned row on its way through shared memory: the words that a warp's pieces lie across, 32 NV and one, and the pieces from them.
// Lanes read each other's words: the warp has to be in step after the copies and before the next ones.  A block's first and last row, whose
// words may reach beyond it, are loaded when they are taken.
template <int NV> constexpr int row_words() { return NV * 32 + 1; }
template <typename T, int NV>
__device__ __forceinline__ void copy_row(const T* row, int first, int d, const Span<T>& in, uint4* to) {
  constexpr int V = Piece<T>::V;
  if (!words_inside(row, d, in)) return;
  const int lane = threadIdx.x & 31, m = before_row(row), words = (m + d + V - 1) / V;
  const uint4* q = reinterpret_cast<const uint4*>(row - m) + first;
#pragma unroll
  for (int p = 0; p < NV; ++p)
    if (first + p * 32 < words) copy_async(to + p * 32 + lane, q + p * 32);
  if (lane == 0 && first + NV * 32 < words) copy_async(to + NV * 32, q + NV * 32);
}
template <typename T, int NV>
__device__ __forceinline__ void take_row(const T* row, int first, int d, const Span<T>& in, const uint4* at, Piece<T> (&p)[NV]) {
  constexpr int V = Piece<T>::V;
  if (words_inside(row, d, in)) {
    const int lane = threadIdx.x & 31, off = before_row(row) * (int)sizeof(T);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = (first + i * 32) * V;
      p[i].q = c < d ? shift_words(at[i * 32 + lane], at[i * 32 + lane + 1], off) : make_uint4(0u, 0u, 0u, 0u);
      if (c < d) clip_piece(p[i], c, d);
    }
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) p[i] = load_piece<T, false>(row, first + i * 32, d, in);
  }
}

// How a row is spread: `group` threads (whole warps) take it, NV pieces of 16 bytes each; `per_cta` groups share a CTA.  A group walks
// through the rows with the grid, so that a thread always has the same columns.
struct NormShape {
  int group = 0;   // 0: too wide, the kernel that reads a row from memory again
  int nv = 1;
  int per_cta = 1;
  int threads() const { return group * per_cta; }
};
// As few warps as can hold the row, 32 columns a lane at most: what a row costs besides its values - two sums over the lanes, the
// joining of the warps, addresses - is paid per warp.
inline NormShape norm_shape(int d, int size, int max_threads) {
  const int v = 16 / size, pieces = (d + v - 1) / v, most = 32 / v, warps = (pieces + 32 * most - 1) / (32 * most);
  NormShape s;
  s.nv = (pieces + 32 * warps - 1) / (32 * warps);
  if (32 * warps > max_threads) return s;
  s.group = 32 * warps;
  s.per_cta = std::max(1, 128 / s.group);
  return s;
}

// Barrier among the threads of one group: a CTA is group x per_cta threads.
__device__ __forceinline__ void group_sync() {
  asm volatile("bar.sync %0, %1;" ::"r"((int)threadIdx.y + 1), "r"((int)blockDim.x) : "memory");
}

// Mean and sum of squared differences from it.  Each warp takes them of its own columns first - its mean, then the differences - and the
// warps join by  M2 = sum of M2_w + n_w (mean_w - mean)^2:  no cancellation as in E x^2 - (E x)^2, and one barrier instead of two.
// 16,384 x 4096 bfloat16 take 45.6 us, 0.90 of the copy rate; 57 % of the issue slots are busy, so a leaner row is what would help.  Weights
// come from L1 for every row: held as float32 they cost 64 registers, and the warps lost cost more (53.8 us).
constexpr int kNormMaxThreads = 512;       // a row's group
constexpr int kNormAhead = 2;              // unaligned rows in shared memory
template <typename T, typename P, int NV, bool ALIGNED>
__global__ void __launch_bounds__(kNormMaxThreads)
norm_rows_kernel(const T* x, long long xs, Span<T> xin, int rows, int d, float inv_d, const P* w, const P* b, float eps, T* y, long long ys,
                 float* mean, float* rstd) {
  constexpr int V = Piece<T>::V, H = V / 2;
  __shared__ float2 red[2][16];      // used in turn: one half may still be read by slower warps
  const int in_group = threadIdx.x, lane = threadIdx.x & 31, warps = blockDim.x / 32;
  const bool w_words = (reinterpret_cast<uintptr_t>(w) & 15) == 0, b_words = (reinterpret_cast<uintptr_t>(b) & 15) == 0;
  // warp i of the group has the 32 NV pieces from i * 32 NV on, each lane every 32nd of them
  const auto columns = [&](int i) { return (float)max(0, min(32 * NV * V, d - i * 32 * NV * V)); };
  const int first = in_group / 32 * (32 * NV) + lane;
  const int have = min(NV, max(0, ((d + V - 1) / V - first + 31) / 32));
  const float n_own = columns(in_group / 32), n_lane = (lane & 15) < warps ? columns(lane & 15) : 0.f;
  const float inv_own = n_own > 0.f ? 1.f / n_own : 0.f, inv_lane = n_lane > 0.f ? 1.f / n_lane : 0.f;
  const int step = gridDim.x * blockDim.y;
  int t = blockIdx.x * blockDim.y + threadIdx.y, turn = 0;
  const auto norm = [&](const Piece<T>(&raw)[NV]) {
    float2 v[NV][H];
#pragma unroll
    for (int p = 0; p < NV; ++p) unpack(raw[p], v[p]);
    float2 s2 = both(0.f);
#pragma unroll
    for (int p = 0; p < NV; ++p)
#pragma unroll
      for (int e = 0; e < H; ++e) s2 = add2(s2, v[p][e]);
    const float s = warp_sum_f(s2.x + s2.y);
    float mu = s * inv_own;
    float2 q2 = both(0.f);
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      if (ALIGNED && p >= have) continue;
      const int c = (first + p * 32) * V;
#pragma unroll
      for (int e = 0; e < H; ++e) {
        float2 o = add2(v[p][e], both(-mu));
        if (!ALIGNED && c + V > d) {
          if (c + 2 * e >= d) o.x = 0.f;
          if (c + 2 * e + 1 >= d) o.y = 0.f;
        }
        q2 = fma2(o, o, q2);
      }
    }
    float q = warp_sum_f(q2.x + q2.y);
    if (warps > 1) {
      float2* mine = red[turn] + threadIdx.y * warps;
      if (lane == 0) mine[in_group / 32] = make_float2(s, q);
      group_sync();
      const float2 o = (lane & 15) < warps ? mine[lane & 15] : both(0.f);      // both halves of the warp alike
      mu = half_warp_sum(o.x) * inv_d;
      const float off = o.x * inv_lane - mu;
      q = half_warp_sum(fmaf(n_lane * off, off, o.y));
    }
    const float r = rsqrtf(fmaf(q, inv_d, eps));
    T* yr = y + (long long)t * ys;
    const auto finish = [&](auto with_w, auto with_b) {
      uint4* out = reinterpret_cast<uint4*>(yr) + first;
      Piece<T> done[NV];
#pragma unroll
      for (int p = 0; p < NV; ++p) {
        const int i = first + p * 32;
        float2 wf[H], bf[H];
        if (with_w()) load_params<P, H, ALIGNED>(w, i, d, p < have, w_words, 1.f, wf);
        if (with_b()) load_params<P, H, ALIGNED>(b, i, d, p < have, b_words, 0.f, bf);
#pragma unroll
        for (int e = 0; e < H; ++e) {
          float2 o = mul2(add2(v[p][e], both(-mu)), both(r));
          if (with_w() && with_b()) o = fma2(o, wf[e], bf[e]);
          else if (with_w()) o = mul2(o, wf[e]);
          else if (with_b()) o = add2(o, bf[e]);
          v[p][e] = o;
        }
        if (ALIGNED) {
          if (p < have) out[p * 32] = pack<T>(v[p]).q;
        } else {
          done[p] = pack<T>(v[p]);
        }
      }
      if (!ALIGNED) store_pieces(yr, first, d, done);
    };
    using std::integral_constant;
    if (w && b) finish(integral_constant<bool, true>(), integral_constant<bool, true>());
    else if (w) finish(integral_constant<bool, true>(), integral_constant<bool, false>());
    else if (b) finish(integral_constant<bool, false>(), integral_constant<bool, true>());
    else finish(integral_constant<bool, false>(), integral_constant<bool, false>());
    if (in_group == 0) {
      if (mean) mean[t] = mu;
      if (rstd) rstd[t] = r;
    }
    t += step;
    turn ^= 1;
  };
  if (ALIGNED) {
    // the next row is on its way into one buffer while the other one's sums are formed
    Piece<T> one[NV], two[NV];
#pragma unroll
    for (int p = 0; p < NV; ++p) one[p].q = two[p].q = make_uint4(0u, 0u, 0u, 0u);
    const auto load = [&](int row, Piece<T>(&p)[NV]) {
      if (row < rows) load_pieces(x + (long long)row * xs, first, have, p);
    };
    load(t, one);
    while (t < rows) {
      load(t + step, two);
      norm(one);
      if (t >= rows) break;
      load(t + step, one);
      norm(two);
    }
  } else {
    // (a piece can be shifted into place only when it has arrived: in registers the next row would be waited for)
    constexpr int S = kNormAhead;
    extern __shared__ uint4 ring[];      // [warp][S][row_words]
    uint4* slots = ring + (threadIdx.y * warps + in_group / 32) * (S * row_words<NV>());
    const auto copy = [&](int row, int slot) {
      if (row < rows) copy_row<T, NV>(x + (long long)row * xs, first, d, xin, slots + slot * row_words<NV>());
      copies_commit();
    };
    for (int i = 0; i < S; ++i) copy(t + i * step, i);
    int slot = 0;
    while (t < rows) {
      Piece<T> raw[NV];
      copies_wait<S - 1>();
      __syncwarp();
      take_row(x + (long long)t * xs, first, d, xin, slots + slot * row_words<NV>(), raw);
      __syncwarp();
      copy(t + S * step, slot);
      norm(raw);
      slot = slot + 1 == S ? 0 : slot + 1;
    }
    copies_wait<0>();
  }
}

// The gradient.  A group walks through the rows with the grid, so that a thread always has the same columns, and adds their dy xh
// and dy; the CTA joins its groups in their order and leaves its sums in part[CTA] (dw then db, d each), which
// norm_grad_sum_kernel adds up in the CTAs' order.
//
// Rows reach a lane through shared memory: it copies its own pieces there asynchronously, rows ahead of the one it works on, and reads
// them back itself, so nothing but its own copies has to be waited for.  In registers there is room for one row ahead beside 64 column
// sums, and 8 warps with one row each on its way are too few bytes for the memory's latency (59 us where this takes
// 48, 30,001 x 784 float32).
constexpr int kNormGradMaxThreads = 256;   // a row's group
constexpr int kNormGradRegs = 168;         // so that 12 warps fit a processor
template <int NV> constexpr int norm_grad_ahead() { return NV <= 4 ? 3 : 2; }      // rows in shared memory: 16 KB a warp at most
template <typename T, typename P, int NV, bool ALIGNED>
__global__ void __maxnreg__(kNormGradRegs)
norm_grad_rows_kernel(const T* dy, long long dys, Span<T> gin, const T* x, long long xs, Span<T> xin, const float* mean, const float* rstd, int rows, int d,
                      float inv_d, const P* w, T* dx, long long dxs, float* part) {
  constexpr int V = Piece<T>::V, H = V / 2, S = norm_grad_ahead<NV>();
  __shared__ float2 red[2][8];      // used in turn: one half may still be read by slower warps
  constexpr int WORDS = ALIGNED ? NV * 32 : row_words<NV>();      // of a warp's share of a row
  extern __shared__ uint4 ring[];   // [warp][S][x, dy][WORDS]; in the end the CTA's sums
  const int group = blockDim.x, per_cta = blockDim.y, which = threadIdx.y, in_group = threadIdx.x, lane = threadIdx.x & 31;
  const int warps = group / 32;
  const bool w_words = (reinterpret_cast<uintptr_t>(w) & 15) == 0;
  const int first = in_group / 32 * (32 * NV) + lane;      // as in norm_rows_kernel
  const int have = min(NV, max(0, ((d + V - 1) / V - first + 31) / 32));
  float2 aw[NV][H], ab[NV][H];
#pragma unroll
  for (int p = 0; p < NV; ++p)
#pragma unroll
    for (int e = 0; e < H; ++e) aw[p][e] = ab[p][e] = both(0.f);
  const int step = gridDim.x * per_cta;
  int t = blockIdx.x * per_cta + which, turn = 0;
  struct Row {
    Piece<T> x[NV], g[NV];
    float mu, r;
  };
  uint4* slots = ring + (which * warps + in_group / 32) * (S * 2 * WORDS);
  const auto copy_block = [&](const T* from, const Span<T>& in, uint4* to) {
    if (ALIGNED) {
      const uint4* q = reinterpret_cast<const uint4*>(from) + first;
#pragma unroll
      for (int p = 0; p < NV; ++p)
        if (p < have) copy_async(to + p * 32 + lane, q + p * 32);
    } else {
      copy_row<T, NV>(from, first, d, in, to);
    }
  };
  const auto copy = [&](int row, int slot) {      // starts the copies of a row
    if (row < rows) {
      uint4* to = slots + slot * (2 * WORDS);
      copy_block(x + (long long)row * xs, xin, to);
      copy_block(dy + (long long)row * dys, gin, to + WORDS);
    }
    copies_commit();
  };
  const auto take = [&](const T* from, const uint4* at, const Span<T>& in, Piece<T>(&p)[NV]) {
    if (ALIGNED) {
#pragma unroll
      for (int i = 0; i < NV; ++i) p[i].q = at[i * 32 + lane];
    } else {
      take_row(from, first, d, in, at, p);
    }
  };
  const auto grad = [&](const Row& row, int slot) {
    const float r = row.r;
    const float2 rr = both(r), off = both(-row.mu);      // (x - mu is exact or nearly so for rows far from zero, x r - mu r would not be)
    float2 xh[NV][H], g[NV][H];
#pragma unroll
    for (int p = 0; p < NV; ++p) {
      unpack(row.x[p], xh[p]);
      unpack(row.g[p], g[p]);
    }
    float2 a2 = both(0.f), b2 = both(0.f);
    const auto sums = [&](auto with_w) {
#pragma unroll
      for (int p = 0; p < NV; ++p) {
        float2 wf[H];
        if (with_w()) load_params<P, H, ALIGNED>(w, first + p * 32, d, p < have, w_words, 1.f, wf);
#pragma unroll
        for (int e = 0; e < H; ++e) {
          xh[p][e] = mul2(add2(xh[p][e], off), rr);     // behind the row's end g is zero
          aw[p][e] = fma2(g[p][e], xh[p][e], aw[p][e]);
          ab[p][e] = add2(ab[p][e], g[p][e]);
          if (with_w()) g[p][e] = mul2(g[p][e], wf[e]);
          a2 = add2(a2, g[p][e]);
          b2 = fma2(g[p][e], xh[p][e], b2);
        }
      }
    };
    if (w) sums(std::integral_constant<bool, true>());
    else sums(std::integral_constant<bool, false>());
    if (!ALIGNED) __syncwarp();        // lanes read each other's words
    copy(t + S * step, slot);          // the row's values have been used: its place is free
    float s1 = warp_sum_f(a2.x + a2.y), s2 = warp_sum_f(b2.x + b2.y);
    if (warps > 1) {
      float2* mine = red[turn] + which * warps;
      if (lane == 0) mine[in_group / 32] = make_float2(s1, s2);
      group_sync();
      const float2 o = (lane & 15) < warps ? mine[lane & 15] : both(0.f);
      s1 = half_warp_sum(o.x);
      s2 = half_warp_sum(o.y);
    }
    const float2 m1 = both(-r * (s1 * inv_d)), m2 = both(-r * (s2 * inv_d));
    T* dr = dx + (long long)t * dxs;
    uint4* out = reinterpret_cast<uint4*>(dr) + first;
    Piece<T> done[NV];
#pragma unroll
    for (int p = 0; p < NV; ++p) {
#pragma unroll
      for (int e = 0; e < H; ++e) g[p][e] = fma2(xh[p][e], m2, fma2(g[p][e], rr, m1));
      if (ALIGNED) {
        if (p < have) out[p * 32] = pack<T>(g[p]).q;
      } else {
        done[p] = pack<T>(g[p]);
      }
    }
    if (!ALIGNED) store_pieces(dr, first, d, done);
    t += step;
    turn ^= 1;
  };
  float nmu = 0.f, nr = 0.f;
  const auto statistics = [&](int row) {
    if (row < rows) {
      nmu = mean[row];
      nr = rstd[row];
    }
  };
  statistics(t);
  if (ALIGNED)
    for (int i = 0; i < S * 2; ++i)
      for (int p = have; p < NV; ++p) slots[i * WORDS + p * 32 + lane] = make_uint4(0u, 0u, 0u, 0u);     // pieces behind the row stay zero
  for (int i = 0; i < S; ++i) copy(t + i * step, i);
  int slot = 0;
  while (t < rows) {
    Row row;
    row.mu = nmu;
    row.r = nr;
    copies_wait<S - 1>();
    if (!ALIGNED) __syncwarp();
    take(x + (long long)t * xs, slots + slot * (2 * WORDS), xin, row.x);
    take(dy + (long long)t * dys, slots + slot * (2 * WORDS) + WORDS, gin, row.g);
    statistics(t + step);
    grad(row, slot);
    slot = slot + 1 == S ? 0 : slot + 1;
  }
  copies_wait<0>();
  if (!part) return;
  float* joined = reinterpret_cast<float*>(ring);     // dw then db of the CTA, d each
  float* pw = part + (size_t)blockIdx.x * 2 * d;
  float* cols = per_cta > 1 ? joined : pw;
  for (int grp = 0; grp < per_cta; ++grp) {
    __syncthreads();
    if (which == grp)
#pragma unroll
      for (int p = 0; p < NV; ++p)
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const int c = (first + p * 32) * V + e;
          if (c < d) {
            const float sw = e & 1 ? aw[p][e / 2].y : aw[p][e / 2].x, sb = e & 1 ? ab[p][e / 2].y : ab[p][e / 2].x;
            cols[c] = grp ? cols[c] + sw : sw;
            cols[d + c] = grp ? cols[d + c] + sb : sb;
          }
        }
  }
  __syncthreads();
  if (per_cta > 1)
    for (int c = which * group + in_group; c < 2 * d; c += group * per_cta) pw[c] = cols[c];
}

// Shared memory of that kernel: the rows on their way.  (The sums of the groups that share a CTA, 2 d floats, take less.)
template <typename T, int NV, bool ALIGNED>
constexpr size_t norm_grad_smem(int threads) {
  return (size_t)threads / 32 * (norm_grad_ahead<NV>() * 2 * (ALIGNED ? NV * 32 : row_words<NV>()) * sizeof(uint4));
}

// Rows wider than the registers take: one CTA per row, the row read again (from L2) for each of its sums.
template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
norm_wide_kernel(const T* x, long long xs, int d, const P* w, const P* b, float eps, T* y, long long ys, float* mean, float* rstd) {
  __shared__ float red[32];
  const T* xr = x + (long long)blockIdx.x * xs;
  T* yr = y + (long long)blockIdx.x * ys;
  float s = 0.f;
  for (int c = threadIdx.x; c < d; c += kNormThreads) s += to_f(xr[c]);
  const float mu = cta_sum(s, red) / (float)d;
  float q = 0.f;
  for (int c = threadIdx.x; c < d; c += kNormThreads) {
    const float v = to_f(xr[c]) - mu;
    q = fmaf(v, v, q);
  }
  const float r = 1.f / sqrtf(cta_sum(q, red) / (float)d + eps);
  for (int c = threadIdx.x; c < d; c += kNormThreads) {
    float v = (to_f(xr[c]) - mu) * r;
    if (w) v *= to_f(w[c]);
    if (b) v += to_f(b[c]);
    yr[c] = from_f<T>(v);
  }
  if (threadIdx.x == 0) {
    if (mean) mean[blockIdx.x] = mu;
    if (rstd) rstd[blockIdx.x] = r;
  }
}

template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
norm_grad_wide_kernel(const T* dy, long long dys, const T* x, long long xs, const float* mean, const float* rstd, int rows, int d,
                      const P* w, T* dx, long long dxs, float* part) {
  __shared__ float red[32];
  float* pw = part ? part + (size_t)blockIdx.x * 2 * d : nullptr;
  if (pw)
    for (int c = threadIdx.x; c < d; c += kNormThreads) pw[c] = pw[d + c] = 0.f;
  for (int t = blockIdx.x; t < rows; t += gridDim.x) {
    const T* xr = x + (long long)t * xs;
    const T* gr = dy + (long long)t * dys;
    T* dr = dx + (long long)t * dxs;
    const float mu = mean[t], r = rstd[t];
    float s1 = 0.f, s2 = 0.f;
    for (int c = threadIdx.x; c < d; c += kNormThreads) {
      const float v = to_f(gr[c]), xh = (to_f(xr[c]) - mu) * r;
      const float g = w ? v * to_f(w[c]) : v;
      s1 += g;
      s2 = fmaf(g, xh, s2);
      if (pw) {   // the same thread owns a column in every row
        pw[c] += v * xh;
        pw[d + c] += v;
      }
    }
    s1 = cta_sum(s1, red) / (float)d;
    s2 = cta_sum(s2, red) / (float)d;
    for (int c = threadIdx.x; c < d; c += kNormThreads) {
      const float v = to_f(gr[c]), xh = (to_f(xr[c]) - mu) * r;
      const float g = w ? v * to_f(w[c]) : v;
      dr[c] = from_f<T>(r * (g - s1 - xh * s2));
    }
  }
}

// dw, db = the parts' sums: a warp-wide strip of columns per CTA, 32 runs of consecutive parts, joined in their order.
__global__ void __launch_bounds__(1024)
norm_grad_sum_kernel(const float* part, int parts, int d, float* dw, float* db) {
  __shared__ float run[32][33];
  const int lane = threadIdx.x, c = blockIdx.x * 32 + lane, per = (parts + 31) / 32;
  float s = 0.f;
  wait_for_previous();
  if (c < 2 * d)
    for (int p = threadIdx.y * per; p < min(parts, (int)(threadIdx.y + 1) * per); ++p) s += part[(size_t)p * 2 * d + c];
  run[threadIdx.y][lane] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < 2 * d) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += run[i][lane];
    if (c < d) dw[c] = s;
    else db[c - d] = s;
  }
}

// CTAs of a walk: as many as run at once (per processor, from the kernel's registers).  Of the gradient's, each leaves a partial sum; their
// number must not depend on more than the sizes and the element size, which is all that the workspace is asked for.
constexpr int kNormGradThreadsPerSm = 384;
inline NormShape norm_grad_shape(int d, int size) { return norm_shape(d, size, kNormGradMaxThreads); }
inline int norm_grid(size_t rows, const NormShape& s, int sms, int threads_per_sm) {
  if (!s.group) return (int)std::min<size_t>(rows, (size_t)sms * 4);
  return (int)std::min<size_t>((rows + s.per_cta - 1) / s.per_cta, (size_t)sms * std::max(1, threads_per_sm / s.threads()));
}

// f(NV) with the number of pieces as a constant.
template <typename T, typename F>
int with_pieces(int nv, F&& f) {
  using std::integral_constant;
  switch (nv) {
    case 1: return f(integral_constant<int, 1>());
    case 2: return f(integral_constant<int, 2>());
    case 3: return f(integral_constant<int, 3>());
    case 4: return f(integral_constant<int, 4>());
  }
  if constexpr (sizeof(T) == 4) switch (nv) {
    case 5: return f(integral_constant<int, 5>());
    case 6: return f(integral_constant<int, 6>());
    case 7: return f(integral_constant<int, 7>());
    case 8: return f(integral_constant<int, 8>());
  }
  return KM_EINVAL;
}

template <typename T, typename P, bool ALIGNED>
int norm_launch(const NormShape& s, int sms, const T* x, long long xs, int rows, int d, const P* w, const P* b, float eps, T* y,
                long long ys, float* mean, float* rstd, cudaStream_t stream) {
  return with_pieces<T>(s.nv, [&](auto nv) -> int {
    static ResidentCtas resident;
    const auto fn = norm_rows_kernel<T, P, nv(), ALIGNED>;
    int per_sm = 0;
    const size_t smem = ALIGNED ? 0 : (size_t)s.threads() / 32 * (kNormAhead * row_words<nv()>() * sizeof(uint4));
    KM_CUDA(allow_smem(fn, smem));
    KM_TRY(resident.get(fn, s.threads(), smem, &per_sm));
    const int grid = norm_grid(rows, s, sms, per_sm * s.threads());
    fn<<<grid, dim3(s.group, s.per_cta), smem, stream>>>(x, xs, span_of<T>(x, xs, rows, d), rows, d, 1.f / (float)d, w, b, eps, y,
                                                                                        ys, mean, rstd);
    KM_CUDA(cudaGetLastError());
    return KM_OK;
  });
}

template <typename T, typename P, bool ALIGNED>
int norm_grad_launch(const NormShape& s, int grid, const T* dy, long long dys, const T* x, long long xs, const float* mean,
                     const float* rstd, int rows, int d, const P* w, T* dx, long long dxs, float* part, cudaStream_t stream) {
  return with_pieces<T>(s.nv, [&](auto nv) -> int {
    const auto fn = norm_grad_rows_kernel<T, P, nv(), ALIGNED>;
    const size_t smem = norm_grad_smem<T, nv(), ALIGNED>(s.threads());
    KM_CUDA(allow_smem(fn, smem));
    fn<<<grid, dim3(s.group, s.per_cta), smem, stream>>>(
        dy, dys, span_of<T>(dy, dys, rows, d), x, xs, span_of<T>(x, xs, rows, d), mean, rstd, rows, d, 1.f / (float)d, w, dx, dxs,
        part);
    KM_CUDA(cudaGetLastError());
    return KM_OK;
  });
}

}  // namespace rows
}  // namespace km

// Layer norm of rows and its gradient.
//   mu = mean x,  r = 1 / sqrt(mean (x - mu)^2 + eps),  xh = (x - mu) r,  y = xh w + b
//   g = dy w,  dx = r (g - mean g - xh mean(g xh)),  dw = sum over rows of dy xh,  db = sum over rows of dy
#pragma once

#include "km_rows.cuh"

namespace km {
namespace rows {

constexpr int kNormThreads = 256;

template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
norm_kernel(const T* x, long long xs, int d, const P* w, const P* b, float eps, T* y, long long ys, float* mean, float* rstd) {
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

// CTA p of `parts` takes rows p, p + parts, ... and leaves its column sums in part[p] (dw then db, d each).
template <typename T, typename P>
__global__ void __launch_bounds__(kNormThreads)
norm_grad_kernel(const T* dy, long long dys, const T* x, long long xs, const float* mean, const float* rstd, int rows, int d,
                 const P* w, T* dx, long long dxs, float* part) {
  __shared__ float red[32];
  float* pw = part ? part + (size_t)blockIdx.x * 2 * d : nullptr;
  if (pw)
    for (int c = threadIdx.x; c < 2 * d; c += kNormThreads) pw[c] = 0.f;
  __syncthreads();
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

// dw, db = the parts' sums, in the parts' order.
__global__ void norm_grad_sum_kernel(const float* part, int parts, int d, float* dw, float* db) {
  const int c = blockIdx.x * blockDim.x + threadIdx.x;
  if (c >= 2 * d) return;
  float s = 0.f;
  for (int p = 0; p < parts; ++p) s += part[(size_t)p * 2 * d + c];
  if (c < d) dw[c] = s;
  else db[c - d] = s;
}

inline int norm_grad_parts(size_t rows, int sms) { return (int)std::min<size_t>(rows, (size_t)sms * 2); }

}  // namespace rows
}  // namespace km

// C entry points of the row operators (section 5 of include/h2o4gpu_kmeans.h): layer norm, rows sorted by cluster and back (routing:
// kmeans_route.cu).  They work on device memory of the current device, enqueue on the caller's stream, never allocate and never wait.
#include "km_rows_move.cuh"
#include "km_rows_norm.cuh"
#include "km_rows_sort.cuh"

using namespace km;
using namespace km::rows;

namespace {

// Type of the norm's weight and bias: float32, or the rows' own.
#define KM_ROWS_PARAM(param_dtype, T, P, ...)                       \
  do {                                                              \
    if ((param_dtype) == KM_DTYPE_F32) { using P = float; __VA_ARGS__; } \
    else { using P = T; __VA_ARGS__; }                              \
  } while (0)

int check_params(const char* name, int dtype, size_t cols, const void* weight, const void* bias, int* param_dtype) {
  if (!weight && !bias) *param_dtype = KM_DTYPE_F32;
  if (*param_dtype != KM_DTYPE_F32 && *param_dtype != dtype)
    KM_FAIL(KM_EINVAL, std::string(name) + ": weight and bias are float32 or of the rows' type");
  const int size = elem_size(*param_dtype);
  if ((weight && !aligned(weight, size)) || (bias && !aligned(bias, size)))
    KM_FAIL(KM_EINVAL, std::string(name) + ": misaligned weight or bias");
  if (cols < 1) KM_FAIL(KM_EINVAL, std::string(name) + ": cols must be at least 1");
  if (cols > kMaxCols) KM_FAIL(KM_EINVAL, std::string(name) + ": too many columns");
  return KM_OK;
}

int layer_norm(int dtype, const void* x, long long xs, size_t rows, size_t cols, const void* weight, const void* bias,
               int param_dtype, double eps, void* y, long long ys, float* mean, float* rstd, cudaStream_t stream) {
  const int size = elem_size(dtype);
  if (!size) KM_FAIL(KM_EINVAL, "kmeans_layer_norm: rows are float32, float16 or bfloat16");
  if (!(eps >= 0.0) || !std::isfinite((float)eps)) KM_FAIL(KM_EINVAL, "kmeans_layer_norm: eps must be finite and not negative");
  KM_TRY(check_params("kmeans_layer_norm", dtype, cols, weight, bias, &param_dtype));
  if (rows == 0) return KM_OK;
  if (rows > kMaxRows || !block_ok(x, xs, rows, cols, size, false) || !block_ok(y, ys, rows, cols, size, true) ||
      !aligned(mean, 4) || !aligned(rstd, 4))
    KM_FAIL(KM_EINVAL, "kmeans_layer_norm: bad argument");
  const int d = (int)cols;
  int sms = 0;
  KM_TRY(sm_count(&sms));
  const NormShape shape = norm_shape(d, size, kNormMaxThreads);
  const bool al = rows_aligned(x, xs, rows, cols, size) && rows_aligned(y, ys, rows, cols, size) && aligned(weight, 16) &&
                  aligned(bias, 16);
  int rc = KM_OK;
  KM_ROWS_DTYPE(dtype, T, KM_ROWS_PARAM(param_dtype, T, P,
      const T* xp = static_cast<const T*>(x);
      const P* wp = static_cast<const P*>(weight);
      const P* bp = static_cast<const P*>(bias);
      T* yp = static_cast<T*>(y);
      if (!shape.group) {
        norm_wide_kernel<T, P><<<(unsigned)rows, kNormThreads, 0, stream>>>(xp, xs, d, wp, bp, (float)eps, yp, ys, mean, rstd);
        KM_CUDA(cudaGetLastError());
      } else if (al) {
        rc = norm_launch<T, P, true>(shape, sms, xp, xs, (int)rows, d, wp, bp, (float)eps, yp, ys, mean, rstd, stream);
      } else {
        rc = norm_launch<T, P, false>(shape, sms, xp, xs, (int)rows, d, wp, bp, (float)eps, yp, ys, mean, rstd, stream);
      }));
  return rc;
}

// Partial sums of the gradient's walk over rows of `size`-byte elements.
int norm_grad_parts(size_t rows, size_t cols, int size, int sms) {
  return norm_grid(rows, norm_grad_shape((int)cols, size), sms, kNormGradThreadsPerSm);
}

int layer_norm_grad_workspace(size_t rows, size_t cols, size_t* bytes) {
  if (!bytes || cols < 1 || cols > kMaxSumCols || rows > kMaxRows) KM_FAIL(KM_EINVAL, "kmeans_layer_norm_grad_workspace: bad argument");
  *bytes = 0;
  if (rows == 0) return KM_OK;
  int sms = 0;
  KM_TRY(sm_count(&sms));
  const int parts = std::max(norm_grad_parts(rows, cols, 2, sms), norm_grad_parts(rows, cols, 4, sms));
  *bytes = (size_t)parts * 2 * cols * sizeof(float);
  return KM_OK;
}

int layer_norm_grad(int dtype, const void* dy, long long dys, const void* x, long long xs, const float* mean, const float* rstd,
                    size_t rows, size_t cols, const void* weight, int param_dtype, void* dx, long long dxs, float* dweight,
                    float* dbias, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  const int size = elem_size(dtype);
  if (!size) KM_FAIL(KM_EINVAL, "kmeans_layer_norm_grad: rows are float32, float16 or bfloat16");
  KM_TRY(check_params("kmeans_layer_norm_grad", dtype, cols, weight, nullptr, &param_dtype));
  if ((dweight == nullptr) != (dbias == nullptr) || !aligned(dweight, 4) || !aligned(dbias, 4))
    KM_FAIL(KM_EINVAL, "kmeans_layer_norm_grad: dweight and dbias go together");
  if (rows > kMaxRows || cols > kMaxSumCols) KM_FAIL(KM_EINVAL, "kmeans_layer_norm_grad: too many rows or columns");
  if (rows == 0) {
    if (dweight) {
      KM_CUDA(cudaMemsetAsync(dweight, 0, cols * sizeof(float), stream));
      KM_CUDA(cudaMemsetAsync(dbias, 0, cols * sizeof(float), stream));
    }
    return KM_OK;
  }
  if (!block_ok(x, xs, rows, cols, size, false) || !block_ok(dy, dys, rows, cols, size, false) ||
      !block_ok(dx, dxs, rows, cols, size, true) || !mean || !rstd || !aligned(mean, 4) || !aligned(rstd, 4))
    KM_FAIL(KM_EINVAL, "kmeans_layer_norm_grad: bad argument");
  int sms = 0;
  KM_TRY(sm_count(&sms));
  const int parts = norm_grad_parts(rows, cols, size, sms), d = (int)cols;
  if (dweight && (!workspace || !aligned(workspace, 16) || workspace_bytes < (size_t)parts * 2 * cols * sizeof(float)))
    KM_FAIL(KM_EINVAL, "kmeans_layer_norm_grad: workspace missing or too small");
  float* part = dweight ? static_cast<float*>(workspace) : nullptr;
  const NormShape shape = norm_grad_shape(d, size);
  const bool al = rows_aligned(x, xs, rows, cols, size) && rows_aligned(dy, dys, rows, cols, size) &&
                  rows_aligned(dx, dxs, rows, cols, size) && aligned(weight, 16);
  int rc = KM_OK;
  KM_ROWS_DTYPE(dtype, T, KM_ROWS_PARAM(param_dtype, T, P,
      const T* gp = static_cast<const T*>(dy);
      const T* xp = static_cast<const T*>(x);
      const P* wp = static_cast<const P*>(weight);
      T* dp = static_cast<T*>(dx);
      if (!shape.group) {
        norm_grad_wide_kernel<T, P><<<parts, kNormThreads, 0, stream>>>(gp, dys, xp, xs, mean, rstd, (int)rows, d, wp, dp, dxs, part);
        KM_CUDA(cudaGetLastError());
      } else if (al) {
        rc = norm_grad_launch<T, P, true>(shape, parts, gp, dys, xp, xs, mean, rstd, (int)rows, d, wp, dp, dxs, part, stream);
      } else {
        rc = norm_grad_launch<T, P, false>(shape, parts, gp, dys, xp, xs, mean, rstd, (int)rows, d, wp, dp, dxs, part, stream);
      }));
  KM_TRY(rc);
  if (part) {
    KM_TRY(launch_early(norm_grad_sum_kernel, dim3((unsigned)((2 * cols + 31) / 32)), dim3(32, 32), 0, stream, part, parts, d, dweight,
                        dbias));
  }
  return KM_OK;
}

int check_sort(const char* name, size_t rows, int n, int k, int align, size_t* capacity) {
  if (n < 1 || k < 1 || align < 1) KM_FAIL(KM_EINVAL, std::string(name) + ": bad argument");
  if (k > kSortMaxK) KM_FAIL(KM_EINVAL, std::string(name) + ": at most " + std::to_string(kSortMaxK) + " clusters");
  if (rows > kMaxRows / (size_t)n) KM_FAIL(KM_EINVAL, std::string(name) + ": too many entries");
  const size_t entries = rows * (size_t)n;
  *capacity = entries + std::min<size_t>((size_t)k, entries) * (size_t)(align - 1);
  if (*capacity > kMaxRows) KM_FAIL(KM_EINVAL, std::string(name) + ": too many places");
  return KM_OK;
}

int sort_rows_sizes(size_t rows, int n, int k, int align, size_t* capacity, size_t* workspace_bytes) {
  if (!capacity || !workspace_bytes) KM_FAIL(KM_EINVAL, "kmeans_sort_rows_sizes: bad argument");
  KM_TRY(check_sort("kmeans_sort_rows_sizes", rows, n, k, align, capacity));
  *workspace_bytes = 0;
  if (rows == 0) return KM_OK;
  int sms = 0;
  KM_TRY(sm_count(&sms));
  const SortPlan plan = sort_plan((long long)rows * n, k, sms);
  if (plan.blocks > 1) *workspace_bytes = (size_t)plan.blocks * k * sizeof(int);
  return KM_OK;
}

int sort_rows(const int32_t* ids, long long stride, size_t rows, int n, int k, int align, int32_t* offsets, int32_t* counts,
              int32_t* slot, int32_t* source, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
  size_t capacity = 0;
  KM_TRY(check_sort("kmeans_sort_rows", rows, n, k, align, &capacity));
  if (!offsets || !counts || !aligned(offsets, 4) || !aligned(counts, 4)) KM_FAIL(KM_EINVAL, "kmeans_sort_rows: bad argument");
  if (rows == 0) {
    KM_CUDA(cudaMemsetAsync(offsets, 0, ((size_t)k + 1) * sizeof(int), stream));
    KM_CUDA(cudaMemsetAsync(counts, 0, (size_t)k * sizeof(int), stream));
    return KM_OK;
  }
  if (!block_ok(ids, stride, rows, (size_t)n, 4, false) || !slot || !source || !aligned(slot, 4) || !aligned(source, 4))
    KM_FAIL(KM_EINVAL, "kmeans_sort_rows: bad argument");
  int sms = 0;
  KM_TRY(sm_count(&sms));
  const int entries = (int)(rows * (size_t)n);
  const SortPlan plan = sort_plan(entries, k, sms);
  int* part = nullptr;
  if (plan.blocks > 1) {
    if (!workspace || !aligned(workspace, 4) || workspace_bytes < (size_t)plan.blocks * k * sizeof(int))
      KM_FAIL(KM_EINVAL, "kmeans_sort_rows: workspace missing or too small");
    part = static_cast<int*>(workspace);
    const size_t smem = (size_t)k * sizeof(int);
    KM_CUDA(allow_smem(sort_count_kernel, smem));
    sort_count_kernel<<<plan.blocks, kSortThreads, smem, stream>>>(ids, stride, n, entries, k, plan.chunk, part);
    KM_CUDA(cudaGetLastError());
  }
  const size_t smem = (size_t)(plan.warps + 2) * k * sizeof(int);
  KM_CUDA(allow_smem(sort_place_kernel, smem));
  if (part)
    return launch_early(sort_place_kernel, dim3(plan.blocks), dim3(kSortThreads), smem, stream, ids, stride, n, entries, k, align, plan, part,
                        offsets, counts, slot, source, (int)capacity);
  sort_place_kernel<<<plan.blocks, kSortThreads, smem, stream>>>(ids, stride, n, entries, k, align, plan, part, offsets, counts, slot,
                                                                 source, (int)capacity);
  KM_CUDA(cudaGetLastError());
  return KM_OK;
}

int check_move(const char* name, int dtype, size_t rows, int n, size_t cols, size_t capacity) {
  if (!elem_size(dtype)) KM_FAIL(KM_EINVAL, std::string(name) + ": rows are float32, float16 or bfloat16");
  if (n < 1 || cols < 1 || cols > kMaxCols || capacity > kMaxRows || rows > kMaxRows / (size_t)n)
    KM_FAIL(KM_EINVAL, std::string(name) + ": bad argument");
  return KM_OK;
}
// CTAs that fill the places without an entry
unsigned pad_ctas(size_t capacity, int sms) {
  return (unsigned)std::min<size_t>((capacity + kMoveThreads - 1) / kMoveThreads, (size_t)sms * 4);
}

int dispatch(int dtype, const void* x, long long xs, size_t rows, size_t cols, int n, const int32_t* slot, const int32_t* source,
             size_t capacity, void* out, long long os, cudaStream_t stream) {
  KM_TRY(check_move("kmeans_dispatch", dtype, rows, n, cols, capacity));
  if (capacity == 0) return KM_OK;
  const int size = elem_size(dtype);
  if ((rows && (!block_ok(x, xs, rows, cols, size, false) || !slot || !aligned(slot, 4))) || !source || !aligned(source, 4) ||
      !block_ok(out, os, capacity, cols, size, true))
    KM_FAIL(KM_EINVAL, "kmeans_dispatch: bad argument");
  int sms = 0;
  KM_TRY(sm_count(&sms));
  const bool al = rows_aligned(x, xs, rows, cols, size) && rows_aligned(out, os, capacity, cols, size);
  const int words = move_words(cols, size, al);
  const long long blocks = move_blocks(rows, words), grid = blocks + pad_ctas(capacity, sms);
  if (grid > 0x7fffffffLL) KM_FAIL(KM_EINVAL, "kmeans_dispatch: too many rows for one launch");
  KM_ROWS_DTYPE(dtype, T,
      const auto fn = al ? dispatch_kernel<T, true> : dispatch_kernel<T, false>;
      fn<<<(unsigned)grid, kMoveThreads, 0, stream>>>(static_cast<const T*>(x), xs, span_of<T>(x, xs, rows, cols), (int)rows, (int)cols,
                                                      words, n, slot, source, (int)capacity, static_cast<T*>(out), os, blocks));
  KM_CUDA(cudaGetLastError());
  return KM_OK;
}

// How many entries of a row are on their way together: no more than there are.
#define KM_ROWS_AT_ONCE(n, U, ...)                                                         \
  do {                                                                                     \
    if ((n) == 1) { constexpr int U = 1; __VA_ARGS__; }                                    \
    else if ((n) == 2) { constexpr int U = 2; __VA_ARGS__; }                               \
    else if ((n) == 3) { constexpr int U = 3; __VA_ARGS__; }                               \
    else { constexpr int U = 4; __VA_ARGS__; }                                             \
  } while (0)

int combine(int dtype, const void* in, long long is, size_t capacity, size_t cols, const int32_t* slot, const float* weights,
            size_t rows, int n, void* y, long long ys, cudaStream_t stream) {
  KM_TRY(check_move("kmeans_combine", dtype, rows, n, cols, capacity));
  if (rows == 0) return KM_OK;
  const int size = elem_size(dtype);
  if ((capacity && !block_ok(in, is, capacity, cols, size, false)) || !slot || !aligned(slot, 4) || !aligned(weights, 4) ||
      !block_ok(y, ys, rows, cols, size, true))
    KM_FAIL(KM_EINVAL, "kmeans_combine: bad argument");
  const bool al = rows_aligned(in, is, capacity, cols, size) && rows_aligned(y, ys, rows, cols, size);
  const int words = move_words(cols, size, al);
  const long long grid = move_blocks(rows, words);
  if (grid > 0x7fffffffLL) KM_FAIL(KM_EINVAL, "kmeans_combine: too many rows for one launch");
  KM_ROWS_DTYPE(dtype, T, KM_ROWS_AT_ONCE(n, U,
      const auto fn = al ? combine_kernel<T, true, U> : combine_kernel<T, false, U>;
      fn<<<(unsigned)grid, kMoveThreads, 0, stream>>>(static_cast<const T*>(in), is, span_of<T>(in, is, capacity, cols), (int)capacity,
                                                      (int)cols, words, slot, weights, (int)rows, n, static_cast<T*>(y), ys)));
  KM_CUDA(cudaGetLastError());
  return KM_OK;
}

int combine_grad(int dtype, const void* dy, long long dys, const void* in, long long is, size_t capacity, size_t cols,
                 const int32_t* slot, const int32_t* source, const float* weights, size_t rows, int n, void* din, long long dis,
                 float* dweights, cudaStream_t stream) {
  KM_TRY(check_move("kmeans_combine_grad", dtype, rows, n, cols, capacity));
  if (rows == 0 && capacity == 0) return KM_OK;
  const int size = elem_size(dtype);
  if ((rows && (!block_ok(dy, dys, rows, cols, size, false) || !slot || !aligned(slot, 4) || !weights || !aligned(weights, 4) ||
                !dweights || !aligned(dweights, 4))) ||
      (capacity && (!block_ok(in, is, capacity, cols, size, false) || !block_ok(din, dis, capacity, cols, size, true) || !source ||
                    !aligned(source, 4))))
    KM_FAIL(KM_EINVAL, "kmeans_combine_grad: bad argument");
  int sms = 0;
  KM_TRY(sm_count(&sms));
  const bool al = rows_aligned(dy, dys, rows, cols, size) && rows_aligned(in, is, capacity, cols, size) &&
                  rows_aligned(din, dis, capacity, cols, size);
  const int words = move_words(cols, size, al), warps = combine_grad_warps(rows, words, sms), per_cta = kCombineGradThreads / 32 / warps;
  const int blocks = (int)((rows + per_cta - 1) / per_cta);
  KM_ROWS_DTYPE(dtype, T, KM_ROWS_AT_ONCE(n, U,
      const auto fn = al ? combine_grad_kernel<T, true, U> : combine_grad_kernel<T, false, U>;
      fn<<<(unsigned)blocks + pad_ctas(capacity, sms), dim3(32 * warps, per_cta), 0, stream>>>(
          static_cast<const T*>(dy), dys, span_of<T>(dy, dys, rows, cols), static_cast<const T*>(in), is,
          span_of<T>(in, is, capacity, cols), (int)capacity, (int)cols, words, slot, source, weights, (int)rows, n,
          static_cast<T*>(din), dis, dweights, blocks)));
  KM_CUDA(cudaGetLastError());
  return KM_OK;
}

}  // namespace

extern "C" {

int kmeans_layer_norm(int dtype, const void* x, long long x_stride, size_t rows, size_t cols, const void* weight, const void* bias,
                      int param_dtype, double eps, void* y, long long y_stride, float* mean, float* rstd, void* stream) {
  return guarded("kmeans_layer_norm", [&] {
    return layer_norm(dtype, x, x_stride, rows, cols, weight, bias, param_dtype, eps, y, y_stride, mean, rstd, as_stream(stream));
  });
}
int kmeans_layer_norm_grad_workspace(size_t rows, size_t cols, size_t* bytes) {
  return guarded("kmeans_layer_norm_grad_workspace", [&] { return layer_norm_grad_workspace(rows, cols, bytes); });
}
int kmeans_layer_norm_grad(int dtype, const void* dy, long long dy_stride, const void* x, long long x_stride, const float* mean,
                           const float* rstd, size_t rows, size_t cols, const void* weight, int param_dtype, void* dx,
                           long long dx_stride, float* dweight, float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded("kmeans_layer_norm_grad", [&] {
    return layer_norm_grad(dtype, dy, dy_stride, x, x_stride, mean, rstd, rows, cols, weight, param_dtype, dx, dx_stride, dweight,
                           dbias, workspace, workspace_bytes, as_stream(stream));
  });
}
int kmeans_sort_rows_sizes(size_t rows, int n, int k, int align, size_t* capacity, size_t* workspace_bytes) {
  return guarded("kmeans_sort_rows_sizes", [&] { return sort_rows_sizes(rows, n, k, align, capacity, workspace_bytes); });
}
int kmeans_sort_rows(const int32_t* ids, long long ids_stride, size_t rows, int n, int k, int align, int32_t* offsets, int32_t* counts,
                     int32_t* slot, int32_t* source, void* workspace, size_t workspace_bytes, void* stream) {
  return guarded("kmeans_sort_rows", [&] {
    return sort_rows(ids, ids_stride, rows, n, k, align, offsets, counts, slot, source, workspace, workspace_bytes, as_stream(stream));
  });
}
int kmeans_dispatch(int dtype, const void* x, long long x_stride, size_t rows, size_t cols, int n, const int32_t* slot,
                    const int32_t* source, size_t capacity, void* out, long long out_stride, void* stream) {
  return guarded("kmeans_dispatch", [&] {
    return dispatch(dtype, x, x_stride, rows, cols, n, slot, source, capacity, out, out_stride, as_stream(stream));
  });
}
int kmeans_combine(int dtype, const void* in, long long in_stride, size_t capacity, size_t cols, const int32_t* slot,
                   const float* weights, size_t rows, int n, void* y, long long y_stride, void* stream) {
  return guarded("kmeans_combine", [&] {
    return combine(dtype, in, in_stride, capacity, cols, slot, weights, rows, n, y, y_stride, as_stream(stream));
  });
}
int kmeans_combine_grad(int dtype, const void* dy, long long dy_stride, const void* in, long long in_stride, size_t capacity,
                        size_t cols, const int32_t* slot, const int32_t* source, const float* weights, size_t rows, int n, void* din,
                        long long din_stride, float* dweights, void* stream) {
  return guarded("kmeans_combine_grad", [&] {
    return combine_grad(dtype, dy, dy_stride, in, in_stride, capacity, cols, slot, source, weights, rows, n, din, din_stride, dweights,
                        as_stream(stream));
  });
}

}  // extern "C"

// C entry points of routing (section 5 of include/h2o4gpu_kmeans.h): the n best clusters of a row, their weights, and the gradient.
#include "km_rows_route.cuh"

using namespace km;
using namespace km::rows;

namespace {

// Scores lie in any two strides; a value's place must fit 63 bits.
bool strides_ok(long long rs, long long cs) { return rs >= 0 && cs >= 0 && rs <= (1LL << 31) && cs <= (1LL << 31); }

int check_route(const char* name, int dtype, size_t rows, int k, int n, float scale) {
  if (!elem_size(dtype)) KM_FAIL(KM_EINVAL, std::string(name) + ": scores are float32, float16 or bfloat16");
  if (rows > kMaxRows || k < 1 || k > kRouteMaxK) KM_FAIL(KM_EINVAL, std::string(name) + ": bad argument");
  if (n < 1 || n > kRouteMax || n > k)
    KM_FAIL(KM_EINVAL, std::string(name) + ": a row takes 1 to " + std::to_string(kRouteMax) + " clusters, and no more than there are");
  if (!std::isfinite(scale) || scale == 0.f) KM_FAIL(KM_EINVAL, std::string(name) + ": scale must be finite and not zero");
  return KM_OK;
}

int route(int dtype, const void* scores, long long rs, long long cs, size_t rows, int k, int n, float scale, int over_all,
          int32_t* ids, float* weights, float* best, float* total, cudaStream_t stream) {
  KM_TRY(check_route("kmeans_route", dtype, rows, k, n, scale));
  if (rows == 0) return KM_OK;
  if (!scores || !aligned(scores, elem_size(dtype)) || !strides_ok(rs, cs) || !ids || !weights || !best || !total ||
      !aligned(ids, 4) || !aligned(weights, 4) || !aligned(best, 4) || !aligned(total, 4))
    KM_FAIL(KM_EINVAL, "kmeans_route: bad argument");
  int sms = 0, rc = KM_OK;
  KM_TRY(sm_count(&sms));
  KM_ROWS_DTYPE(dtype, T,
      rc = route_launch<T>(static_cast<const T*>(scores), rs, cs, (int)rows, k, n, scale, over_all != 0, ids, weights, best, total, sms,
                           stream));
  return rc;
}

int route_grad(int dtype, const float* dweights, const void* scores, long long rs, long long cs, size_t rows, int k, int n,
               float scale, int over_all, const int32_t* ids, const float* weights, const float* best, const float* total,
               void* dscores, long long drs, long long dcs, cudaStream_t stream) {
  KM_TRY(check_route("kmeans_route_grad", dtype, rows, k, n, scale));
  if (rows == 0) return KM_OK;
  const int size = elem_size(dtype);
  if (!dweights || !ids || !weights || !aligned(dweights, 4) || !aligned(ids, 4) || !aligned(weights, 4) || !dscores ||
      !aligned(dscores, size) || !strides_ok(drs, dcs))
    KM_FAIL(KM_EINVAL, "kmeans_route_grad: bad argument");
  if (over_all && (!scores || !aligned(scores, size) || !strides_ok(rs, cs) || !best || !total || !aligned(best, 4) || !aligned(total, 4)))
    KM_FAIL(KM_EINVAL, "kmeans_route_grad: weights over all clusters need the scores, best and total");
  if (!((dcs == 1 && (drs >= k || rows == 1)) || (drs == 1 && (dcs >= (long long)rows || k == 1))))
    KM_FAIL(KM_EINVAL, "kmeans_route_grad: dscores must lie row after row or cluster after cluster");
  int sms = 0, rc = KM_OK;
  KM_TRY(sm_count(&sms));
  KM_ROWS_DTYPE(dtype, T,
      rc = route_grad_launch<T>(dweights, static_cast<const T*>(scores), rs, cs, (int)rows, k, n, scale, over_all != 0, ids, weights,
                                best, total, static_cast<T*>(dscores), drs, dcs, sms, stream));
  return rc;
}

}  // namespace

extern "C" {

int kmeans_route(int dtype, const void* scores, long long row_stride, long long col_stride, size_t rows, int k, int n, float scale,
                 int over_all, int32_t* ids, float* weights, float* best, float* total, void* stream) {
  return guarded("kmeans_route", [&] {
    return route(dtype, scores, row_stride, col_stride, rows, k, n, scale, over_all, ids, weights, best, total, as_stream(stream));
  });
}
int kmeans_route_grad(int dtype, const float* dweights, const void* scores, long long row_stride, long long col_stride, size_t rows,
                      int k, int n, float scale, int over_all, const int32_t* ids, const float* weights, const float* best,
                      const float* total, void* dscores, long long drow_stride, long long dcol_stride, void* stream) {
  return guarded("kmeans_route_grad", [&] {
    return route_grad(dtype, dweights, scores, row_stride, col_stride, rows, k, n, scale, over_all, ids, weights, best, total, dscores,
                      drow_stride, dcol_stride, as_stream(stream));
  });
}

}  // extern "C"

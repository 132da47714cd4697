// Shared by the row operators (kmeans_rows.cu): element types, argument checks, launch helpers.
#pragma once

#include <cuda_bf16.h>

#include <atomic>
#include <cmath>
#include <exception>

#include "km_common.cuh"

namespace km {
namespace rows {

// ---- elements -----------------------------------------------------------------
// Everything is computed in float32; a value is rounded once, to nearest, when it is stored.
template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_f<__half>(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f<float>(float v) { return v; }
template <> __device__ __forceinline__ __half from_f<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ float warp_sum_f(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over each half of the warp, the same in all its lanes.
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the CTA, the same in every thread; `red` holds 32 floats and may be used again after the next barrier.
__device__ __forceinline__ float cta_sum(float v, float* red) {
  v = warp_sum_f(v);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = (threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0.f;
  s = warp_sum_f(s);
  __syncthreads();
  return s;
}

// ---- host side ----------------------------------------------------------------
constexpr size_t kMaxRows = 0x7fff0000ULL;   // a row or a place is an int, and a grid has room for a few CTAs more
constexpr size_t kMaxCols = 0x7fff0000ULL;   // a column is an int, and a walk steps behind the last one by what a CTA takes at a time
constexpr size_t kMaxSumCols = 0x3fff0000ULL;   // the same of the gradients of weight and bias, which lie behind each other

inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }
inline int elem_size(int dtype) {
  switch (dtype) {
    case KM_DTYPE_F32: return 4;
    case KM_DTYPE_F16: return 2;
    case KM_DTYPE_BF16: return 2;
    default: return 0;
  }
}
inline bool aligned(const void* p, size_t to) { return (reinterpret_cast<uintptr_t>(p) & (to - 1)) == 0; }

// A row-major block the caller passes: pointer, row stride in elements.  Row starts must fit 63 bits of bytes.
inline bool block_ok(const void* p, long long stride, size_t rows, size_t cols, int size, bool output) {
  if (!p || !aligned(p, size) || stride < 0) return false;
  if (output && rows > 1 && (unsigned long long)stride < cols) return false;   // rows would overlap
  return rows <= kMaxRows && cols <= kMaxCols && (unsigned long long)stride <= (1ULL << 31);
}

// Whether every row of a block starts on a 16-byte boundary and is whole pieces of 16 bytes long.
inline bool rows_aligned(const void* p, long long stride, size_t rows, size_t cols, int size) {
  return aligned(p, 16) && (cols * size) % 16 == 0 && (rows <= 1 || (stride * size) % 16 == 0);
}

// Multiprocessors of the current device, asked once per device.
inline int sm_count(int* out) {
  static std::mutex m;
  static int count[64] = {};
  int dev = 0;
  cudaError_t ce = cudaGetDevice(&dev);
  if (ce == cudaErrorNoDevice || ce == cudaErrorInsufficientDriver) KM_FAIL(KM_ENODEV, "no CUDA device visible");
  KM_CUDA(ce);
  if (dev < 0 || dev >= 64) KM_FAIL(KM_ENODEV, "device index out of range");
  std::lock_guard<std::mutex> lock(m);
  if (count[dev] == 0) KM_CUDA(cudaDeviceGetAttribute(&count[dev], cudaDevAttrMultiProcessorCount, dev));
  *out = count[dev];
  return KM_OK;
}

// CTAs of a kernel that fit a multiprocessor at once, asked once per number of threads.
struct ResidentCtas {
  std::atomic<int> known[33] = {};     // by warps
  template <typename F>
  int get(F fn, int threads, size_t smem, int* out) {
    std::atomic<int>& k = known[threads / 32];
    *out = k.load(std::memory_order_relaxed);
    if (*out == 0) {
      KM_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(out, fn, threads, smem));
      *out = std::max(1, *out);
      k.store(*out, std::memory_order_relaxed);
    }
    return KM_OK;
  }
};

// A kernel that is put in place while the one before it on the stream still runs.  Before it waits for that one (wait_for_previous) it may
// read only what was there when that one began - an input of both - and write nothing but its own shared memory.
template <typename... P, typename... A>
int launch_early(void (*fn)(P...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, A... args) {
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  KM_CUDA(cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...));
  return KM_OK;
}
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// What a C entry point runs: nothing may leave it but a code.
template <typename F>
int guarded(const char* name, F&& f) noexcept {
  try {
    return f();
  } catch (const std::bad_alloc&) {
    return KM_ENOMEM;
  } catch (const std::exception& e) {
    try { set_error(std::string(name) + ": " + e.what()); } catch (...) {}
    return KM_EINVAL;
  } catch (...) {
    return KM_EINVAL;
  }
}

#define KM_ROWS_DTYPE(dtype, T, ...)                                     \
  do {                                                                   \
    switch (dtype) {                                                     \
      case KM_DTYPE_F32: { using T = float; __VA_ARGS__; } break;        \
      case KM_DTYPE_F16: { using T = __half; __VA_ARGS__; } break;       \
      case KM_DTYPE_BF16: { using T = __nv_bfloat16; __VA_ARGS__; } break; \
      default: break;                                                    \
    }                                                                    \
  } while (0)

}  // namespace rows
}  // namespace km

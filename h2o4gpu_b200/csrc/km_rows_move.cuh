// Rows to their places and back (slot and source as in km_rows_sort.cuh).
//   dispatch: out[slot(t, j)] = x[t]              combine: y[t] = sum over j of w(t, j) in[slot(t, j)]
//   combine's gradient: din[slot(t, j)] = w(t, j) dy[t],  dw(t, j) = <dy[t], in[slot(t, j)]>
// All are bound by memory.  They walk over the rows in the caller's order, so that a row of x, y or dy moves once and a sorted row once.
#pragma once

#include "km_rows_vec.cuh"

namespace km {
namespace rows {

constexpr int kMoveThreads = 256;

// Work is cut into pieces of 16 bytes.  Aligned rows: piece i of all rows together goes to thread i, so narrow rows fill warps too.  Others:
// a warp takes 32 consecutive pieces of one row (the lanes pass each other what lies across two words).
struct MoveItem {
  int row, piece;
  bool valid;
};
template <bool ALIGNED>
__device__ __forceinline__ MoveItem move_item(long long block, int rows, int pieces) {
  MoveItem m;
  const long long thread = block * kMoveThreads + threadIdx.x;
  if (ALIGNED) {
    // (32-bit division while the numbers allow it)
    const long long r = thread <= 0xffffffffLL ? (long long)((unsigned int)thread / (unsigned int)pieces) : thread / pieces;
    m.row = (int)r;
    m.piece = (int)(thread - r * pieces);
    m.valid = r < rows;
  } else {
    const int per_row = (pieces + 31) / 32;
    const long long warp = thread / 32, r = warp / per_row;
    m.row = (int)r;
    m.piece = (int)(warp - r * per_row) * 32 + (threadIdx.x & 31);
    m.valid = r < rows;      // a whole warp
  }
  return m;
}
inline long long move_blocks(size_t rows, int pieces, bool al) {
  const long long threads = al ? (long long)rows * pieces : (long long)rows * ((pieces + 31) / 32) * 32;
  return (threads + kMoveThreads - 1) / kMoveThreads;
}

template <typename T>
__device__ __forceinline__ Piece<T> zero_piece() {
  Piece<T> p;
  p.q = make_uint4(0u, 0u, 0u, 0u);
  return p;
}

// Zero rows at the places without an entry: warp by warp over the places.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void zero_unused(T* out, long long os, int d, const int* source, int capacity, long long block,
                                            long long blocks) {
  const int lane = threadIdx.x & 31, pieces = (d + Piece<T>::V - 1) / Piece<T>::V;
  for (long long p0 = (block * blockDim.x + threadIdx.x) / 32 * 32; p0 < capacity; p0 += blocks * blockDim.x) {
    const bool mine = p0 + lane < capacity && source[p0 + lane] < 0;
    for (unsigned int left = __ballot_sync(0xffffffffu, mine); left; left &= left - 1) {
      T* row = out + (p0 + __ffs(left) - 1) * os;
      for (int i = lane; i < (pieces + 31) / 32 * 32; i += 32) store_piece<T, ALIGNED>(row, i, d, zero_piece<T>());
    }
  }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kMoveThreads)
dispatch_kernel(const T* x, long long xs, int rows, int d, int n, const int* slot, const int* source, int capacity, T* out,
                long long os, long long blocks) {
  if (blockIdx.x >= blocks) {
    zero_unused<T, ALIGNED>(out, os, d, source, capacity, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const MoveItem m = move_item<ALIGNED>(blockIdx.x, rows, (d + Piece<T>::V - 1) / Piece<T>::V);
  if (!m.valid) return;
  const Piece<T> v = load_piece<T, ALIGNED>(x + m.row * xs, m.piece, d);
  const int* sl = slot + (long long)m.row * n;
  for (int j = 0; j < n; ++j) {
    const int p = sl[j];
    if (p >= 0 && p < capacity) store_piece<T, ALIGNED>(out + p * os, m.piece, d, v);
  }
}

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kMoveThreads)
combine_kernel(const T* in, long long is, int capacity, int d, const int* slot, const float* weights, int rows, int n, T* y,
               long long ys) {
  constexpr int H = Piece<T>::V / 2, AT_ONCE = 4;
  const MoveItem m = move_item<ALIGNED>(blockIdx.x, rows, (d + Piece<T>::V - 1) / Piece<T>::V);
  if (!m.valid) return;
  const int* sl = slot + (long long)m.row * n;
  const float* w = weights ? weights + (long long)m.row * n : nullptr;
  float2 sum[H];
#pragma unroll
  for (int e = 0; e < H; ++e) sum[e] = both(0.f);
  for (int j0 = 0; j0 < n; j0 += AT_ONCE) {
    Piece<T> v[AT_ONCE];
    float f[AT_ONCE];
    bool there[AT_ONCE];
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      const int p = j0 + u < n ? sl[j0 + u] : -1;
      there[u] = p >= 0 && p < capacity;
      f[u] = there[u] && w ? w[j0 + u] : 1.f;
      v[u] = there[u] ? load_piece<T, ALIGNED>(in + p * is, m.piece, d) : zero_piece<T>();
    }
#pragma unroll
    for (int u = 0; u < AT_ONCE; ++u) {
      if (!there[u]) continue;
      float2 g[H];
      unpack(v[u], g);
#pragma unroll
      for (int e = 0; e < H; ++e) sum[e] = fma2(both(f[u]), g[e], sum[e]);
    }
  }
  store_piece<T, ALIGNED>(y + m.row * ys, m.piece, d, pack<T>(sum));
}

// One CTA per row, its threads over the row's pieces; the dot products of up to 32 entries are joined over the warps at once.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kMoveThreads)
combine_grad_kernel(const T* dy, long long dys, const T* in, long long is, int capacity, int d, const int* slot, const int* source,
                    const float* weights, int rows, int n, T* din, long long dis, float* dweights) {
  constexpr int H = Piece<T>::V / 2;
  __shared__ float red[32][kMoveThreads / 32 + 1];
  if ((int)blockIdx.x >= rows) {
    zero_unused<T, ALIGNED>(din, dis, d, source, capacity, blockIdx.x - rows, gridDim.x - rows);
    return;
  }
  const int t = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x / 32, warps = blockDim.x / 32;
  const int pieces = ((d + Piece<T>::V - 1) / Piece<T>::V + 31) / 32 * 32;
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int nj = min(32, n - j0);
    for (int j = 0; j < nj; ++j) {
      const long long at = (long long)t * n + j0 + j;
      const int p = slot[at];
      float dot = 0.f;
      if (p >= 0 && p < capacity) {
        const float2 w = both(weights[at]);
        float2 s = both(0.f);
        for (int i = threadIdx.x; i < pieces; i += blockDim.x) {
          float2 g[H], v[H];
          unpack(load_piece<T, ALIGNED>(dy + t * dys, i, d), g);
          unpack(load_piece<T, ALIGNED>(in + p * is, i, d), v);
#pragma unroll
          for (int e = 0; e < H; ++e) {
            s = fma2(g[e], v[e], s);
            g[e] = mul2(g[e], w);
          }
          store_piece<T, ALIGNED>(din + p * dis, i, d, pack<T>(g));
        }
        dot = warp_sum_f(s.x + s.y);
      }
      if (lane == 0) red[j][warp] = dot;
    }
    __syncthreads();
    if ((int)threadIdx.x < nj) {
      float s = 0.f;
      for (int i = 0; i < warps; ++i) s += red[threadIdx.x][i];
      dweights[(long long)t * n + j0 + threadIdx.x] = s;
    }
    __syncthreads();
  }
}

}  // namespace rows
}  // namespace km

// Rows to their places and back (slot and source as in km_rows_sort.cuh).
//   dispatch: out[slot(t, j)] = x[t]              combine: y[t] = sum over j of w(t, j) in[slot(t, j)]
//   combine's gradient: din[slot(t, j)] = w(t, j) dy[t],  dw(t, j) = <dy[t], in[slot(t, j)]>
// All are bound by memory.  They walk over the rows in the caller's order, so that a row of x, y or dy moves once and a sorted row once.
#pragma once

#include "km_rows_vec.cuh"

namespace km {
namespace rows {

constexpr int kMoveThreads = 256;

// Work is cut into words of 16 bytes of the rows that are written: word i of a row holds its columns from i V - before_row on.  Those of
// the rows that are read may lie across two words there (load_window).  Words of all rows together go to consecutive threads, so that
// narrow rows fill warps too.
struct MoveItem {
  int row, word;
};
__device__ __forceinline__ MoveItem move_item(int words) {
  const long long thread = (long long)blockIdx.x * kMoveThreads + threadIdx.x;
  // (32-bit division while the numbers allow it)
  const long long r = thread <= 0xffffffffLL ? (long long)((unsigned int)thread / (unsigned int)words) : thread / words;
  return {(int)min(r, 0x7fffffffLL), (int)(thread - r * words)};
}
// Words that a row can lie across.
inline int move_words(size_t cols, int size, bool al) {
  const size_t v = 16 / size;
  return (int)(al ? cols / v : (cols + 2 * v - 2) / v);
}
inline long long move_blocks(size_t rows, int words) { return ((long long)rows * words + kMoveThreads - 1) / kMoveThreads; }

template <typename T>
__device__ __forceinline__ Piece<T> zero_piece() {
  Piece<T> p;
  p.q = make_uint4(0u, 0u, 0u, 0u);
  return p;
}
// The V elements at column c of a row.
template <typename T, bool ALIGNED>
__device__ __forceinline__ Piece<T> load_at(const T* row, int c, const Span<T>& in) {
  if (!ALIGNED) return load_window(row + c, in);
  Piece<T> p;
  p.q = *reinterpret_cast<const uint4*>(row + c);
  return p;
}

// Zero rows at the places without an entry: warp by warp over the places.
template <typename T>
__device__ __forceinline__ void zero_unused(T* out, long long os, int d, const int* source, int capacity, long long block,
                                            long long blocks) {
  constexpr int V = Piece<T>::V;
  const int tid = threadIdx.x + threadIdx.y * blockDim.x, threads = blockDim.x * blockDim.y, lane = tid & 31;
  for (long long p0 = (block * threads + tid) / 32 * 32; p0 < capacity; p0 += blocks * threads) {
    const bool mine = p0 + lane < capacity && source[p0 + lane] < 0;
    for (unsigned int left = __ballot_sync(0xffffffffu, mine); left; left &= left - 1) {
      T* row = out + (p0 + __ffs(left) - 1) * os;
      for (int c = lane * V - before_row(row); c < d; c += 32 * V) store_word(row, c, d, zero_piece<T>());
    }
  }
}

// Bound by memory: 32,768 x 2048 bfloat16 to four places each take 105 us, 6.4 TB/s (0.97 of the copy rate), four fifths of it written; with 64
// groups on multiples of 128, 137 us: a warp zeroes the places without an entry among its 32 one after the other, after the rows.  Unaligned
// rows are read anew for each place, from L1, as each has a shift of its own.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(kMoveThreads)
dispatch_kernel(const T* x, long long xs, Span<T> xin, int rows, int d, int words, int n, const int* slot, const int* source,
                int capacity, T* out, long long os, long long blocks) {
  constexpr int V = Piece<T>::V;
  if (blockIdx.x >= blocks) {
    zero_unused(out, os, d, source, capacity, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const MoveItem m = move_item(words);
  if (m.row >= rows) return;
  const T* row = x + m.row * xs;
  const int* sl = slot + (long long)m.row * n;
  Piece<T> v;
  if (ALIGNED) v = load_at<T, true>(row, m.word * V, xin);
  for (int j = 0; j < n; ++j) {
    const int p = sl[j];
    if (p < 0 || p >= capacity) continue;
    T* to = out + p * os;
    if (ALIGNED) {
      *reinterpret_cast<uint4*>(to + m.word * V) = v.q;
    } else {
      const int c = m.word * V - before_row(to);
      if (c < d) store_word(to, c, d, load_at<T, false>(row, c, xin));
    }
  }
}

// AT_ONCE entries are on their way together.  Bound by memory: 16,384 x 2048 bfloat16, eight each, take 93 us, 0.99 of the copy rate.
// Many warps hide more than many loads a thread do: two rows a thread with twice the registers took 55 us where this takes 37 (20,011 x 1021
// float16, two entries), two words a thread the same 37.
template <typename T, bool ALIGNED, int AT_ONCE>
__global__ void __launch_bounds__(kMoveThreads, AT_ONCE > 2 ? 5 : ALIGNED ? 6 : 8)
combine_kernel(const T* in, long long is, Span<T> iin, int capacity, int d, int words, const int* slot, const float* weights, int rows,
               int n, T* y, long long ys) {
  constexpr int V = Piece<T>::V, H = V / 2;
  const MoveItem m = move_item(words);
  if (m.row >= rows) return;
  T* to = y + m.row * ys;
  const int c = m.word * V - (ALIGNED ? 0 : before_row(to));
  if (c >= d) return;
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
      if (!there[u]) continue;
      f[u] = w ? w[j0 + u] : 1.f;
      v[u] = load_at<T, ALIGNED>(in + p * is, c, iin);
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
  const Piece<T> o = pack<T>(sum);
  if (ALIGNED) *reinterpret_cast<uint4*>(to + c) = o.q;
  else store_word(to, c, d, o);
}

// blockDim.x threads (whole warps) take a row, blockDim.y rows share a CTA; the dot products are joined over a row's warps, 32 entries at
// a time.  AT_ONCE entries share a row of dy and are on their way together.  Bound by the latency of scattered rows: 15,013 x 784 float32, three
// each, take 64 us, 0.80 of the copy rate; CTAs of 256 threads with 60 registers took 77.
constexpr int kCombineGradThreads = 128;
// The row that row y of a CTA's threads takes, -1 behind the last one: those threads leave at once, before an address is formed from it.
__host__ __device__ __forceinline__ int combine_grad_row(int block, int per_cta, int y, int rows) {
  const int t = block * per_cta + y;
  return t < rows ? t : -1;
}
// CTAs a processor: ten hold four 16-bit entries at once only with spills (8192 x 2048 bfloat16, four entries: 68.2 us, 66.2 with nine; in
// float32, 8192 x 1024: 62.7 and 63.2).
template <typename T, bool ALIGNED, int AT_ONCE>
constexpr int combine_grad_ctas() { return !ALIGNED ? 6 : AT_ONCE == 4 && sizeof(T) == 2 ? 9 : 10; }
template <typename T, bool ALIGNED, int AT_ONCE>
__global__ void __launch_bounds__(kCombineGradThreads, combine_grad_ctas<T, ALIGNED, AT_ONCE>())
combine_grad_kernel(const T* dy, long long dys, Span<T> gin, const T* in, long long is, Span<T> iin, int capacity, int d, int words,
                    const int* slot, const int* source, const float* weights, int rows, int n, T* din, long long dis, float* dweights,
                    int blocks) {
  constexpr int V = Piece<T>::V, H = V / 2;
  __shared__ float red[kCombineGradThreads / 32][32];
  if ((int)blockIdx.x >= blocks) {
    zero_unused(din, dis, d, source, capacity, blockIdx.x - blocks, gridDim.x - blocks);
    return;
  }
  const int t = combine_grad_row(blockIdx.x, blockDim.y, threadIdx.y, rows), lane = threadIdx.x & 31, warps = blockDim.x / 32;
  if (t < 0) return;      // (a barrier waits for the threads that have not left)
  const T* gr = dy + t * dys;
  for (int j0 = 0; j0 < n; j0 += 32) {
    const int nj = min(32, n - j0);
    float mine = 0.f;       // lane j: this warp's part of entry j
    for (int u0 = 0; u0 < nj; u0 += AT_ONCE) {
      int p[AT_ONCE];
      float w[AT_ONCE];
      float2 dot[AT_ONCE];
      const T* from[AT_ONCE];
      T* to[AT_ONCE];
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const long long at = (long long)t * n + j0 + u0 + u;
        p[u] = u0 + u < nj ? slot[at] : -1;
        if (p[u] >= capacity) p[u] = -1;
        w[u] = p[u] >= 0 ? weights[at] : 0.f;
        from[u] = in + (long long)max(p[u], 0) * is;
        to[u] = din + (long long)max(p[u], 0) * dis;
        dot[u] = both(0.f);
      }
      for (int i = threadIdx.x; i < words; i += blockDim.x) {
        Piece<T> g, v[AT_ONCE], gu[AT_ONCE];
        if (ALIGNED) g = load_at<T, true>(gr, i * V, gin);
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          if (p[u] < 0) continue;
          const int c = i * V - (ALIGNED ? 0 : before_row(to[u]));
          if (!ALIGNED && c >= d) {
            gu[u] = v[u] = zero_piece<T>();
            continue;
          }
          v[u] = load_at<T, ALIGNED>(from[u], c, iin);
          if (!ALIGNED) {
            gu[u] = load_at<T, false>(gr, c, gin);
            clip_piece(gu[u], c, d);
            clip_piece(v[u], c, d);
          }
        }
#pragma unroll
        for (int u = 0; u < AT_ONCE; ++u) {
          if (p[u] < 0) continue;
          float2 a[H], b[H];
          unpack(ALIGNED ? g : gu[u], a);
          unpack(v[u], b);
#pragma unroll
          for (int e = 0; e < H; ++e) {
            dot[u] = fma2(a[e], b[e], dot[u]);
            a[e] = mul2(a[e], both(w[u]));
          }
          const Piece<T> o = pack<T>(a);
          if (ALIGNED) {
            *reinterpret_cast<uint4*>(to[u] + i * V) = o.q;
          } else {
            const int c = i * V - before_row(to[u]);
            if (c < d) store_word(to[u], c, d, o);
          }
        }
      }
#pragma unroll
      for (int u = 0; u < AT_ONCE; ++u) {
        const float s = warp_sum_f(dot[u].x + dot[u].y);
        if (lane == u0 + u) mine = s;
      }
    }
    if (warps > 1) {
      float* row = red[threadIdx.y * warps];
      red[threadIdx.y * warps + threadIdx.x / 32][lane] = mine;
      __syncthreads();
      mine = 0.f;
      if (threadIdx.x < 32)
        for (int i = 0; i < warps; ++i) mine += row[i * 32 + lane];
      __syncthreads();
    }
    if (threadIdx.x < 32 && lane < nj) dweights[(long long)t * n + j0 + lane] = mine;
  }
}

// Warps for a row: one (its lanes keep many loads on their way, nothing is joined) while there are rows for all warps that fit the device
// (64 a processor), more for fewer rows.
inline int combine_grad_warps(size_t rows, int words, int sms) {
  int w = 1;
  while (w < kCombineGradThreads / 32 && (words + 31) / 32 > w && rows * w < (size_t)sms * 64) w *= 2;
  return w;
}

}  // namespace rows
}  // namespace km

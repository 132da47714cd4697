// Rows in 16-byte pieces, whatever their alignment.
// Piece i of a row is its elements [i V, i V + V).  Where rows start on 16-byte boundaries a piece is one load or store.  Elsewhere a
// piece lies across two aligned words of 16 bytes: a load takes both and shifts (the second is the next lane's first, so it comes from
// L1), a store passes what does not fit its own word to the next lane.  A word may hold elements beside the row, but never any outside the
// block that the rows belong to (Span): there it is taken apart element by element.
#pragma once

#include "km_rows.cuh"

namespace km {
namespace rows {

template <typename T> struct Piece {
  static constexpr int V = 16 / (int)sizeof(T);
  union {
    uint4 q;
    unsigned int w[4];
    T e[V];
  };
  __device__ __forceinline__ Piece() {}
};

// Two float32 operations in one instruction.
__device__ __forceinline__ unsigned long long as_u64(float2 a) {
  unsigned long long r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a.x), "f"(a.y));
  return r;
}
__device__ __forceinline__ float2 as_f2(unsigned long long a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a));
  return r;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  unsigned long long r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as_u64(a)), "l"(as_u64(b)));
  return as_f2(r);
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(as_u64(a)), "l"(as_u64(b)));
  return as_f2(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(as_u64(a)), "l"(as_u64(b)), "l"(as_u64(c)));
  return as_f2(r);
}
__device__ __forceinline__ float2 both(float a) { return make_float2(a, a); }

// A piece as pairs of float32 and back (each value rounded once, to nearest).
template <typename T> __device__ __forceinline__ float2 word_pair(unsigned int w);
template <> __device__ __forceinline__ float2 word_pair<__nv_bfloat16>(unsigned int w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <> __device__ __forceinline__ float2 word_pair<__half>(unsigned int w) {
  __half2 h;
  memcpy(&h, &w, 4);
  return __half22float2(h);
}
template <typename T> __device__ __forceinline__ unsigned int pair_word(float2 f);
template <> __device__ __forceinline__ unsigned int pair_word<__nv_bfloat16>(float2 f) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(f.x, f.y);
  unsigned int w;
  memcpy(&w, &h, 4);
  return w;
}
template <> __device__ __forceinline__ unsigned int pair_word<__half>(float2 f) {
  const __half2 h = __floats2half2_rn(f.x, f.y);
  unsigned int w;
  memcpy(&w, &h, 4);
  return w;
}
template <typename T>
__device__ __forceinline__ void unpack(const Piece<T>& p, float2 (&f)[Piece<T>::V / 2]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = make_float2(__uint_as_float(p.w[0]), __uint_as_float(p.w[1]));
    f[1] = make_float2(__uint_as_float(p.w[2]), __uint_as_float(p.w[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = word_pair<T>(p.w[i]);
  }
}
template <typename T>
__device__ __forceinline__ Piece<T> pack(const float2 (&f)[Piece<T>::V / 2]) {
  Piece<T> p;
  if constexpr (sizeof(T) == 4) {
    p.q = make_uint4(__float_as_uint(f[0].x), __float_as_uint(f[0].y), __float_as_uint(f[1].x), __float_as_uint(f[1].y));
  } else {
    p.q = make_uint4(pair_word<T>(f[0]), pair_word<T>(f[1]), pair_word<T>(f[2]), pair_word<T>(f[3]));
  }
  return p;
}

// Asynchronous copies of 16 bytes to shared memory, past L1; a thread waits for its own, all but the `N` newest groups.
__device__ __forceinline__ void copy_async(uint4* to, const uint4* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned int)__cvta_generic_to_shared(to)), "l"(from) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// Bytes [shift, shift + 16) of the 32 bytes a, b.
__device__ __forceinline__ uint4 shift_words(uint4 a, uint4 b, unsigned int shift) {
  unsigned int w0 = a.x, w1 = a.y, w2 = a.z, w3 = a.w, w4 = b.x, w5 = b.y, w6 = b.z, w7 = b.w;
  if (shift & 8) { w0 = w2; w1 = w3; w2 = w4; w3 = w5; w4 = w6; w5 = w7; }
  if (shift & 4) { w0 = w1; w1 = w2; w2 = w3; w3 = w4; w4 = w5; }
  const unsigned int bits = (shift & 3) * 8;
  return make_uint4(__funnelshift_r(w0, w1, bits), __funnelshift_r(w1, w2, bits), __funnelshift_r(w2, w3, bits),
                    __funnelshift_r(w3, w4, bits));
}

// From the first element of a block's first row to behind the last one of its last row.
template <typename T>
struct Span {
  const T* lo;
  const T* hi;
};
template <typename T>
inline Span<T> span_of(const void* p, long long stride, size_t rows, size_t cols) {
  const T* lo = static_cast<const T*>(p);
  return {lo, rows ? lo + (long long)(rows - 1) * stride + cols : lo};
}

// V elements from `from` on (any alignment); what lies outside the span is zero.
template <typename T>
__device__ __forceinline__ Piece<T> load_window(const T* from, const Span<T>& in) {
  constexpr int V = Piece<T>::V;
  Piece<T> p;
  const unsigned int off = (unsigned int)(reinterpret_cast<uintptr_t>(from) & 15);
  const T* word = from - off / sizeof(T);
  if (off == 0) {      // (as a rule the same for a whole row)
    if (from >= in.lo && from + V <= in.hi) {
      p.q = *reinterpret_cast<const uint4*>(from);
      return p;
    }
  } else if (word >= in.lo && word + 2 * V <= in.hi) {
    p.q = shift_words(*reinterpret_cast<const uint4*>(word), *reinterpret_cast<const uint4*>(word + V), off);
    return p;
  }
  p.q = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (from + e >= in.lo && from + e < in.hi) p.e[e] = from[e];
  return p;
}

// The elements of a piece that starts at column c and lie outside [0, d) become zero.
template <typename T>
__device__ __forceinline__ void clip_piece(Piece<T>& p, int c, int d) {
  constexpr int V = Piece<T>::V;
  if (c >= 0 && c + V <= d) return;
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (c + e < 0 || c + e >= d) p.e[e] = from_f<T>(0.f);
}

// Piece i of the row at `row` with d elements; zeros behind the row's end.  ALIGNED: the row starts on a 16-byte boundary and is
// whole pieces long.
template <typename T, bool ALIGNED>
__device__ __forceinline__ Piece<T> load_piece(const T* row, int i, int d, const Span<T>& in) {
  constexpr int V = Piece<T>::V;
  Piece<T> p;
  const int c = i * V;
  if (ALIGNED) {
    p.q = c < d ? *reinterpret_cast<const uint4*>(row + c) : make_uint4(0u, 0u, 0u, 0u);
    return p;
  }
  if (c >= d) {
    p.q = make_uint4(0u, 0u, 0u, 0u);
    return p;
  }
  p = load_window(row + c, in);
  clip_piece(p, c, d);
  return p;
}

// Stores the elements of `p` that lie in [0, d), the first at column c of the row; row + c is a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void store_word(T* row, int c, int d, const Piece<T>& p) {
  constexpr int V = Piece<T>::V;
  if (c >= 0 && c + V <= d) {
    *reinterpret_cast<uint4*>(row + c) = p.q;
    return;
  }
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (c + e >= 0 && c + e < d) row[c + e] = p.e[e];
}
// Elements of the row's first word that lie before the row.
template <typename T>
__device__ __forceinline__ int before_row(const T* row) { return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T)); }

// Stores piece i of the row.  Not ALIGNED: all 32 lanes call it with consecutive pieces (store_pieces with one piece a lane).
template <typename T, bool ALIGNED>
__device__ __forceinline__ void store_piece(T* row, int i, int d, const Piece<T>& p);

// Stores NV pieces a lane, piece first + 32 p of the row in lane `first % 32` of its warp: what does not fit a piece's own word goes to the
// next lane, and from the last lane to the first one's next piece.  All 32 lanes call it; pieces behind the row's end store nothing.
template <typename T, int NV>
__device__ __forceinline__ void store_pieces(T* row, int first, int d, const Piece<T> (&p)[NV]) {
  constexpr int V = Piece<T>::V;
  const unsigned int off = (unsigned int)(reinterpret_cast<uintptr_t>(row) & 15);   // the same in every lane
  const int lane = threadIdx.x & 31, m = (int)(off / sizeof(T));
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = (first + i * 32) * V;
    if (m == 0) {
      if (c < d) store_word(row, c, d, p[i]);
      continue;
    }
    // this lane's word: the last m elements of the piece before, then its own first V - m
    const Piece<T>& last = p[i ? i - 1 : 0];
    Piece<T> before;
#pragma unroll
    for (int k = 0; k < 4; ++k) before.w[k] = __shfl_sync(0xffffffffu, lane == 31 ? last.w[k] : p[i].w[k], (lane + 31) & 31);
    if (i == 0 && lane == 0) {      // the piece before is another warp's, or none
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (e < V - m && c + e < d) row[c + e] = p[i].e[e];
    } else if (c - m < d) {
      before.q = shift_words(before.q, p[i].q, 16 - off);
      store_word(row, c - m, d, before);
    }
  }
  const int c = (first + (NV - 1) * 32) * V;
  if (lane == 31)
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e >= V - m && c + e < d) row[c + e] = p[NV - 1].e[e];
}

template <typename T, bool ALIGNED>
__device__ __forceinline__ void store_piece(T* row, int i, int d, const Piece<T>& p) {
  if (ALIGNED) {
    if (i * Piece<T>::V < d) *reinterpret_cast<uint4*>(row + i * Piece<T>::V) = p.q;
  } else {
    const Piece<T> one[1] = {p};
    store_pieces(row, i, d, one);
  }
}

// Whether all words that hold elements of the row lie in the span.
template <typename T>
__device__ __forceinline__ bool words_inside(const T* row, int d, const Span<T>& in) {
  constexpr int V = Piece<T>::V;
  const T* lo = row - before_row(row);
  return lo >= in.lo && lo + (before_row(row) + d + V - 1) / V * V <= in.hi;
}

}  // namespace rows
}  // namespace km

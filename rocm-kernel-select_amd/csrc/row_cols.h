// Rows in registers: what the kernels of the norms share.  A row's columns are loaded as vectors of any
// alignment, and reduced over the threads that have them.
#pragma once
#include "atk_common.h"

namespace atk {

// V columns of a row of N from c on, as they are in memory (element alignment only: rows of any width).
// No branch and no conversion, so a thread's loads are all in flight together: with a branch around each,
// every load waited for the one before it (8192 x 2048, residual, fp8, 33 us).  What would pass the row's
// end is loaded from further left.  TINY: rows shorter than V.
template <typename T, int V>
struct Cols {
  T e[V];
};
template <typename T, int V, bool TINY>
__device__ __forceinline__ Cols<T, V> load_raw(const T* __restrict__ p, int c, int N) {
  Cols<T, V> o;
  if constexpr (TINY) {
#pragma unroll
    for (int i = 0; i < V; ++i) o.e[i] = c + i < N ? p[c + i] : static_cast<T>(0.f);
  } else {
    __builtin_memcpy(o.e, p + (c < N - V ? c : N - V), V * sizeof(T));
  }
  return o;
}
// In their places, fp32, zeros from column N on.
template <typename T, int V, bool TINY>
__device__ __forceinline__ void to_cols(Cols<T, V> r, int c, int N, float* o) {
  if constexpr (!TINY) {
    const int past = c + V - N;
    if (past > 0) {
      unsigned __int128 u;
      __builtin_memcpy(&u, r.e, sizeof(u));
      u = past < V ? u >> (past * (int)sizeof(T) * 8) : 0;
      __builtin_memcpy(r.e, &u, sizeof(u));
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = to_f32(r.e[i]);
}
// Loads before this are issued before anything after it.
__device__ __forceinline__ void loads_issued() { asm volatile("" ::: "memory"); }

template <typename T, int V>
__device__ __forceinline__ void store_cols(T* __restrict__ p, int c, int N, const float* v) {
  if (c + V <= N) {
    T e[V];
#pragma unroll
    for (int i = 0; i < V; ++i) e[i] = from_f32<T>(v[i]);
    __builtin_memcpy(p + c, e, V * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < N) p[c + i] = from_f32<T>(v[i]);
  }
}

// The weight's columns of a thread's vectors: of the rows' type they come with the loads of the rows
// (raw), as fp32 later, for vectors j0 .. j0 + J - 1 at once; ones without a weight.
template <typename T, int V, bool TINY, int TPR, int J>
__device__ __forceinline__ void weight_raw(const void* w, int w_f32, int t, int j0, int N, Cols<T, V> (&r)[J]) {
  if (!w || w_f32) return;
#pragma unroll
  for (int j = 0; j < J; ++j) r[j] = load_raw<T, V, TINY>(static_cast<const T*>(w), (t + (j0 + j) * TPR) * V, N);
}
template <typename T, int V, bool TINY, int TPR, int J>
__device__ __forceinline__ void to_weight(const Cols<T, V> (&r)[J], const void* w, int w_f32, int t, int j0, int N,
                                          float (&o)[J][V]) {
  if (!w) {
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] = 1.f;
  } else if (!w_f32) {
#pragma unroll
    for (int j = 0; j < J; ++j) to_cols<T, V, TINY>(r[j], (t + (j0 + j) * TPR) * V, N, o[j]);
  } else {
    Cols<float, 4> e[J][V / 4];
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        e[j][i] = load_raw<float, 4, TINY>(static_cast<const float*>(w), (t + (j0 + j) * TPR) * V + 4 * i, N);
    loads_issued();
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V / 4; ++i)
        to_cols<float, 4, TINY>(e[j][i], (t + (j0 + j) * TPR) * V + 4 * i, N, o[j] + 4 * i);
  }
}

// Over each run of L lanes (a power of two up to 64), the same in each of them, order fixed; lane
// exchanges up to 16 lanes need no LDS.  Every lane of the wave takes part.
template <int L, typename F>
__device__ __forceinline__ float lanes_reduce(float v, F f) {
  if constexpr (L >= 2) v = f(v, dpp_mov<0xB1>(v));   // lane ^ 1
  if constexpr (L >= 4) v = f(v, dpp_mov<0x4E>(v));   // lane ^ 2
  if constexpr (L >= 8) v = f(v, dpp_mov<0x141>(v));  // mirrored in 8, whose fours have one value each
  if constexpr (L >= 16) v = f(v, dpp_mov<0x140>(v));
  if constexpr (L >= 32) v = f(v, __shfl_xor(v, 16, 64));
  if constexpr (L >= 64) v = f(v, __shfl_xor(v, 32, 64));
  return v;
}
// The larger of two magnitudes, a NaN above all: their bits are in that order.
__device__ __forceinline__ float max_abs(float a, float b) {
  const uint32_t x = __float_as_uint(a), y = __float_as_uint(b);
  return __uint_as_float(x > y ? x : y);
}
struct Max {
  __device__ __forceinline__ float operator()(float a, float b) const { return max_abs(a, b); }
};
struct Add {
  __device__ __forceinline__ float operator()(float a, float b) const { return a + b; }
};
// Over the TPR threads of a row.  TPR > 64 uses `red` (one float a wave), which the next call but one may
// use again, and has one barrier.
template <int TPR, typename F>
__device__ __forceinline__ float row_reduce(float v, float* red, F f) {
  v = lanes_reduce<TPR < 64 ? TPR : 64>(v, f);
  if constexpr (TPR > 64) {
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = red[0];
#pragma unroll
    for (int i = 1; i < TPR / 64; ++i) v = f(v, red[i]);
  }
  return v;
}

// Threads to a row and vectors to a thread.
struct RmsShape {
  int tpr, vpt;
};

// dw[c] = sum over parts of part[p][c], p < P, c < N, in a fixed order, rounded once to w_dtype.
int rows_dw(const float* part, void* dw, int P, int N, int w_dtype, hipStream_t s);

}  // namespace atk

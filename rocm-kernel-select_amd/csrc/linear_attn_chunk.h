// Linear attention over sequences in chunks of CT tokens: the kernels, one set for each type.
//
// With G the running sum of the log decays within a chunk, D_ij = exp(G_i - G_j) and S the state before it:
//   O  = scale (exp(G) (Q S) + lower(Q K^T * D) V)
//   S' = exp(G_last) S + K^T (exp(G_last - G) V)
// A workgroup of four waves has one head's segment of a sequence and a tile of V's columns, each wave NT times
// 16 of them.  The state stays in the accumulators from chunk to chunk: as it is, it is the next product's
// second operand.  Rows of a, b and c are staged in LDS in bf16 parts, the next chunk's loads in flight
// meanwhile; products over tokens read them transposed (ds_read_tr).
//
// Measured, bf16: 8192 tokens, 16 and 32 heads of 128 x 128, in 16 segments: states 44 us (100 MB read, 31 written), outputs
// 100 (134 + 31 and 67).  LDS is busy for 11 and 28 us of these, 34 and 41 % of that with bank conflicts, the matrix units
// for 10 and 26; a third of a wave's cycles it waits for memory or LDS, a third for its turn or a result, a quarter it
// issues vector instructions, most of them the splitting of S, of P and of the decayed c in parts.  Two workgroups a
// CU.  Without an effect: loads two chunks ahead, eight waves, chunks of 32, other pitches, raised priority.  S, P and the
// decayed c keep all their bits: two parts of S and P towards 16-bit outputs took a call from 143 to 133 us, and
// rounded results to the wrong side that are within 2^-17 of half way between two values.
#pragma once
#include <limits.h>

#include "linear_attn.h"

namespace atk {
namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

// Tokens of a chunk: 64, or 32 where the parts of 64 rows would not fit LDS twice.
template <typename T, int DA> inline constexpr int kLaC = kParts<T> == 1 ? 64 : 32;
// parts of fp32 factors (S, P, the decayed c): all their bits, also towards 16-bit outputs
constexpr int kLaOut = 3;

// Running sum over the wave of v / ln 2 in 64 bits, as two floats each; lane 63's sum in *last.
template <int CTRL, int ROWS>
__device__ __forceinline__ double la_dpp(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float2 la_running(float v, float2* last) {
  double s = (double)v * 1.4426950408889634;
  s += la_dpp<0x111, 0xF>(s);  // row_shr 1, 2, 4, 8: sums within 16 lanes
  s += la_dpp<0x112, 0xF>(s);
  s += la_dpp<0x114, 0xF>(s);
  s += la_dpp<0x118, 0xF>(s);
  s += la_dpp<0x142, 0xA>(s);  // row_bcast 15 into rows 1 and 3
  s += la_dpp<0x143, 0xC>(s);  // row_bcast 31 into rows 2 and 3
  const float2 r = make_float2((float)s, (float)(s - (double)(float)s));
  last->x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, r.x), 63));
  last->y = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, r.y), 63));
  return r;
}

// v[0..N) as NP parts of N bf16 each; WIDE: of any fp32 value.  Those from 3.39e38 on round up to infinity in bf16, so
// there the first part is bf16's largest value, and the others have what is left of it.
template <int NP, int N, bool WIDE, typename P>
__device__ __forceinline__ void la_parts(const float* v, P (&out)[NP]) {
  if constexpr (WIDE && NP > 1) {
    constexpr float kMost = 3.3895313892515355e38f;
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    float rest[N];
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      // (a NaN becomes some value here, and stays one in what is left)
      const b2 h = __builtin_convertvector((f2{__builtin_amdgcn_fmed3f(v[i], -kMost, kMost),
                                               __builtin_amdgcn_fmed3f(v[i + 1], -kMost, kMost)}), b2);
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        out[0][i + e] = h[e];
        rest[i + e] = v[i + e] - (float)h[e];
      }
    }
    P more[NP - 1];
    split_parts<NP - 1, N>(rest, more);
#pragma unroll
    for (int p = 1; p < NP; ++p) out[p] = more[p - 1];
  } else {
    split_parts<NP, N>(v, out);
  }
}

// ROWS x W elements in registers on their way to LDS, vectors of 16 bytes: a thread's loads all in flight at
// once, without branches.  Rows and columns that are not there are loaded from where there are some, and
// become zeros when they are put down.
template <typename T, int ROWS, int W>
struct LaTile {
  static constexpr int V = 16 / sizeof(T), PER = W / V, N = ROWS * PER / 256;
  static_assert(ROWS * PER % 256 == 0, "whole vectors a thread");
  uint4 r[N];
  // `p` the same in all lanes; 64 rows are within 2^31 bytes (host check).  A tile that is not a row's first may
  // have fewer columns than a vector: its loads begin in the tile before it, offsets stay positive.
  __device__ __forceinline__ void load(const T* __restrict__ p, int stride, int rows, int cols) {
    const int back = cols < V ? V - cols : 0, row0 = threadIdx.x / PER, c = threadIdx.x % PER * V;
    const uint32_t col = (uint32_t)((c + V <= cols ? c : cols - V) + back);
    constexpr int STEP = 256 / PER;  // rows from one vector of a thread to its next
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // row0 + i STEP, or the last row
      const int row = row0 < rows - 1 - i * STEP ? row0 : rows - 1 - i * STEP;
      const uint32_t off = ((uint32_t)(row + i * STEP) * (uint32_t)stride + col) * (uint32_t)sizeof(T);
      __builtin_memcpy(&r[i], reinterpret_cast<const char*>(p - back) + (size_t)off, 16);  // element alignment only
    }
  }
  // NaN or not zero where one of a vector's elements is not finite
  static __device__ __forceinline__ float spoilt_by(uint4 v) {
    float z = 0.f;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        z = fmaf(__uint_as_float(w[j]), 0.f, z);
      } else if constexpr (__is_same(T, __bf16)) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        z = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, w[j]), b2{0, 0}, z, false);
      } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        z = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, w[j]), h2{0, 0}, z, false);
      }
    }
    return z;
  }
  // as bf16 parts, `pitch` elements from row to row.  GUARD: a zero of the triangular factor times a NaN or an
  // infinity is NaN and would carry it to the tokens before its own, so such elements become zeros
  // here; `bad` learns of each column's first one (at `from` + row), and *spoilt that there is any.
  template <int NP, bool GUARD = false>
  __device__ __forceinline__ void put(__bf16* lds, int pitch, int part, int rows, int cols, int from = 0, int* bad = nullptr,
                                      int* spoilt = nullptr) {
    const int row0 = threadIdx.x / PER, c = threadIdx.x % PER * V;
    constexpr int STEP = 256 / PER;
    if (rows < ROWS || cols < W) {  // (no branch for each lane where all is there)
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int past = c + V - cols;
        if (past > 0) {
          unsigned __int128 u = __builtin_bit_cast(unsigned __int128, r[i]);
          u = past < V ? u >> (past * (int)sizeof(T) * 8) : 0;
          r[i] = __builtin_bit_cast(uint4, u);
        }
        if (row0 + i * STEP >= rows) r[i] = make_uint4(0, 0, 0, 0);
      }
    }
    if constexpr (GUARD) {
      float z = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) z += spoilt_by(r[i]);
      if (__any(z != 0.f)) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          T e[V];
          __builtin_memcpy(e, &r[i], 16);
#pragma unroll
          for (int j = 0; j < V; ++j) {
            if (to_f32(e[j]) * 0.f != 0.f) {
              atomicMin(&bad[c + j], from + row0 + i * STEP);
              *spoilt = 1;
              e[j] = from_f32<T>(0.f);
            }
          }
          __builtin_memcpy(&r[i], e, 16);
        }
      }
    }
    __bf16* const to = lds + row0 * pitch + c;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (NP == 1) {
        *reinterpret_cast<uint4*>(to + i * STEP * pitch) = r[i];
      } else {
        T e[V];
        float f[V];
        typedef __bf16 part_t __attribute__((ext_vector_type(V)));
        part_t parts[NP];
        __builtin_memcpy(e, &r[i], 16);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = to_f32(e[j]);
        la_parts<NP, V, sizeof(T) == 4>(f, parts);
#pragma unroll
        for (int q = 0; q < NP; ++q) __builtin_memcpy(to + i * STEP * pitch + q * part, &parts[q], V * 2);
      }
    }
  }
};

// 8 of 32 columns of a staged row, in gdr_at's order
__device__ __forceinline__ uint4 la_row(const __bf16* p, int g) {
  const uint2 lo = *reinterpret_cast<const uint2*>(p + 4 * g), hi = *reinterpret_cast<const uint2*>(p + 16 + 4 * g);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}
// 8 of 32 staged rows (tokens) of a column, in gdr_at's order: 16 lanes read four rows of four times four
// columns, JUMP columns apart, and each gets a column of them.
template <int JUMP = 4>
__device__ __forceinline__ uint4 la_col(const __bf16* p, int pitch, int lane) {
  typedef __attribute__((address_space(3))) s16x4 lds_t;
  const __bf16* at = p + (4 * (lane >> 4) + ((lane >> 2) & 3)) * pitch + JUMP * (lane & 3);
  const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(at));
  const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t*)(at + 16 * pitch));
  const uint2 x = __builtin_bit_cast(uint2, lo), y = __builtin_bit_cast(uint2, hi);
  return make_uint4(x.x, x.y, y.x, y.y);
}
// The wave's column of c and S that lane index c of tile x has: with two tiles a lane that holds rows 4 g .. of
// both as results has 8 columns in a row.
template <int NT>
__device__ __forceinline__ int la_at(int c, int x) { return NT == 2 ? 8 * (c >> 2) + 4 * x + (c & 3) : c; }
__device__ __forceinline__ float la_bf(uint32_t pair, int i) { return __uint_as_float(i ? pair & 0xffff0000u : pair << 16); }
// the 8 values that a fragment's parts stand for
template <int NP>
__device__ __forceinline__ void la_values(const uint4 (&f)[NP], float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = 0.f;
#pragma unroll
    for (int p = NP - 1; p >= 0; --p) {
      const uint32_t w[4] = {f[p].x, f[p].y, f[p].z, f[p].w};
      v[i] += la_bf(w[i / 2], i & 1);
    }
  }
}
template <int NP, bool WIDE>
__device__ __forceinline__ void la_split(const float (&v)[8], uint4 (&f)[NP]) {
  bf16x8 parts[NP];
  la_parts<NP, 8, WIDE>(v, parts);
#pragma unroll
  for (int p = 0; p < NP; ++p) f[p] = __builtin_bit_cast(uint4, parts[p]);
}

// M x N accumulators, from M first and N second operands: none waits for the one before it.
template <int M, int N, int NA, int NB>
__device__ __forceinline__ void la_mma(const uint4 (&a)[M][NA], const uint4 (&b)[N][NB], f32x4 (&c)[M][N]) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int p = 0; p < NA; ++p)
#pragma unroll
      for (int q = 0; q < NB; ++q)
        if (p + q == s) {
#pragma unroll
          for (int m = 0; m < M; ++m)
#pragma unroll
            for (int n = 0; n < N; ++n) c[m][n] = mma(a[m][p], b[n][q], c[m][n]);
        }
}

// A chunk's decays, by one wave: G / ln 2 in two floats, exp(G), exp(G_last - G), exp(G_last).
template <int CT>
struct LaDecays {
  float2 gd[CT];
  float grown[CT], rest[CT];
  float all, pad[3];
  __device__ __forceinline__ void put(float g, int lane, int rows) {
    float2 last;
    // below -120 the decay is 0 in fp32 whatever follows, and sums with -inf have no differences
    const float v = lane < rows ? g : 0.f;
    const float2 s = la_running(v < -120.f ? -120.f : v, &last);
    if (lane < CT) {
      gd[lane] = s;
      grown[lane] = gdr_decay(s, make_float2(0.f, 0.f));
      rest[lane] = gdr_decay(last, s);
    }
    if (lane == 0) all = gdr_decay(last, make_float2(0.f, 0.f));
  }
};

// Where S (or another matrix of its layout) has element (16 t + 4 g + e, la_at(c, x)) of a tile: f(t, x, e, whether
// it is there, its address, or another element's where it is not).  No branch around what f loads.  (A state has
// fewer than 2^29 elements: host check.)
template <int RT, int NT, bool SWAP, typename P, typename F>
__device__ __forceinline__ void la_each(const LaArgs& a, const LaRole& r, int i0, int col, int c, int g, P* p, F f) {
  const int si = SWAP ? 1 : a.V, sj = SWAP ? a.V : 1;
#pragma unroll
  for (int x = 0; x < NT; ++x) {
    const int j = col + la_at<NT>(c, x);
    const uint32_t at = (uint32_t)((j < r.CD ? j : 0) * sj);
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int i = i0 + 16 * t + 4 * g + e;
        f(t, x, e, i < r.AD && j < r.CD, p + (at + (uint32_t)((i < r.AD ? i : 0) * si)));
      }
  }
}
// full: the tile has no rows or columns past the state's.  `col`: the wave's first column.
template <int RT, int NT, bool SWAP>
__device__ __forceinline__ void la_load(const LaArgs& a, const LaRole& r, bool full, int i0, int col, int c, int g, const float* from,
                                        f32x4 (&S)[RT][NT]) {
  if (full && (!SWAP || a.V % 4 == 0)) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      const int j = col + la_at<NT>(c, x);
      const float* __restrict__ at = from + (SWAP ? (uint32_t)(j * a.V + i0 + 4 * g) : (uint32_t)(4 * g * a.V + j));
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        if constexpr (SWAP) {
          __builtin_memcpy(&S[t][x], at + 16 * t, 16);  // (a state may begin at any element)
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) S[t][x][e] = at[(uint32_t)((16 * t + e) * a.V)];
        }
      }
    }
  } else {
    la_each<RT, NT, SWAP>(a, r, i0, col, c, g, from, [&](int t, int x, int e, bool in, const float* p) {
      const float v = *p;
      S[t][x][e] = in ? v : 0.f;
    });
  }
}
template <int RT, int NT>
__device__ __forceinline__ void la_store(const LaArgs& a, const LaRole& r, bool full, int col, int c, int g, float* to,
                                         const f32x4 (&S)[RT][NT]) {
  if (full) {
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      float* __restrict__ at = to + (uint32_t)(4 * g * a.V + col + la_at<NT>(c, x));
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) at[(uint32_t)((16 * t + e) * a.V)] = S[t][x][e];
    }
  } else {
    la_each<RT, NT, false>(a, r, 0, col, c, g, to, [&](int t, int x, int e, bool in, float* p) { if (in) *p = S[t][x][e]; });
  }
}
// S after a chunk (in reverse: before it): S all + B^T (C f), 32 staged tokens at a time
template <int RT, int NT, int HS, int NP>
__device__ __forceinline__ void la_update(const __bf16* b, int b_pitch, int b_part, const __bf16* c, int c_pitch, int c_part, const float* f,
                                          float factor, float all, int lane, f32x4 (&S)[RT][NT]) {
  const int g = lane >> 4;
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int x = 0; x < NT; ++x) S[t][x] *= all;
#pragma unroll
  for (int s = 0; s < HS; ++s) {
    uint4 cw[NT][kLaOut];
    f32x4 w[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) w[u] = *reinterpret_cast<const f32x4*>(f + 32 * s + 16 * u + 4 * g) * factor;
#pragma unroll
    for (int x = 0; x < NT; ++x) {
      uint4 cf[NP];
      float v[8];
#pragma unroll
      for (int p = 0; p < NP; ++p) cf[p] = la_col<4 * NT>(c + p * c_part + 32 * s * c_pitch + 4 * x, c_pitch, lane);
      la_values<NP>(cf, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] *= w[e / 4][e & 3];
      la_split<kLaOut, NP == 3>(v, cw[x]);
    }
#pragma unroll
    for (int t = 0; t < RT; t += 4) {
      uint4 bf[4][NP];
      f32x4 y[4][NT];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
#pragma unroll
        for (int p = 0; p < NP; ++p) bf[u][p] = la_col(b + p * b_part + 32 * s * b_pitch + 16 * (t + u), b_pitch, lane);
#pragma unroll
        for (int x = 0; x < NT; ++x) y[u][x] = S[t + u][x];
      }
      la_mma<4, NT, NP, kLaOut>(bf, cw, y);
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int x = 0; x < NT; ++x) S[t + u][x] = y[u][x];
    }
  }
}

template <typename T, int DA, int NT, bool DOTS>
struct LaLds {
  static constexpr int NP = kParts<T>, CT = kLaC<T, DA>, W = 64 * NT, PA = DA + 8, PC = W + 8;
  static constexpr int PF = CT == 64 ? kTri : 2;
  __bf16 a[NP][CT][PA];
  __bf16 b[NP][CT][PA];
  __bf16 c[NP][CT][PC];
  uint4 p[PF][kLaOut][64];
  LaDecays<CT> d;
  float self[DOTS ? CT : 1];  // each token's product with itself, scaled: P's diagonal
  union {
    float dots[DOTS ? 4 : 1][CT];
    int bad[W];  // (forward) each column's first token whose c is not finite
  };
  int spoilt;
};

// the first n of N values, one at a time
template <int N, typename T>
__device__ __forceinline__ void la_tail(T* to, const float* v, int n) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) to[i] = from_f32<T>(v[i]);
  asm volatile("");  // (else the last store is shared with the whole vector's, which is then split)
}

// The outputs of one segment, and its last state.  Products that make outputs are taken transposed, so that a
// lane has 4 NT columns of one token.  (Gradients, 2 x 2048 tokens of 16 heads of 128 x 128: dq, dk and dv 88 us.)
// DOTS: a token's term with itself has no decay, so it is no part of a decay's gradient.  It is in q . dq and in
// k . dk alike, and 2^-24 of it would stay of their difference, where exp(g) leaves less of that.  So the dots
// are taken before it is added, of the triangle without its diagonal; and of what the state at the segment's
// end and the gradient of it have in common, without the last token's own term, the one without a decay there.
template <typename T, int DA, int NT, int MODE, bool DOTS>
__device__ __forceinline__ void la_segment(const LaArgs& a, const LaRole& r, const LaGrid& gr, char* lds) {
  using Lds = LaLds<T, DA, NT, DOTS>;
  constexpr int NP = Lds::NP, CT = Lds::CT, W = Lds::W, RT = DA / 16, KS = DA / 32, MT = CT / 16, HS = CT / 32;
  constexpr int OP = kLaOut, OW = 4 * NT;
  constexpr bool rev = la_reverse(MODE), swapped = la_swapped(MODE);
  Lds& L = *reinterpret_cast<Lds*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile, h, slot;
  if (!la_place(a, gr, &tile, &h, &slot)) return;
  const int hk = h / a.group, c_tiles = (r.CD + W - 1) / W, c_tile = swapped ? tile % c_tiles : tile, a_tile = swapped ? tile / c_tiles : 0;
  const int a0 = a_tile * DA, col0 = c_tile * W, col = col0 + wave * 16 * NT;
  const int acols = r.AD - a0 < DA ? r.AD - a0 : DA, ccols = r.CD - col0 < W ? r.CD - col0 : W;
  const bool full = acols == DA && ccols == W;
  const int ha = swapped ? h : hk, hc = swapped ? hk : h;
  if (a_tile == 0)
    la_outside(a, slot, [&](int64_t from, int64_t to) {
      for (int64_t t = from + tid / 64; t < to; t += 4)
        for (int j = lane; j < ccols; j += 64) {
          if (swapped && r.parts) {
            for (int q = 0; q < r.a_tiles; ++q)
              r.parts[((((int64_t)(h % a.group) * r.a_tiles + q) * a.B * a.T + t) * a.Hk + hk) * r.CD + col0 + j] = 0.f;
          } else {
            static_cast<T*>(r.out)[(t * (swapped ? a.Hk : a.Hv) + hc) * r.CD + col0 + j] = from_f32<T>(0.f);
          }
        }
    });
  const int n = la_seq_of_slot(a, slot);
  const LaSeq seq = la_seq(a, n);
  const int z = slot - seq.slot;
  if (z < 0 || z >= seq.segs) return;
  const int t0 = z * a.seg, len = seq.len - t0 < a.seg ? seq.len - t0 : a.seg;  // tokens of this segment
  const int chunks = (len + CT - 1) / CT;
  const int64_t first = seq.begin + t0;
  const T* __restrict__ pa = static_cast<const T*>(r.a) + seq.batch * r.a_s[0] + first * r.a_s[1] + ha * r.a_s[2] + a0;
  const T* __restrict__ pb = static_cast<const T*>(r.b) + seq.batch * r.b_s[0] + first * r.b_s[1] + ha * r.b_s[2] + a0;
  const T* __restrict__ pc = static_cast<const T*>(r.c) + seq.batch * r.c_s[0] + first * r.c_s[1] + hc * r.c_s[2] + col0;
  const int64_t pg = seq.batch * a.g_s[0] + first * a.g_s[1] + h * a.g_s[2];
  // a lane's columns of a result, and of e's rows where they are all there
  const int oc = wave * 16 * NT + OW * g;
  const bool whole = col0 + oc + OW <= r.CD;
  const T* __restrict__ pe = DOTS ? static_cast<const T*>(r.e) + seq.batch * r.e_s[0] + first * r.e_s[1] + hk * r.e_s[2] + (whole ? col0 + oc : 0) : nullptr;

  LaTile<T, CT, DA> ta, tb;
  LaTile<T, CT, W> tc;
  GdrGate tg;
  auto load = [&](int ch) {
    const int at = ch * CT, rows = len - at < CT ? len - at : CT;
    ta.load(pa + at * r.a_s[1], (int)r.a_s[1], rows, acols);
    tb.load(pb + at * r.b_s[1], (int)r.b_s[1], rows, acols);
    tc.load(pc + at * r.c_s[1], (int)r.c_s[1], rows, ccols);
    tg = gdr_gate_load(a.g, a.g_dtype, pg + (at + (lane < rows ? lane : 0)) * a.g_s[1]);
  };
  if (chunks > 0) load(rev ? chunks - 1 : 0);
  f32x4 S[RT][NT];
  const float* from = (rev ? z == seq.segs - 1 : z == 0) ? r.s_first : r.s_between;
  bool have = from != nullptr;
  if (have) {
    const int64_t at = (int64_t)((rev ? z == seq.segs - 1 : z == 0) ? n : seq.end + z - (rev ? 0 : 1)) * a.Hv + h;
    la_load<RT, NT, swapped>(a, r, full, a0, col, c, g, from + at * a.K * a.V, S);
  } else {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int x = 0; x < NT; ++x) S[t][x] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if constexpr (MODE == kLaFwd) {
    for (int i = tid; i < W; i += 256) L.bad[i] = INT_MAX;
    if (tid == 0) L.spoilt = 0;
    __syncthreads();
  }
  for (int k = 0; k < chunks; ++k) {
    const int ch = rev ? chunks - 1 - k : k, at = ch * CT, rows = len - at < CT ? len - at : CT;
    ta.template put<NP>(&L.a[0][0][0], Lds::PA, CT * Lds::PA, rows, acols);
    tb.template put<NP>(&L.b[0][0][0], Lds::PA, CT * Lds::PA, rows, acols);
    tc.template put<NP, MODE == kLaFwd>(&L.c[0][0][0], Lds::PC, CT * Lds::PC, rows, ccols, at, L.bad, &L.spoilt);
    if (wave == 3) {
      L.d.put(gdr_gate<T>(tg, a.g_dtype), lane, rows);
      // (here S is read once more, for that inner product)
      if (DOTS && MODE == kLaDq && k + 1 == chunks && lane == rows - 1) L.d.rest[lane] = 0.f;
    }
    __syncthreads();
    // scale lower(A B^T * D), or upper in reverse, as the results of its transpose: a lane has 8 of 32 columns
    // of a row, one fragment.  The fragments within the triangle are shared out to the waves.
#pragma unroll
    for (int f0 = 0; f0 < Lds::PF; f0 += 4) {
      const int f = f0 + wave;
      if (f >= Lds::PF) continue;
      int m = f, s = 0;  // row tile, half of the columns
      if constexpr (HS > 1) {
        m = rev ? (f < 4 ? f >> 1 : f - 2) : f < 2 ? f : 1 + (f >> 1);
        s = rev ? (f < 4 ? f & 1 : 1) : f < 2 ? 0 : f & 1;
      }
      f32x4 y[2][1] = {{f32x4{0.f, 0.f, 0.f, 0.f}}, {f32x4{0.f, 0.f, 0.f, 0.f}}};
      constexpr int Q = KS * NP <= 4 ? KS : 1;  // products whose operands are on their way together
#pragma unroll
      for (int q0 = 0; q0 < KS; q0 += Q) {
        uint4 bf[Q][2][NP], af[Q][1][NP];
#pragma unroll
        for (int q = 0; q < Q; ++q)
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            af[q][0][p] = la_row(&L.a[p][16 * m + c][32 * (q0 + q)], g);
            bf[q][0][p] = la_row(&L.b[p][32 * s + c][32 * (q0 + q)], g);
            bf[q][1][p] = la_row(&L.b[p][32 * s + 16 + c][32 * (q0 + q)], g);
          }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int q = 0; q < Q; ++q) la_mma<2, 1, NP, NP>(bf[q], af[q], y);
      }
      const int out = 16 * m + c;
      const float2 go = L.d.gd[out];
      float v[8], self = 0.f;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        float4 gi[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) gi[e] = *reinterpret_cast<const float4*>(&L.d.gd[32 * s + 16 * u + 4 * g + 2 * e]);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 i = e & 1 ? make_float2(gi[e / 2].z, gi[e / 2].w) : make_float2(gi[e / 2].x, gi[e / 2].y);
          float p = y[u][0][e] * gdr_decay(rev ? i : go, rev ? go : i) * a.scale;
          asm("" : "+v"(p));  // (else a branch for each)
          const int in = 32 * s + 16 * u + 4 * g + e;
          if (DOTS) self = in == out ? p : self;
          v[4 * u + e] = (DOTS ? rev ? in > out : in < out : rev ? in >= out : in <= out) ? p : 0.f;
        }
      }
      if (DOTS && s == m >> 1 && g == c >> 2) L.self[out] = self;
      uint4 w[OP];
      la_split<OP, sizeof(T) == 4>(v, w);
#pragma unroll
      for (int p = 0; p < OP; ++p) L.p[f][p][lane] = w[p];
    }
    __syncthreads();
    f32x4 acc[NT][MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int x = 0; x < NT; ++x) acc[x][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (have) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 sf[NT][OP], af[MT][NP];
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int p = 0; p < NP; ++p) af[m][p] = la_row(&L.a[p][16 * m + c][32 * s], g);
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          float v[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) v[e] = S[2 * s + e / 4][x][e & 3];
          la_split<OP, sizeof(T) == 4>(v, sf[x]);
        }
        la_mma<NT, MT, OP, NP>(sf, af, acc);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        const float f = rev ? L.d.rest[16 * m + c] : L.d.grown[16 * m + c] * a.scale;
#pragma unroll
        for (int x = 0; x < NT; ++x) acc[x][m] *= f;
      }
    }
#pragma unroll
    for (int s = 0; s < HS; ++s) {
      uint4 cf[NT][NP], pf[MT][OP];
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int p = 0; p < NP; ++p) cf[x][p] = la_col<4 * NT>(&L.c[p][32 * s][wave * 16 * NT + 4 * x], Lds::PC, lane);
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        if (HS > 1 && (rev ? s < m >> 1 : s > m >> 1)) continue;
        const int f = HS == 1 ? m : rev ? tri_upper(m, s) : tri_lower(m, s);
#pragma unroll
        for (int p = 0; p < OP; ++p) pf[m][p] = L.p[f][p][lane];
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int z = 2; z >= 0; --z)
#pragma unroll
        for (int p = 0; p < NP; ++p)
#pragma unroll
          for (int q = 0; q < OP; ++q)
            if (p + q == z) {
#pragma unroll
              for (int m = 0; m < MT; ++m) {
                if (HS > 1 && (rev ? s < m >> 1 : s > m >> 1)) continue;
#pragma unroll
                for (int x = 0; x < NT; ++x) acc[x][m] = mma(cf[x][p], pf[m][q], acc[x][m]);
              }
            }
    }
    T ev[DOTS ? MT : 1][OW];
    if constexpr (DOTS) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
        __builtin_memcpy(ev[m], pe + (at + (16 * m + c < rows ? 16 * m + c : 0)) * r.e_s[1], OW * sizeof(T));
    }
    if constexpr (MODE == kLaFwd) {
      if (L.spoilt) {  // outputs from a column's first c on that is not finite are not either
#pragma unroll
        for (int x = 0; x < NT; ++x)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int bad = L.bad[oc + 4 * x + e];
#pragma unroll
            for (int m = 0; m < MT; ++m) acc[x][m][e] = at + 16 * m + c >= bad ? gdr_nan() : acc[x][m][e];
          }
      }
    }
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      const int row = 16 * m + c;
      float o[OW];
#pragma unroll
      for (int x = 0; x < NT; ++x)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[4 * x + e] = acc[x][m][e];
      if constexpr (DOTS) {
        float dot = 0.f;
        if (whole) {
#pragma unroll
          for (int q = 0; q < OW; ++q) dot += o[q] * to_f32(ev[m][q]);
        } else if (row < rows) {
          const T* __restrict__ e = pe + (at + row) * r.e_s[1];
#pragma unroll
          for (int q = 0; q < OW; ++q) {
            const int j = col0 + oc + q;
            dot += j < r.CD ? o[q] * to_f32(e[j < r.CD ? j : 0]) : 0.f;
          }
        }
        dot += __shfl_xor(dot, 16, 64);
        dot += __shfl_xor(dot, 32, 64);
        // (of the segment's last token k . dk has nothing but that term)
        if (g == 0) L.dots[wave][row] = MODE == kLaDk && k == 0 && row == rows - 1 ? 0.f : dot;
        const float self = L.self[row];
        uint4 cw[NP];
        float own[8];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          cw[p] = make_uint4(0, 0, 0, 0);
          __builtin_memcpy(&cw[p], __builtin_assume_aligned(&L.c[p][row][oc], 2 * OW), 2 * OW);
        }
        la_values<NP>(cw, own);
#pragma unroll
        for (int q = 0; q < OW; ++q) o[q] = fmaf(self, own[q], o[q]);
      }
      if (row < rows) {
        const int64_t tok = seq.batch * a.T + first + at + row;
        if (swapped && r.parts) {
          float* __restrict__ to = r.parts + ((((int64_t)(h % a.group) * r.a_tiles + a_tile) * a.B * a.T + tok) * a.Hk + hk) * r.CD + col0 + oc;
          if (whole) __builtin_memcpy(to, o, OW * 4);
          else la_tail<OW>(to, o, r.CD - col0 - oc);
        } else {
          T* __restrict__ to = static_cast<T*>(r.out) + (tok * (swapped ? a.Hk : a.Hv) + hc) * r.CD + col0 + oc;
          T v[OW];
#pragma unroll
          for (int q = 0; q < OW; ++q) v[q] = from_f32<T>(o[q]);
          if (whole) __builtin_memcpy(to, v, OW * sizeof(T));
          else la_tail<OW>(to, o, r.CD - col0 - oc);
        }
      }
    }
    // here the outputs' registers are free (at the end the last chunk's again)
    load(k + 1 < chunks ? (rev ? ch - 1 : ch + 1) : ch);
    la_update<RT, NT, HS, NP>(&L.b[0][0][0], Lds::PA, CT * Lds::PA, &L.c[0][0][wave * 16 * NT], Lds::PC, CT * Lds::PC,
                              rev ? L.d.grown : L.d.rest, rev ? a.scale : 1.f, L.d.all, lane, S);
    have = true;
    __syncthreads();  // the chunk's LDS is free
    if constexpr (DOTS) {
      if (tid < rows)
        r.dots[((int64_t)tile * a.Hv + h) * a.B * a.T + seq.batch * a.T + first + at + tid] =
            (L.dots[0][tid] + L.dots[1][tid]) + (L.dots[2][tid] + L.dots[3][tid]);
    }
  }
  if (!swapped && r.s_last && (rev ? z == 0 : z == seq.segs - 1)) {
    if constexpr (MODE == kLaFwd) {
      if (L.spoilt) {
#pragma unroll
        for (int x = 0; x < NT; ++x) {
          const bool bad = L.bad[wave * 16 * NT + la_at<NT>(c, x)] != INT_MAX;
#pragma unroll
          for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) S[t][x][e] = bad ? gdr_nan() : S[t][x][e];
        }
      }
    }
    la_store<RT, NT>(a, r, full, col, c, g, r.s_last + ((int64_t)n * a.Hv + h) * a.K * a.V, S);
  }
  if constexpr (DOTS) {
    if (MODE == kLaDq) {  // the state at the segment's end, and the gradient of it from what follows
      float x = 0.f;
      const float* d = z == seq.segs - 1 ? r.x_last : r.x_between;
      if (d) {
        f32x4 D[RT][NT];
        la_load<RT, NT, true>(a, r, full, a0, col, c, g, d + ((int64_t)(z == seq.segs - 1 ? n : seq.end + z) * a.Hv + h) * a.K * a.V, D);
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int y = 0; y < NT; ++y)
#pragma unroll
            for (int e = 0; e < 4; ++e) x += S[t][y][e] * D[t][y][e];
      }
      x = wave_sum(x);
      __syncthreads();
      if (lane == 0) L.dots[wave][0] = x;
      __syncthreads();
      if (tid == 0)
        r.x_out[((int64_t)tile * a.slots + slot) * a.Hv + h] = (L.dots[0][0] + L.dots[1][0]) + (L.dots[2][0] + L.dots[3][0]);
    }
  }
}

// Waves of a SIMD that a kernel is compiled for: two workgroups share a CU where their LDS lets them.
template <typename Lds> inline constexpr int kLaWaves = 2 * sizeof(Lds) <= 163840 ? 2 : 1;

template <typename T, int DA, int NT, int MODE>
__global__ __launch_bounds__(256, (kLaWaves<LaLds<T, DA, NT, false>>)) void la_out_kernel(LaArgs a, LaGrid gr) {
  __shared__ __align__(16) char lds[sizeof(LaLds<T, DA, NT, false>)];
  la_segment<T, DA, NT, MODE, false>(a, a.role[0], gr, lds);
}
// dq, dk and, where its tiles are as many, dv: a row of workgroups each.
template <typename T, int DA, int NT, bool DOTS>
__global__ __launch_bounds__(256, (kLaWaves<LaLds<T, DA, NT, DOTS>>)) void la_grads_kernel(LaArgs a, LaGrid gr) {
  __shared__ __align__(16) char lds[sizeof(LaLds<T, DA, NT, DOTS>)];
  if (blockIdx.y == 0) la_segment<T, DA, NT, kLaDq, DOTS>(a, a.role[0], gr, lds);
  else if (blockIdx.y == 1) la_segment<T, DA, NT, kLaDk, DOTS>(a, a.role[1], gr, lds);
  else la_segment<T, DA, NT, kLaDv, false>(a, a.role[2], gr, lds);
}

template <typename T, int DA>
struct LaStateLds {
  static constexpr int NP = kParts<T>, CT = kLaC<T, DA>, W = 64, PA = DA + 8, PC = W + 8;
  __bf16 b[NP][CT][PA];
  __bf16 c[NP][CT][PC];
  LaDecays<CT> d;
};

// (64 columns a workgroup, also where there are more: it is bound by loads on their way, and twice as many
// workgroups have more of them: 4 % off a call of 8192 tokens of 32 heads of 128 x 128.)
// What a segment adds to the state, and its decay: b and c alone.  The last segment's (in reverse the
// first's) nobody asks for.
template <typename T, int DA, bool rev>
__device__ __forceinline__ void la_state(const LaArgs& a, const LaRole& r, const LaGrid& gr, char* lds, float* to, float* decays) {
  using Lds = LaStateLds<T, DA>;
  constexpr int NP = Lds::NP, CT = Lds::CT, W = Lds::W, RT = DA / 16, NT = 1, HS = CT / 32;
  Lds& L = *reinterpret_cast<Lds*>(lds);
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile, h, slot;
  if (!la_place(a, gr, &tile, &h, &slot)) return;
  const int hk = h / a.group;
  int n, z;
  LaSeq seq;
  if (a.cu) {
    if (!la_segment_at(a, slot, &n, &seq, &z)) return;
  } else {
    n = la_seq_of_slot(a, slot);
    seq = la_seq(a, n);
    z = slot - seq.slot;
  }
  if (z == seq.segs - 1) return;
  const int64_t end = (int64_t)(seq.end + z) * a.Hv + h;
  z += rev;
  const int t0 = z * a.seg, len = seq.len - t0 < a.seg ? seq.len - t0 : a.seg, chunks = (len + CT - 1) / CT;
  const int col0 = tile * W, col = col0 + wave * 16 * NT;
  const int acols = r.AD, ccols = r.CD - col0 < W ? r.CD - col0 : W;
  const int64_t first = seq.begin + t0;
  const T* __restrict__ pb = static_cast<const T*>(r.b) + seq.batch * r.b_s[0] + first * r.b_s[1] + hk * r.b_s[2];
  const T* __restrict__ pc = static_cast<const T*>(r.c) + seq.batch * r.c_s[0] + first * r.c_s[1] + h * r.c_s[2] + col0;
  const int64_t pg = seq.batch * a.g_s[0] + first * a.g_s[1] + h * a.g_s[2];
  f32x4 S[RT][NT];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int x = 0; x < NT; ++x) S[t][x] = f32x4{0.f, 0.f, 0.f, 0.f};
  float2 total = make_float2(0.f, 0.f);
  LaTile<T, CT, DA> tb;
  LaTile<T, CT, W> tc;
  GdrGate tg;
  auto load = [&](int ch) {
    const int at = ch * CT, rows = len - at < CT ? len - at : CT;
    tb.load(pb + at * r.b_s[1], (int)r.b_s[1], rows, acols);
    tc.load(pc + at * r.c_s[1], (int)r.c_s[1], rows, ccols);
    tg = gdr_gate_load(a.g, a.g_dtype, pg + (at + (lane < rows ? lane : 0)) * a.g_s[1]);
  };
  load(rev ? chunks - 1 : 0);
  for (int k = 0; k < chunks; ++k) {
    const int ch = rev ? chunks - 1 - k : k, at = ch * CT, rows = len - at < CT ? len - at : CT;
    tb.template put<NP>(&L.b[0][0][0], Lds::PA, CT * Lds::PA, rows, acols);
    tc.template put<NP>(&L.c[0][0][0], Lds::PC, CT * Lds::PC, rows, ccols);
    if (wave == 3) L.d.put(gdr_gate<T>(tg, a.g_dtype), lane, rows);
    __syncthreads();
    load(k + 1 < chunks ? (rev ? ch - 1 : ch + 1) : ch);
    const float2 last = L.d.gd[CT - 1];
    total.x += last.x;
    total.y += last.y;
    la_update<RT, NT, HS, NP>(&L.b[0][0][0], Lds::PA, CT * Lds::PA, &L.c[0][0][wave * 16 * NT], Lds::PC, CT * Lds::PC,
                              rev ? L.d.grown : L.d.rest, rev ? a.scale : 1.f, L.d.all, lane, S);
    __syncthreads();
  }
  la_store<RT, NT>(a, r, acols == DA && ccols == W, col, c, g, to + end * a.K * a.V, S);
  if (tile == 0 && tid == 0) decays[end] = gdr_decay(total, make_float2(0.f, 0.f));
}
// Roles 0 and, where there is a second row of workgroups, 1 in reverse.
template <typename T, int DA>
__global__ __launch_bounds__(256, 2) void la_state_kernel(LaArgs a, LaGrid gr, float* to0, float* to1, float* decays) {
  __shared__ __align__(16) char lds[sizeof(LaStateLds<T, DA>)];
  if (blockIdx.y == 0) la_state<T, DA, false>(a, a.role[0], gr, lds, to0, decays);
  else la_state<T, DA, true>(a, a.role[1], gr, lds, to1, decays + (int64_t)a.ends * a.Hv);
}

// launch(grid, its place) for workgroups of all tiles, heads and segments, in as many launches as it takes
template <typename F>
int la_launches(const LaArgs& a, int slots, int64_t tiles, const char* what, F launch) {
  const int64_t per = tiles * a.group, units = ((int64_t)slots * a.Hk + 7) / 8 * 8;
  if (per > kLaBlocks / 8) return fail(ATK_UNSUPPORTED, "linear attention: too many value heads and columns of a key head");
  const int64_t most = kLaBlocks / 8 / per * 8;
  for (int64_t u = 0; u < units; u += most) {
    launch((unsigned)((units - u < most ? units - u : most) * per),
           LaGrid{make_fastdiv((uint32_t)per), make_fastdiv((uint32_t)tiles), (int)u, slots});
    if (int rc = check_launch(what)) return rc;
  }
  return ATK_OK;
}
template <typename T, int DA, int NT, int MODE>
int la_run_out(const LaArgs& a, hipStream_t s) {
  return la_launches(a, a.slots, (a.role[0].CD + 64 * NT - 1) / (64 * NT), "la_out_kernel", [&](unsigned n, LaGrid g) {
    hipLaunchKernelGGL((la_out_kernel<T, DA, NT, MODE>), dim3(n), dim3(256), 0, s, a, g);
  });
}
template <typename T, int DA, int NT>
int la_run_grads(const LaArgs& a, bool dots, unsigned roles, hipStream_t s) {
  const LaRole& r = a.role[0];
  return la_launches(a, a.slots, (int64_t)((r.CD + 64 * NT - 1) / (64 * NT)) * r.a_tiles, "la_grads_kernel", [&](unsigned n, LaGrid g) {
    if (dots) hipLaunchKernelGGL((la_grads_kernel<T, DA, NT, true>), dim3(n, roles), dim3(256), 0, s, a, g);
    else hipLaunchKernelGGL((la_grads_kernel<T, DA, NT, false>), dim3(n, roles), dim3(256), 0, s, a, g);
  });
}
template <typename T, int DA>
int la_run_states(const LaArgs& a, int roles, float* const* to, float* decays, hipStream_t s) {
  return la_launches(a, a.ends, (a.V + 63) / 64, "la_state_kernel", [&](unsigned n, LaGrid g) {
    hipLaunchKernelGGL((la_state_kernel<T, DA>), dim3(n, (unsigned)roles), dim3(256), 0, s, a, g, to[0], roles > 1 ? to[1] : nullptr, decays);
  });
}

}  // namespace

#define ATK_LA_TILED(DA, NT, FN)                                                        \
  [&]() {                                                                              \
    if (NT == 2) return DA == 128 ? FN(128, 2) : FN(64, 2);                            \
    return DA == 256 ? FN(256, 1) : DA == 128 ? FN(128, 1) : FN(64, 1);                \
  }()
template <typename T>
int la_launch_out(const LaArgs& a, hipStream_t s) {
  const int da = la_padded(a.K), nt = la_wide(a, da, a.V, 1);
#define ATK_LA_OUT(DA, NT) la_run_out<T, DA, NT, kLaFwd>(a, s)
  return ATK_LA_TILED(da, nt, ATK_LA_OUT);
}
template <typename T>
int la_launch_grads(const LaArgs& a, bool dots, hipStream_t s) {
  const int dk = la_padded(a.K), dv = la_padded(a.V), nv = la_wide(a, dk, a.V, 3), nt = la_wide(a, dv, a.K, 3);
  // dv shares the launch where its workgroups are shaped as those of dq and dk, and as many
  const bool one = dk == dv && nv == nt && (a.V + 64 * nt - 1) / (64 * nt) == (a.K + 64 * nt - 1) / (64 * nt) * a.role[0].a_tiles;
  const unsigned roles = one ? 3 : 2;
#define ATK_LA_GRADS(DA, NT) la_run_grads<T, DA, NT>(a, dots, roles, s)
  if (int rc = ATK_LA_TILED(dv, nt, ATK_LA_GRADS)) return rc;
  if (one) return ATK_OK;
  LaArgs b = a;
  b.role[0] = a.role[2];
#define ATK_LA_DV(DA, NT) la_run_out<T, DA, NT, kLaDv>(b, s)
  return ATK_LA_TILED(dk, nv, ATK_LA_DV);
}
template <typename T>
int la_launch_states(const LaArgs& a, int roles, float* const* to, float* decays, hipStream_t s) {
  const int da = la_padded(a.K);
  if (da == 256) return la_run_states<T, 256>(a, roles, to, decays, s);
  return da == 128 ? la_run_states<T, 128>(a, roles, to, decays, s) : la_run_states<T, 64>(a, roles, to, decays, s);
}

}  // namespace atk

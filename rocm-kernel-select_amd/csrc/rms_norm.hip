// Root-mean-square norm over the last axis, with the residual's addition in front and an 8-bit
// output with scales behind, and its backward.
//
//   h = x + residual, rounded to the tensors' type (the residual stream as later layers read it)
//   y = h * rstd * w,  rstd = 1 / sqrt(mean(h^2) + eps)
//   8 bits: scale = max(max|y| / top, 2^-126) over the row or each group of columns,
//           q = round(y / scale) (fp8 e4m3: top 448; int8: top 127)
//   dh = rstd * (w dy - h rstd^2 mean(w dy h)) + dh_in;  dw = sum over rows of dy h rstd
//
// HBM-bound: every input is read and every output written once.  A row stays in registers as fp32
// between its loads and its stores, so the statistics need no second read; sums and maxima are fp32.
// TPR threads share a row, VPT vectors of 16 input bytes each: a quarter wave for a head's 128
// columns (four rows to a wave), one wave up to 2048, a workgroup above.  Measured, bf16, no input in any
// cache: 8192 x 2048 with a residual 25 us for 134 MB, into fp8 by groups of 128 27 to 31 us for 118 MB, the
// backward with dw 32 us for 134 MB; 262144 x 128 23 us for 134 MB, 5.8 TB/s.
#include "row_cols.h"

namespace atk {
namespace {

constexpr int kQNone = 0, kQFp8 = 1, kQInt8 = 2;

struct RmsArgs {
  const void* x; const void* r; const void* w;
  void* y; void* h; float* rstd; float* scales;
  int64_t M, x_stride, r_stride;
  int N, group, groups, w_f32;
  float eps;
};

struct RmsBwdArgs {
  const void* h; const void* dy; const void* dh; const void* w; const float* rstd;
  void* dx; float* dw_part;
  int64_t M, h_stride, dy_stride, dh_stride;
  int N, w_f32;
};

// How many vectors at once: a workgroup of 1024 has 128 registers a thread.
template <int TPR, int VPT>
inline constexpr int kTogether = TPR == 1024 ? 1 : VPT;

// magnitudes v[0..N) each over runs of `lanes` lanes
template <int N>
__device__ __forceinline__ void group_max(float (&v)[N], int lanes) {
#pragma unroll
  for (int j = 0; j < N; ++j) v[j] = lanes_reduce<2>(v[j], Max());
  if (lanes >= 4)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = max_abs(v[j], dpp_mov<0x4E>(v[j]));
  if (lanes >= 8)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = max_abs(v[j], dpp_mov<0x141>(v[j]));
  if (lanes >= 16)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = max_abs(v[j], dpp_mov<0x140>(v[j]));
  if (lanes >= 32)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = max_abs(v[j], __shfl_xor(v[j], 16, 64));
  if (lanes >= 64)
#pragma unroll
    for (int j = 0; j < N; ++j) v[j] = max_abs(v[j], __shfl_xor(v[j], 32, 64));
}

// two values into the low or high half of `old` as fp8 e4m3, nearest even; beyond +-448 saturates,
// NaN stays NaN (fmin / fmax alone would drop it)
__device__ __forceinline__ float clamp_keep_nan(float v, float top) {
  const float c = fminf(fmaxf(v, -top), top);
  return v != v ? v : c;
}
// What 8-bit values of at most `top` are multiplied by; a NaN stays one, so a row or group that holds
// one reads back as NaN in int8 too.
__device__ __forceinline__ float scale_of(float amax, float top) {
  const float s = amax / top;
  return s < 0x1p-126f ? 0x1p-126f : s;
}
template <int Q, int V>
__device__ __forceinline__ void store_q(uint8_t* __restrict__ p, int c, int N, const float* v, float inv) {
  uint32_t d[V / 4];
  if constexpr (Q == kQFp8) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      float s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = clamp_keep_nan(v[i + j] * inv, 448.f);
      int t = __builtin_amdgcn_cvt_pk_fp8_f32(s[0], s[1], 0, false);
      t = __builtin_amdgcn_cvt_pk_fp8_f32(s[2], s[3], t, true);
      d[i / 4] = (uint32_t)t;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      uint32_t t = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int q = (int)rintf(fminf(fmaxf(v[i + j] * inv, -127.f), 127.f));  // NaN -> -127
        t |= (uint32_t)(q & 255) << (8 * j);
      }
      d[i / 4] = t;
    }
  }
  if (c + V <= N) {
    __builtin_memcpy(p + c, d, V);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i < N) p[c + i] = (uint8_t)(d[i / 4] >> (8 * (i & 3)));
  }
}

template <typename T, int Q, int TPR, int VPT, bool RES>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_fwd_kernel(RmsArgs a) {
  constexpr int V = 16 / sizeof(T), NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  constexpr bool TINY = TPR == 8;
  __shared__ float red[2][NT / 64];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR;
  const bool live = row < a.M;  // a dead row takes part in its wave's reductions, and stores nothing
  const T* __restrict__ x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride;
  constexpr int J = kTogether<TPR, VPT>;
  // (opaque where vectors take turns: the compiler would keep all of their addresses in registers)
  const auto lane = [&] {
    int u = t;
    if constexpr (J < VPT) asm volatile("" : "+v"(u));
    return u;
  };
  float f[VPT][V];
  Cols<T, V> wr[J];
#pragma unroll
  for (int j0 = 0; j0 < VPT; j0 += J) {
    const int t = lane();
    Cols<T, V> xr[J], rr[J];
#pragma unroll
    for (int j = 0; j < J; ++j) xr[j] = load_raw<T, V, TINY>(x, (t + (j0 + j) * TPR) * V, a.N);
    if constexpr (RES) {
      const T* __restrict__ r = static_cast<const T*>(a.r) + (live ? row : 0) * a.r_stride;
#pragma unroll
      for (int j = 0; j < J; ++j) rr[j] = load_raw<T, V, TINY>(r, (t + (j0 + j) * TPR) * V, a.N);
    }
    if constexpr (J == VPT) weight_raw<T, V, TINY, TPR>(a.w, a.w_f32, t, 0, a.N, wr);
    loads_issued();
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const int c = (t + (j0 + j) * TPR) * V;
      to_cols<T, V, TINY>(xr[j], c, a.N, f[j0 + j]);
      if constexpr (RES) {
        float g[V];
        to_cols<T, V, TINY>(rr[j], c, a.N, g);
        // the norm is of h as it is stored: one rounding, the stream's own
#pragma unroll
        for (int i = 0; i < V; ++i) f[j0 + j][i] = to_f32(from_f32<T>(f[j0 + j][i] + g[i]));
        if (live) store_cols<T, V>(static_cast<T*>(a.h) + row * a.N, c, a.N, f[j0 + j]);
      }
    }
  }
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) ss += f[j][i] * f[j][i];
  ss = row_reduce<TPR>(ss, red[0], Add());
  const float rstd = rsqrtf(ss / (float)a.N + a.eps);
  if (a.rstd && live && t == 0) a.rstd[row] = rstd;
  #pragma unroll
  for (int j0 = 0; j0 < VPT; j0 += J) {
    const int t = lane();
    float w[J][V];
    if constexpr (J < VPT) weight_raw<T, V, TINY, TPR>(a.w, a.w_f32, t, j0, a.N, wr);
    to_weight<T, V, TINY, TPR>(wr, a.w, a.w_f32, t, j0, a.N, w);
#pragma unroll
    for (int j = 0; j < J; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) f[j0 + j][i] = f[j0 + j][i] * rstd * w[j][i];
  }
  if constexpr (Q == kQNone) {
    T* __restrict__ y = static_cast<T*>(a.y) + row * a.N;
    if (live) {
#pragma unroll
      for (int j = 0; j < VPT; ++j) store_cols<T, V>(y, (lane() + j * TPR) * V, a.N, f[j]);
    }
  } else {
    constexpr float top = Q == kQFp8 ? 448.f : 127.f;
    uint8_t* __restrict__ y = static_cast<uint8_t*>(a.y) + row * a.N;
    float amax[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      amax[j] = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) amax[j] = max_abs(amax[j], fabsf(f[j][i]));
    }
    if (a.groups == 1) {
#pragma unroll
      for (int j = 1; j < VPT; ++j) amax[0] = max_abs(amax[0], amax[j]);
      const float scale = scale_of(row_reduce<TPR>(amax[0], red[1], Max()), top), inv = 1.f / scale;
      if (!live) return;
      if (t == 0) a.scales[row] = scale;
#pragma unroll
      for (int j = 0; j < VPT; ++j) store_q<Q, V>(y, (lane() + j * TPR) * V, a.N, f[j], inv);
    } else {
      // a group is a run of group / V lanes (both powers of two, at most TPR and 64; host check)
      const int lanes = a.group / V;
      group_max(amax, lanes);
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const float scale = scale_of(amax[j], top), inv = 1.f / scale;
        const int c = (lane() + j * TPR) * V;
        if (live && c < a.N) {
          if (t % lanes == 0) a.scales[row * a.groups + c / a.group] = scale;
          store_q<Q, V>(y, c, a.N, f[j], inv);
        }
      }
    }
  }
}

// dx for every row, and the sum of dy h rstd over this workgroup's rows (every gridDim.x-th row
// group) in dw_part[workgroup][N].  The rows of a workgroup are summed in a fixed order, so equal
// inputs give equal bits.  HBM-bound as the forward.
template <typename T, int TPR, int VPT>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_bwd_kernel(RmsBwdArgs a) {
  constexpr int V = 16 / sizeof(T), NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;
  constexpr bool TINY = TPR == 8;
  __shared__ float red[2][NT / 64];
  __shared__ float acc[RPB > 1 ? (RPB - 1) * TPR * VPT * V : 1];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  float w[VPT][V], dw[VPT][V];
  {
    Cols<T, V> wr[VPT];
    weight_raw<T, V, TINY, TPR>(a.w, a.w_f32, t, 0, a.N, wr);
    to_weight<T, V, TINY, TPR>(wr, a.w, a.w_f32, t, 0, a.N, w);
  }
#pragma unroll
  for (int j = 0; j < VPT; ++j)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[j][i] = 0.f;
  int turn = 0;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.M; row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + slot;
    const bool live = row < a.M;
    const int64_t rl = live ? row : 0;
    const T* __restrict__ h = static_cast<const T*>(a.h) + rl * a.h_stride;
    const T* __restrict__ dy = static_cast<const T*>(a.dy) + rl * a.dy_stride;
    float f[VPT][V], g[VPT][V], s = 0.f;
    Cols<T, V> hr[VPT], yr[VPT], er[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      hr[j] = load_raw<T, V, TINY>(h, (t + j * TPR) * V, a.N);
      yr[j] = load_raw<T, V, TINY>(dy, (t + j * TPR) * V, a.N);
    }
    const float rstd = a.rstd[rl];
    const T* __restrict__ dh = static_cast<const T*>(a.dh) + rl * a.dh_stride;
    if (TPR < 512 && a.dh) {  // (late where a workgroup's size leaves few registers)
#pragma unroll
      for (int j = 0; j < VPT; ++j) er[j] = load_raw<T, V, TINY>(dh, (t + j * TPR) * V, a.N);
    }
    loads_issued();
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      to_cols<T, V, TINY>(hr[j], (t + j * TPR) * V, a.N, f[j]);
      to_cols<T, V, TINY>(yr[j], (t + j * TPR) * V, a.N, g[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        f[j][i] *= rstd;
        if (live) dw[j][i] += g[j][i] * f[j][i];
        g[j][i] *= w[j][i];
        s += g[j][i] * f[j][i];
      }
    }
    s = row_reduce<TPR>(s, red[turn], Add()) / (float)a.N;
    turn ^= 1;
    if (live) {
      T* __restrict__ dx = static_cast<T*>(a.dx) + row * a.N;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        float e[V];
        if (a.dh) {
          if (TPR >= 512) er[j] = load_raw<T, V, TINY>(dh, (t + j * TPR) * V, a.N);
          to_cols<T, V, TINY>(er[j], (t + j * TPR) * V, a.N, e);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) e[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < V; ++i) e[i] += rstd * (g[j][i] - f[j][i] * s);
        store_cols<T, V>(dx, (t + j * TPR) * V, a.N, e);
      }
    }
  }
  if (!a.dw_part) return;
  if constexpr (RPB > 1) {
    if (slot > 0) {
#pragma unroll
      for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) acc[((slot - 1) * VPT * V + j * V + i) * TPR + t] = dw[j][i];
    }
    __syncthreads();
    if (slot > 0) return;
    for (int q = 0; q < RPB - 1; ++q)
#pragma unroll
      for (int j = 0; j < VPT; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) dw[j][i] += acc[(q * VPT * V + j * V + i) * TPR + t];
  }
  float* __restrict__ p = a.dw_part + (int64_t)blockIdx.x * a.N;
#pragma unroll
  for (int j = 0; j < VPT; ++j) store_cols<float, V>(p, (t + j * TPR) * V, a.N, dw[j]);
}

// dw[c] = sum of part[0..P)[c], rounded once to the weight's type: 64 columns a workgroup, 16 threads
// to 4 columns, joined in a fixed order (512 parts of 2048 columns: 4.1 us; 20 with a thread to a column)
template <typename WT, bool TINY>
__global__ __launch_bounds__(256) void rms_dw_kernel(const float* __restrict__ part, WT* __restrict__ dw, int P, int N) {
  __shared__ float s[16][65];
  const int c = blockIdx.x * 64 + threadIdx.x % 16 * 4, k = threadIdx.x / 16;
  Cols<float, 4> sum = {};
#pragma unroll 8
  for (int p = k; p < P; p += 16) {
    const Cols<float, 4> e = load_raw<float, 4, TINY>(part + (int64_t)p * N, c, N);
#pragma unroll
    for (int i = 0; i < 4; ++i) sum.e[i] += e.e[i];
  }
  float v[4];
  to_cols<float, 4, TINY>(sum, c, N, v);
#pragma unroll
  for (int i = 0; i < 4; ++i) s[k][threadIdx.x % 16 * 4 + i] = v[i];
  __syncthreads();
  if (threadIdx.x < 64 && blockIdx.x * 64 + threadIdx.x < N) {
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) t += s[i][threadIdx.x];
    dw[blockIdx.x * 64 + threadIdx.x] = from_f32<WT>(t);
  }
}

// Few rows leave most of the chip without one: there a row of over 128 vectors is a workgroup's (bf16,
// residual, fp8; a wave's against a workgroup's.  2048 columns: 64 rows 4.8 and 3.6 us, 1024 rows 5.8
// and 5.5, 2048 rows 7.4 and 7.7; 1024 columns: 64 rows 3.7 and 3.8, 1024 rows 4.4 and 5.3).
RmsShape rms_shape(int64_t N, int vec, int64_t rows) {
  if (N < vec) return {8, 1};
  const int64_t nv = (N + vec - 1) / vec;
  if (nv <= 16) return {16, 1};
  if (nv <= 64) return {64, 1};
  if (nv <= 128) return {64, 2};
  if (nv <= 256 && rows <= 1024) return {256, 1};
  if (nv <= 256) return {64, 4};
  if (nv <= 512) return {256, 2};
  if (nv <= 1024) return {256, 4};
  if (nv <= 2048) return {256, 8};
  if (nv <= 4096) return {512, 8};
  return {1024, 8};
}

#define ATK_RMS_SHAPES(X) X(8, 1) X(16, 1) X(64, 1) X(64, 2) X(64, 4) X(256, 1) X(256, 2) X(256, 4) X(256, 8) X(512, 8) X(1024, 8)

// `rows` rows from `row` on
template <typename T, int Q>
RmsArgs rows_from(RmsArgs a, int64_t row, int64_t rows) {
  a.x = static_cast<const T*>(a.x) + row * a.x_stride;
  if (a.r) a.r = static_cast<const T*>(a.r) + row * a.r_stride;
  if (a.h) a.h = static_cast<T*>(a.h) + row * a.N;
  a.y = static_cast<char*>(a.y) + row * a.N * (Q == kQNone ? sizeof(T) : 1);
  if (a.rstd) a.rstd += row;
  if (a.scales) a.scales += row * a.groups;
  a.M = rows;
  return a;
}

// A launch has fewer than 2^32 threads, so a call of very many rows takes several.
template <typename T, int Q>
int launch_fwd(const RmsArgs& a, RmsShape sh, hipStream_t s) {
#define X(TPR, VPT)                                                                                     \
  if (sh.tpr == TPR && sh.vpt == VPT) {                                                                 \
    constexpr int NT = TPR < 256 ? 256 : TPR, RPB = NT / TPR;                                           \
    constexpr int64_t most = ((int64_t)1 << 31) / TPR;                                                  \
    for (int64_t row = 0; row < a.M; row += most) {                                                     \
      const RmsArgs b = rows_from<T, Q>(a, row, a.M - row < most ? a.M - row : most);                   \
      const dim3 grid((unsigned)((b.M + RPB - 1) / RPB));                                               \
      if (a.r) hipLaunchKernelGGL((rms_fwd_kernel<T, Q, TPR, VPT, true>), grid, dim3(NT), 0, s, b);     \
      else hipLaunchKernelGGL((rms_fwd_kernel<T, Q, TPR, VPT, false>), grid, dim3(NT), 0, s, b);        \
      if (int rc = check_launch("rms_fwd_kernel")) return rc;                                           \
    }                                                                                                   \
    return ATK_OK;                                                                                      \
  }
  ATK_RMS_SHAPES(X)
#undef X
  return fail(ATK_UNSUPPORTED, "rms_norm: no kernel for this row width");
}

template <typename T>
int launch_bwd(const RmsBwdArgs& a, RmsShape sh, int grid, hipStream_t s) {
#define X(TPR, VPT)                                                                                     \
  if (sh.tpr == TPR && sh.vpt == VPT) {                                                                 \
    hipLaunchKernelGGL((rms_bwd_kernel<T, TPR, VPT>), dim3((unsigned)grid), dim3(TPR < 256 ? 256 : TPR), 0, s, a); \
    return check_launch("rms_bwd_kernel");                                                              \
  }
  ATK_RMS_SHAPES(X)
#undef X
  return fail(ATK_UNSUPPORTED, "rms_norm backward: no kernel for this row width");
}

template <typename WT>
void launch_dw(const float* part, void* dw, int P, int N, hipStream_t s) {
  const dim3 g((unsigned)((N + 63) / 64));
  if (N >= 4) hipLaunchKernelGGL((rms_dw_kernel<WT, false>), g, dim3(256), 0, s, part, static_cast<WT*>(dw), P, N);
  else hipLaunchKernelGGL((rms_dw_kernel<WT, true>), g, dim3(256), 0, s, part, static_cast<WT*>(dw), P, N);
}

template <int Q>
int launch_fwd_typed(const RmsArgs& a, int dtype, RmsShape sh, hipStream_t s) {
  if (dtype == ATK_F32) return launch_fwd<float, Q>(a, sh, s);
  if (dtype == ATK_F16) return launch_fwd<_Float16, Q>(a, sh, s);
  return launch_fwd<__bf16, Q>(a, sh, s);
}

// columns that 1024 threads hold in registers: 65536 of 16 bits, 32768 of 32
int64_t max_cols(int dtype) { return (int64_t)1024 * 8 * (16 / (int64_t)dtype_size(dtype)); }

int check_rows(const char* what, int64_t M, int64_t N, int dtype, int w_dtype, bool has_w) {
  if (!dtype_ok(dtype)) return fail(ATK_EINVAL, "%s: unknown dtype code %d", what, dtype);
  if (has_w && w_dtype != dtype && w_dtype != ATK_F32)
    return fail(ATK_EINVAL, "%s: weight must be of the input's type or fp32", what);
  if (M < 0 || N < 0) return fail(ATK_EINVAL, "%s: negative size", what);
  if (N > max_cols(dtype)) return fail(ATK_UNSUPPORTED, "%s: rows of more than %lld columns", what, (long long)max_cols(dtype));
  if (M > 0x7fffffff) return fail(ATK_UNSUPPORTED, "%s: too many rows", what);
  return ATK_OK;
}

// Workgroups of the backward: enough to fill the chip, few enough that the partial sums of dw stay
// small beside the rows (each workgroup writes one row of fp32).  With dw's sum, at one, two and four to a
// CU, bf16: 8192 x 2048 26.5, 22.7 and 25.4 us; 8192 x 8192 93.9, 75.0 and 80.3; 65536 x 128 20.4, 15.7
// and 15.4; where one fills a CU's registers, 1024 x 16384, 30.9, 37.0 and 49.6.
int bwd_grid(int64_t M, RmsShape sh) {
  const int rpb = sh.tpr < 256 ? 256 / sh.tpr : 1;
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int64_t most = (int64_t)cus * (sh.vpt >= 8 ? 1 : 2), need = (M + rpb - 1) / rpb;
  return (int)(need < most ? need : most);
}

}  // namespace

int rows_dw(const float* part, void* dw, int P, int N, int w_dtype, hipStream_t s) {
  if (w_dtype == ATK_F32) launch_dw<float>(part, dw, P, N, s);
  else if (w_dtype == ATK_F16) launch_dw<_Float16>(part, dw, P, N, s);
  else launch_dw<__bf16>(part, dw, P, N, s);
  return check_launch("rms_dw_kernel");
}

}  // namespace atk

extern "C" int atk_rms_norm_fwd(const atk_rms_norm_args* p) {
  using namespace atk;
  if (!p) return fail(ATK_EINVAL, "rms_norm: null arguments");
  const int64_t M = p->M, N = p->N;
  const int dtype = p->dtype, quant = p->quant, group = p->group;
  if (int rc = check_rows("rms_norm", M, N, dtype, p->w_dtype, p->weight != nullptr)) return rc;
  if (quant < ATK_QUANT_NONE || quant > ATK_QUANT_INT8) return fail(ATK_EINVAL, "rms_norm: unknown output code %d", quant);
  if (M == 0 || N == 0) return ATK_OK;
  if (!p->x || !p->y || (p->residual && !p->h) || (quant && !p->scales)) return fail(ATK_EINVAL, "rms_norm: null pointer");
  if (M > 1 && (p->x_stride < N || (p->residual && p->residual_stride < N)))
    return fail(ATK_EINVAL, "rms_norm: rows overlap");
  const int vec = 16 / (int)dtype_size(dtype);
  RmsArgs a;
  a.groups = 1;
  if (quant && group > 0) {
    if ((group & (group - 1)) || group < 16 || group > 256)
      return fail(ATK_EINVAL, "rms_norm: groups of 16 to 256 columns, a power of two");
    a.groups = (int)((N + group - 1) / group);
  }
  a.x = p->x; a.r = p->residual; a.w = p->weight; a.y = p->y; a.h = p->h; a.rstd = p->rstd; a.scales = p->scales;
  a.M = M; a.x_stride = p->x_stride; a.r_stride = p->residual_stride;
  a.N = (int)N; a.group = group; a.w_f32 = p->w_dtype == ATK_F32; a.eps = p->eps;
  const RmsShape sh = rms_shape(N, vec, M);
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  if (quant == ATK_QUANT_FP8) return launch_fwd_typed<kQFp8>(a, dtype, sh, s);
  if (quant == ATK_QUANT_INT8) return launch_fwd_typed<kQInt8>(a, dtype, sh, s);
  return launch_fwd_typed<kQNone>(a, dtype, sh, s);
}

extern "C" size_t atk_rms_norm_bwd_workspace_bytes(int64_t M, int64_t N, int dtype) {
  using namespace atk;
  if (check_rows("rms_norm backward", M, N, dtype, dtype, false) || M == 0 || N == 0) return 0;
  const int vec = 16 / (int)dtype_size(dtype);
  return (size_t)bwd_grid(M, rms_shape(N, vec, M)) * (size_t)N * sizeof(float);
}

extern "C" int atk_rms_norm_bwd(const void* h, const void* dy, const void* dh, const void* weight, const float* rstd,
                                void* dx, void* dw, int64_t M, int64_t N, int64_t h_stride, int64_t dy_stride,
                                int64_t dh_stride, int dtype, int w_dtype, void* workspace, size_t workspace_bytes,
                                atk_stream_t stream) {
  using namespace atk;
  if (int rc = check_rows("rms_norm backward", M, N, dtype, w_dtype, weight != nullptr)) return rc;
  if (M == 0 || N == 0) return ATK_OK;
  if (!h || !dy || !rstd || !dx || (dw && !weight)) return fail(ATK_EINVAL, "rms_norm backward: null pointer");
  if (M > 1 && (h_stride < N || dy_stride < N || (dh && dh_stride < N)))
    return fail(ATK_EINVAL, "rms_norm backward: rows overlap");
  const int vec = 16 / (int)dtype_size(dtype);
  const RmsShape sh = rms_shape(N, vec, M);
  const int grid = bwd_grid(M, sh);
  if (dw && (!workspace || workspace_bytes < (size_t)grid * (size_t)N * sizeof(float)))
    return fail(ATK_EINVAL, "rms_norm backward: workspace too small");
  RmsBwdArgs a;
  a.h = h; a.dy = dy; a.dh = dh; a.w = weight; a.rstd = rstd; a.dx = dx;
  a.dw_part = dw ? static_cast<float*>(workspace) : nullptr;
  a.M = M; a.h_stride = h_stride; a.dy_stride = dy_stride; a.dh_stride = dh_stride;
  a.N = (int)N; a.w_f32 = w_dtype == ATK_F32;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  int rc = dtype == ATK_F32 ? launch_bwd<float>(a, sh, grid, s)
           : dtype == ATK_F16 ? launch_bwd<_Float16>(a, sh, grid, s) : launch_bwd<__bf16>(a, sh, grid, s);
  if (rc || !dw) return rc;
  return rows_dw(a.dw_part, dw, grid, (int)N, w_dtype, s);
}

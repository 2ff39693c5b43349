// Root-mean-square norm with a gate, over each group of a row's columns, and its backward.
//
//   gate behind:  y = n w act(z),  n = x rstd,  rstd = 1 / sqrt(mean(x^2) + eps)
//   gate first:   y = n w,         n = u rstd,  u = x act(z),  rstd = 1 / sqrt(mean(u^2) + eps)
//   with t = dy w act(z) (behind) or dy w (first), the gradient of what is normalised is
//     du = rstd (t - n mean(t n))
//   behind:  dx = du,         dz = dy w n act'(z),  dw = sum over rows of dy n act(z)
//   first:   dx = du act(z),  dz = du x act'(z),    dw = sum over rows of dy n
// act: SiLU, z s with s = 1 / (1 + exp(-z)), or s itself.
//
// HBM-bound: x, z (and dy) are read once and every output written once.  A row stays in registers between,
// the backward's as it was loaded (three inputs in fp32 would not fit), so no statistics are kept from the
// forward: mean(u^2) and mean(t u) come out of one reduction.  The threads of a row and the loads are those
// of the norm without a gate.  [8192, 2048] bf16, gate first: 19.5 us for 101 MB (5.2 TB/s), its backward 38.6 for
// 168 MB (4.3 TB/s) and 4 for the weight's sums; [64, 2048] in groups of 128 2.9 us, a launch's own time.
#include "row_cols.h"

namespace atk {
namespace {

struct GatedArgs {
  const void* x; const void* z; const void* w; const void* dy;
  void* y;                               // forward
  void* dx; void* dz; float* dw_part;    // backward
  int64_t M, x_stride, z_stride, dy_stride;
  int64_t N;                             // columns of a row, all of its groups'
  int n, w_f32, silu;                    // columns of a group
  float eps;
};

__device__ __forceinline__ float sigmoid_f32(float z) { return __builtin_amdgcn_rcpf(1.0f + __expf(-z)); }
__device__ __forceinline__ float gate_of(float z, int silu) {
  const float s = sigmoid_f32(z);
  return silu ? z * s : s;
}

// A group of columns for each blockIdx.y, rows of it for each blockIdx.x.
template <typename T, int TPR, int VPT, bool FIRST>
__global__ __launch_bounds__(256) void gated_fwd_kernel(GatedArgs a) {
  constexpr int V = 16 / sizeof(T), RPB = 256 / TPR;
  constexpr bool TINY = TPR == 8;
  __shared__ float red[4];
  const int t = threadIdx.x % TPR;
  const int64_t row = (int64_t)blockIdx.x * RPB + threadIdx.x / TPR, c0 = (int64_t)blockIdx.y * a.n;
  const bool live = row < a.M;  // a dead row takes part in its wave's reductions, and stores nothing
  const T* __restrict__ x = static_cast<const T*>(a.x) + (live ? row : 0) * a.x_stride + c0;
  const T* __restrict__ z = static_cast<const T*>(a.z) + (live ? row : 0) * a.z_stride + c0;
  const void* w = a.w ? static_cast<const char*>(a.w) + c0 * (a.w_f32 ? 4 : (int)sizeof(T)) : nullptr;
  Cols<T, V> xr[VPT], zr[VPT], wr[VPT];
#pragma unroll
  for (int j = 0; j < VPT; ++j) xr[j] = load_raw<T, V, TINY>(x, (t + j * TPR) * V, a.n);
#pragma unroll
  for (int j = 0; j < VPT; ++j) zr[j] = load_raw<T, V, TINY>(z, (t + j * TPR) * V, a.n);
  weight_raw<T, V, TINY, TPR>(w, a.w_f32, t, 0, a.n, wr);
  loads_issued();
  float f[VPT][V], ss = 0.f;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (t + j * TPR) * V;
    to_cols<T, V, TINY>(xr[j], c, a.n, f[j]);
    if constexpr (FIRST) {
      float g[V];
      to_cols<T, V, TINY>(zr[j], c, a.n, g);
#pragma unroll
      for (int i = 0; i < V; ++i) f[j][i] *= gate_of(g[i], a.silu);
    }
#pragma unroll
    for (int i = 0; i < V; ++i) ss += f[j][i] * f[j][i];
  }
  ss = row_reduce<TPR>(ss, red, Add());
  const float rstd = rsqrtf(ss / (float)a.n + a.eps);
  float wf[VPT][V];
  to_weight<T, V, TINY, TPR>(wr, w, a.w_f32, t, 0, a.n, wf);
  if (!live) return;
  T* __restrict__ y = static_cast<T*>(a.y) + row * a.N + c0;
#pragma unroll
  for (int j = 0; j < VPT; ++j) {
    const int c = (t + j * TPR) * V;
#pragma unroll
    for (int i = 0; i < V; ++i) f[j][i] = f[j][i] * rstd * wf[j][i];
    if constexpr (!FIRST) {
      float g[V];
      to_cols<T, V, TINY>(zr[j], c, a.n, g);
#pragma unroll
      for (int i = 0; i < V; ++i) f[j][i] *= gate_of(g[i], a.silu);
    }
    store_cols<T, V>(y, c, a.n, f[j]);
  }
}

// dx and dz of every row, and the sum over this workgroup's rows (every gridDim.x-th group of rows) of the
// weight's gradient in dw_part[blockIdx.x][N], in a fixed order: equal inputs give equal bits.
template <typename T, int TPR, int VPT, bool FIRST>
__global__ __launch_bounds__(256) void gated_bwd_kernel(GatedArgs a) {
  constexpr int V = 16 / sizeof(T), RPB = 256 / TPR;
  constexpr bool TINY = TPR == 8;
  __shared__ float red[2][2][4];
  __shared__ float acc[RPB > 1 ? (RPB - 1) * TPR * VPT * V : 1];
  const int t = threadIdx.x % TPR, slot = threadIdx.x / TPR;
  const int64_t c0 = (int64_t)blockIdx.y * a.n;
  const void* wp = a.w ? static_cast<const char*>(a.w) + c0 * (a.w_f32 ? 4 : (int)sizeof(T)) : nullptr;
  float w[VPT][V], dw[VPT][V];
  {
    Cols<T, V> wr[VPT];
    weight_raw<T, V, TINY, TPR>(wp, a.w_f32, t, 0, a.n, wr);
    to_weight<T, V, TINY, TPR>(wr, wp, a.w_f32, t, 0, a.n, w);
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
    const T* __restrict__ x = static_cast<const T*>(a.x) + rl * a.x_stride + c0;
    const T* __restrict__ z = static_cast<const T*>(a.z) + rl * a.z_stride + c0;
    const T* __restrict__ dy = static_cast<const T*>(a.dy) + rl * a.dy_stride + c0;
    Cols<T, V> xr[VPT], zr[VPT], yr[VPT];
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      xr[j] = load_raw<T, V, TINY>(x, (t + j * TPR) * V, a.n);
      zr[j] = load_raw<T, V, TINY>(z, (t + j * TPR) * V, a.n);
      yr[j] = load_raw<T, V, TINY>(dy, (t + j * TPR) * V, a.n);
    }
    loads_issued();
    float ss = 0.f, st = 0.f;  // of u^2 and of t u
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int c = (t + j * TPR) * V;
      float f[V], g[V], d[V];
      to_cols<T, V, TINY>(xr[j], c, a.n, f);
      to_cols<T, V, TINY>(zr[j], c, a.n, g);
      to_cols<T, V, TINY>(yr[j], c, a.n, d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float e = gate_of(g[i], a.silu), u = FIRST ? f[i] * e : f[i];
        const float up = d[i] * w[j][i];
        ss += u * u;
        st += FIRST ? up * u : up * e * u;
      }
    }
    ss = row_reduce<TPR>(ss, red[turn][0], Add());
    st = row_reduce<TPR>(st, red[turn][1], Add());
    turn ^= 1;
    const float rstd = rsqrtf(ss / (float)a.n + a.eps), mean = st * rstd / (float)a.n;
    if (live) {
      T* __restrict__ dx = static_cast<T*>(a.dx) + row * a.N + c0;
      T* __restrict__ dz = static_cast<T*>(a.dz) + row * a.N + c0;
#pragma unroll
      for (int j = 0; j < VPT; ++j) {
        const int c = (t + j * TPR) * V;
        float f[V], g[V], d[V];
        to_cols<T, V, TINY>(xr[j], c, a.n, f);
        to_cols<T, V, TINY>(zr[j], c, a.n, g);
        to_cols<T, V, TINY>(yr[j], c, a.n, d);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float s = sigmoid_f32(g[i]);
          const float e = a.silu ? g[i] * s : s;
          const float slope = s * (a.silu ? fmaf(g[i], 1.f - s, 1.f) : 1.f - s);
          const float n = (FIRST ? f[i] * e : f[i]) * rstd, up = d[i] * w[j][i];
          const float du = rstd * ((FIRST ? up : up * e) - n * mean);
          dw[j][i] += d[i] * n * (FIRST ? 1.f : e);
          g[i] = (FIRST ? du * f[i] : up * n) * slope;
          f[i] = FIRST ? du * e : du;
        }
        store_cols<T, V>(dx, c, a.n, f);
        store_cols<T, V>(dz, c, a.n, g);
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
  float* __restrict__ p = a.dw_part + (int64_t)blockIdx.x * a.N + c0;
#pragma unroll
  for (int j = 0; j < VPT; ++j) store_cols<float, V>(p, (t + j * TPR) * V, a.n, dw[j]);
}

#define ATK_GATED_SHAPES(X) X(8, 1) X(16, 1) X(64, 1) X(64, 2) X(64, 4) X(256, 1) X(256, 2) X(256, 4) X(256, 8)

constexpr int64_t kGatedVectors = 2048;  // of a group that 256 threads hold, 8 each

// Threads to a row and vectors to a thread, as for the norm without a gate.
RmsShape gated_shape(int64_t n, int vec, int64_t rows) {
  if (n < vec) return {8, 1};
  const int64_t nv = (n + vec - 1) / vec;
  if (nv <= 16) return {16, 1};
  if (nv <= 64) return {64, 1};
  if (nv <= 128) return {64, 2};
  if (nv <= 256) return rows <= 1024 ? RmsShape{256, 1} : RmsShape{64, 4};
  if (nv <= 512) return {256, 2};
  if (nv <= 1024) return {256, 4};
  return {256, 8};
}

template <typename T>
int launch_gated(const GatedArgs& all, bool first, RmsShape sh, hipStream_t s) {
  const int64_t groups = all.N / all.n;
#define X(TPR, VPT)                                                                                              \
  if (sh.tpr == TPR && sh.vpt == VPT) {                                                                          \
    /* a launch has fewer than 2^32 threads */                                                                   \
    const int64_t most = (((int64_t)1 << 31) / 256 / groups > 0 ? ((int64_t)1 << 31) / 256 / groups : 1) * (256 / TPR); \
    for (int64_t row = 0; row < all.M; row += most) {                                                            \
      GatedArgs a = all;                                                                                         \
      a.x = static_cast<const T*>(a.x) + row * a.x_stride;                                                       \
      a.z = static_cast<const T*>(a.z) + row * a.z_stride;                                                       \
      a.y = static_cast<T*>(a.y) + row * a.N;                                                                    \
      a.M = a.M - row < most ? a.M - row : most;                                                                 \
      const dim3 grid((unsigned)((a.M + 256 / TPR - 1) / (256 / TPR)), (unsigned)groups);                        \
      if (first) hipLaunchKernelGGL((gated_fwd_kernel<T, TPR, VPT, true>), grid, dim3(256), 0, s, a);            \
      else hipLaunchKernelGGL((gated_fwd_kernel<T, TPR, VPT, false>), grid, dim3(256), 0, s, a);                 \
      if (int rc = check_launch("gated_fwd_kernel")) return rc;                                                  \
    }                                                                                                            \
    return ATK_OK;                                                                                               \
  }
  ATK_GATED_SHAPES(X)
#undef X
  return fail(ATK_UNSUPPORTED, "rms_norm_gated: no kernel for this group");
}

template <typename T>
int launch_gated_bwd(const GatedArgs& a, bool first, RmsShape sh, int grid, hipStream_t s) {
  const dim3 g((unsigned)grid, (unsigned)(a.N / a.n));
#define X(TPR, VPT)                                                                                       \
  if (sh.tpr == TPR && sh.vpt == VPT) {                                                                   \
    if (first) hipLaunchKernelGGL((gated_bwd_kernel<T, TPR, VPT, true>), g, dim3(256), 0, s, a);          \
    else hipLaunchKernelGGL((gated_bwd_kernel<T, TPR, VPT, false>), g, dim3(256), 0, s, a);               \
    return check_launch("gated_bwd_kernel");                                                              \
  }
  ATK_GATED_SHAPES(X)
#undef X
  return fail(ATK_UNSUPPORTED, "rms_norm_gated backward: no kernel for this group");
}

int gated_check(const char* what, int64_t M, int64_t N, int64_t n, int dtype, int w_dtype, bool has_w, int act) {
  if (!dtype_ok(dtype)) return fail(ATK_EINVAL, "%s: unknown dtype code %d", what, dtype);
  if (has_w && w_dtype != dtype && w_dtype != ATK_F32)
    return fail(ATK_EINVAL, "%s: weight must be of the input's type or fp32", what);
  if (act != ATK_GATE_SILU && act != ATK_GATE_SIGMOID) return fail(ATK_EINVAL, "%s: unknown gate code %d", what, act);
  if (M < 0 || N < 0 || n < 0 || (N > 0 && (n == 0 || N % n))) return fail(ATK_EINVAL, "%s: bad sizes", what);
  if (M > 0x7fffffff || N > 0x7fffffff - 64) return fail(ATK_UNSUPPORTED, "%s: too many rows or columns", what);
  if (N > 0 && (N / n > 65535 || n > kGatedVectors * (16 / (int64_t)dtype_size(dtype))))
    return fail(ATK_UNSUPPORTED, "%s: groups of more than %lld columns, or more than 65535 of them", what,
                (long long)(kGatedVectors * (16 / (int64_t)dtype_size(dtype))));
  return ATK_OK;
}

// Workgroups of the backward for each group of columns: two to a CU in all, and no more than there are rows.
int gated_grid(int64_t M, int64_t groups, RmsShape sh) {
  const int cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int64_t rpb = 256 / sh.tpr, need = (M + rpb - 1) / rpb;
  const int64_t most = (int64_t)cus * (sh.vpt >= 8 ? 1 : 2) / groups;
  return (int)(need < most ? need : most > 0 ? most : 1);
}

}  // namespace
}  // namespace atk

extern "C" int atk_rms_norm_gated_fwd(const atk_rms_norm_gated_args* p) {
  using namespace atk;
  if (!p) return fail(ATK_EINVAL, "rms_norm_gated: null arguments");
  if (int rc = gated_check("rms_norm_gated", p->M, p->N, p->group, p->dtype, p->w_dtype, p->weight != nullptr, p->activation))
    return rc;
  if (p->M == 0 || p->N == 0) return ATK_OK;
  if (!p->x || !p->gate || !p->y) return fail(ATK_EINVAL, "rms_norm_gated: null pointer");
  if (p->M > 1 && (p->x_stride < p->N || p->gate_stride < p->N)) return fail(ATK_EINVAL, "rms_norm_gated: rows overlap");
  GatedArgs a = {};
  a.x = p->x; a.z = p->gate; a.w = p->weight; a.y = p->y;
  a.M = p->M; a.N = p->N; a.n = (int)p->group; a.x_stride = p->x_stride; a.z_stride = p->gate_stride;
  a.w_f32 = p->w_dtype == ATK_F32; a.silu = p->activation == ATK_GATE_SILU; a.eps = p->eps;
  const RmsShape sh = gated_shape(a.n, 16 / (int)dtype_size(p->dtype), a.M);
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  const bool first = p->gate_first != 0;
  if (p->dtype == ATK_F32) return launch_gated<float>(a, first, sh, s);
  if (p->dtype == ATK_F16) return launch_gated<_Float16>(a, first, sh, s);
  return launch_gated<__bf16>(a, first, sh, s);
}

extern "C" size_t atk_rms_norm_gated_bwd_workspace_bytes(int64_t M, int64_t N, int64_t group, int dtype) {
  using namespace atk;
  if (gated_check("rms_norm_gated backward", M, N, group, dtype, dtype, false, ATK_GATE_SILU) || M == 0 || N == 0) return 0;
  return (size_t)gated_grid(M, N / group, gated_shape(group, 16 / (int)dtype_size(dtype), M)) * (size_t)N * sizeof(float);
}

extern "C" int atk_rms_norm_gated_bwd(const atk_rms_norm_gated_args* p, const void* dy, int64_t dy_stride, void* dx, void* dgate,
                                      void* dw, void* workspace, size_t workspace_bytes) {
  using namespace atk;
  if (!p) return fail(ATK_EINVAL, "rms_norm_gated backward: null arguments");
  if (int rc = gated_check("rms_norm_gated backward", p->M, p->N, p->group, p->dtype, p->w_dtype, p->weight != nullptr,
                           p->activation))
    return rc;
  if (p->M == 0 || p->N == 0) return ATK_OK;
  if (!p->x || !p->gate || !dy || !dx || !dgate || (dw && !p->weight))
    return fail(ATK_EINVAL, "rms_norm_gated backward: null pointer");
  if (p->M > 1 && (p->x_stride < p->N || p->gate_stride < p->N || dy_stride < p->N))
    return fail(ATK_EINVAL, "rms_norm_gated backward: rows overlap");
  const RmsShape sh = gated_shape(p->group, 16 / (int)dtype_size(p->dtype), p->M);
  const int grid = gated_grid(p->M, p->N / p->group, sh);
  if (dw && (!workspace || workspace_bytes < (size_t)grid * (size_t)p->N * sizeof(float)))
    return fail(ATK_EINVAL, "rms_norm_gated backward: workspace too small");
  GatedArgs a = {};
  a.x = p->x; a.z = p->gate; a.w = p->weight; a.dy = dy; a.dx = dx; a.dz = dgate;
  a.dw_part = dw ? static_cast<float*>(workspace) : nullptr;
  a.M = p->M; a.N = p->N; a.n = (int)p->group; a.x_stride = p->x_stride; a.z_stride = p->gate_stride; a.dy_stride = dy_stride;
  a.w_f32 = p->w_dtype == ATK_F32; a.silu = p->activation == ATK_GATE_SILU; a.eps = p->eps;
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  const bool first = p->gate_first != 0;
  const int rc = p->dtype == ATK_F32 ? launch_gated_bwd<float>(a, first, sh, grid, s)
                 : p->dtype == ATK_F16 ? launch_gated_bwd<_Float16>(a, first, sh, grid, s)
                                       : launch_gated_bwd<__bf16>(a, first, sh, grid, s);
  if (rc || !dw) return rc;
  return rows_dw(a.dw_part, dw, grid, (int)p->N, p->w_dtype, s);
}

// The gated delta rule, one token at a time: the decode step over a cache of states, and short sequences.
//
//   S~ = exp(g) S;  u = beta (v - S~^T k);  S' = S~ + k u^T;  o = scale S'^T q
//
// S is [K, V] fp32 for each sequence and value head; value head h reads key head h / (Hv / Hk).
// HBM-bound: the state is read and written once and everything else is small, so the state stays
// in registers in between.  Both products over K are taken in the same pass over S, since
// S'^T q = exp(g) S^T q + (k . q) u; the one reduction across the workgroup carries both and k . q.
// The state is loaded and stored past the caches' replacement (nontemporal): by the next step every
// other layer has gone through them.  64 sequences, 32 heads, 128 x 128: 46 to 48 us for 268 MB, 5.7 TB/s
// (50.2 us with small loads that waited for each other, 58.2 with plain state accesses as well).
#include "gated_delta.h"

namespace atk {
namespace {

// A workgroup has NV * VW columns of one head's state: NV threads of VW columns side by side, 256 / NV
// groups of rows, RPT rows a thread.
template <typename T, int VW, int NV, int RPT>
__global__ __launch_bounds__(256) void gdr_step_kernel(GdrStepArgs a) {
  constexpr int RG = 256 / NV, W = 2 * VW;
  __shared__ float kf[RG * RPT], qf[RG * RPT];
  __shared__ float red[4][NV][W];
  __shared__ float red_kq[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int cg = tid % NV, rg = tid / NV;
  const int64_t n = blockIdx.z;
  const int h = blockIdx.y, hk = h / a.group;
  const int c0 = (blockIdx.x * NV + cg) * VW;
  const int64_t slot = a.slots ? (int64_t)a.slots[n] : n;
  T* __restrict__ o = static_cast<T*>(a.o) + (n * a.Hv + h) * (int64_t)a.V;
  if (slot < 0 || slot >= a.n_slots) {  // a row of padding: no state, an output of zeros
    if (rg == 0)
#pragma unroll
      for (int j = 0; j < VW; ++j)
        if (c0 + j < a.V) o[c0 + j] = from_f32<T>(0.f);
    return;
  }
  float* __restrict__ S = a.state + slot * a.state_stride + (int64_t)h * a.K * a.V;
  // All loads at once, none in a branch that converts: the small ones first, the state while they arrive.
  const T* __restrict__ k = static_cast<const T*>(a.k) + n * a.k_sb + hk * a.k_sh;
  const T* __restrict__ q = static_cast<const T*>(a.q) + n * a.q_sb + hk * a.q_sh;
  const T* __restrict__ v = static_cast<const T*>(a.v) + n * a.v_sb + h * a.v_sh;
  const GdrGate gr = gdr_gate_load(a.g, a.g_dtype, n * a.g_sb + h * a.g_sh);
  const GdrGate br = gdr_gate_load(a.beta, a.b_dtype, n * a.b_sb + h * a.b_sh);
  constexpr int KL = (RG * RPT + 255) / 256;
  T kr0[KL], qr0[KL], vr[VW];
#pragma unroll
  for (int z = 0; z < KL; ++z) {
    const int r = tid + 256 * z < a.K ? tid + 256 * z : 0;
    kr0[z] = k[r];
    qr0[z] = q[r];
  }
  __builtin_memcpy(vr, v + (c0 < a.V ? c0 : 0), VW * sizeof(T));  // V is a multiple of VW (host check)
  float s[RPT][VW];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg + i * RG;
    const bool in = r < a.K && c0 < a.V;
    if constexpr (VW == 4) {
      const uint4 t = in ? ld16<true>(S + (int64_t)r * a.V + c0) : make_uint4(0, 0, 0, 0);
      s[i][0] = __uint_as_float(t.x); s[i][1] = __uint_as_float(t.y);
      s[i][2] = __uint_as_float(t.z); s[i][3] = __uint_as_float(t.w);
    } else {
      s[i][0] = in ? S[(int64_t)r * a.V + c0] : 0.f;
    }
  }
#pragma unroll
  for (int z = 0; z < KL; ++z) {
    const int r = tid + 256 * z;
    if (r < RG * RPT) {
      kf[r] = r < a.K ? to_f32(kr0[z]) : 0.f;
      qf[r] = r < a.K ? to_f32(qr0[z]) : 0.f;
    }
  }
  const float decay = expf(gdr_gate<T>(gr, a.g_dtype)), beta = gdr_gate<T>(br, a.b_dtype);
  float vv[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) vv[j] = c0 < a.V ? to_f32(vr[j]) : 0.f;
  __syncthreads();
  float p[W], kq = 0.f;
#pragma unroll
  for (int j = 0; j < W; ++j) p[j] = 0.f;
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const float kr = kf[rg + i * RG], qr = qf[rg + i * RG];
    kq += kr * qr;
#pragma unroll
    for (int j = 0; j < VW; ++j) {
      p[j] += s[i][j] * kr;
      p[VW + j] += s[i][j] * qr;
    }
  }
#pragma unroll
  for (int off = NV; off < 64; off <<= 1) {
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] += __shfl_xor(p[j], off, 64);
    kq += __shfl_xor(kq, off, 64);
  }
  if (lane < NV) {
#pragma unroll
    for (int j = 0; j < W; ++j) red[wave][cg][j] = p[j];
    if (lane == 0) red_kq[wave] = kq;
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < W; ++j) p[j] = (red[0][cg][j] + red[1][cg][j]) + (red[2][cg][j] + red[3][cg][j]);
  kq = (red_kq[0] + red_kq[1]) + (red_kq[2] + red_kq[3]);
  float u[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) u[j] = beta * (vv[j] - decay * p[j]);
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg + i * RG;
    const float kr = kf[r];
    if (r < a.K && c0 < a.V) {
      if constexpr (VW == 4) {
        const float x[4] = {decay * s[i][0] + kr * u[0], decay * s[i][1] + kr * u[1], decay * s[i][2] + kr * u[2],
                            decay * s[i][3] + kr * u[3]};
        st16<true>(S + (int64_t)r * a.V + c0, pack16<float>(x));
      } else {
        S[(int64_t)r * a.V + c0] = decay * s[i][0] + kr * u[0];
      }
    }
  }
  if (rg == 0) {
#pragma unroll
    for (int j = 0; j < VW; ++j)
      if (c0 + j < a.V) o[c0 + j] = from_f32<T>(a.scale * (decay * p[VW + j] + kq * u[j]));
  }
}

template <typename T, int VW, int NV, int RPT>
void launch_step(const GdrStepArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.V + NV * VW - 1) / (NV * VW)), (unsigned)a.Hv, (unsigned)a.n);
  hipLaunchKernelGGL((gdr_step_kernel<T, VW, NV, RPT>), grid, dim3(256), 0, s, a);
}

template <typename T>
void launch_step_typed(const GdrStepArgs& a, hipStream_t s) {
  const bool vec = a.V % 4 == 0 && aligned16(a.state) && a.state_stride % 4 == 0;
  // 128 columns a workgroup (its waves then read whole rows) where that is one for each CU at least; 32
  // below, to spread the state over the chip.  32 heads of 128 x 128, states not in any cache: 16
  // sequences 11.6 us against 15.0, 64 sequences 45.8 against 50.7; 4 sequences 5.8 against 5.2.
  const bool wide = (a.V + 127) / 128 * (int64_t)a.Hv * a.n >= (device_cu_count() > 0 ? device_cu_count() : 256);
  if (!vec) {
    if (a.K <= 64) launch_step<T, 1, 64, 16>(a, s);
    else if (a.K <= 128) launch_step<T, 1, 64, 32>(a, s);
    else launch_step<T, 1, 64, 64>(a, s);
  } else if (wide) {
    if (a.K <= 64) launch_step<T, 4, 32, 8>(a, s);
    else if (a.K <= 128) launch_step<T, 4, 32, 16>(a, s);
    else launch_step<T, 4, 32, 32>(a, s);
  } else {
    if (a.K <= 64) launch_step<T, 4, 8, 2>(a, s);
    else if (a.K <= 128) launch_step<T, 4, 8, 4>(a, s);
    else launch_step<T, 4, 8, 8>(a, s);
  }
}

// A few tokens of each sequence, one after the other, with the state in registers throughout: what
// short calls take (a chunk's two launches are as long as 10 tokens here).  A workgroup has 32
// columns (VW 4) or 64 (VW 1) of a head; the next token's inputs are on their way meanwhile.
template <typename T, int VW, int NV, int RPT>
__global__ __launch_bounds__(256) void gdr_tokens_kernel(GdrArgs a) {
  constexpr int RG = 256 / NV, W = 2 * VW, KL = (RG * RPT + 255) / 256;
  __shared__ float kf[2][RG * RPT], qf[2][RG * RPT];
  __shared__ float red[2][4][NV][W];
  __shared__ float red_kq[2][4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int cg = tid % NV, rg = tid / NV;
  const int64_t n = blockIdx.z;
  const int h = blockIdx.y, hk = h / a.group;
  const int c0 = (blockIdx.x * NV + cg) * VW;
  const bool live = c0 < a.V;  // V is a multiple of VW (host check)
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t at = (n * a.Hv + h) * (int64_t)a.K * a.V + c0;
  float s[RPT][VW];
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg + i * RG;
    if constexpr (VW == 4) {
      const float4 t = a.s0 && live && r < a.K ? *reinterpret_cast<const float4*>(a.s0 + at + (int64_t)r * a.V) : make_float4(0.f, 0.f, 0.f, 0.f);
      s[i][0] = t.x; s[i][1] = t.y; s[i][2] = t.z; s[i][3] = t.w;
    } else {
      s[i][0] = a.s0 && live && r < a.K ? a.s0[at + (int64_t)r * a.V] : 0.f;
    }
  }
  const T* __restrict__ k = static_cast<const T*>(a.k) + seq.batch * a.k_s[0] + seq.begin * a.k_s[1] + hk * a.k_s[2];
  const T* __restrict__ q = static_cast<const T*>(a.q) + seq.batch * a.q_s[0] + seq.begin * a.q_s[1] + hk * a.q_s[2];
  const T* __restrict__ v = static_cast<const T*>(a.v) + seq.batch * a.v_s[0] + seq.begin * a.v_s[1] + h * a.v_s[2];
  T* __restrict__ o = static_cast<T*>(a.o) + ((seq.batch * a.T + seq.begin) * a.Hv + h) * (int64_t)a.V;
  T kn[KL], qn[KL], vn[VW];  // as they are in memory: a conversion would wait for its load
  GdrGate gn, bn;
  auto load = [&](int64_t t) {
    gn = gdr_gate_load(a.g, a.g_dtype, seq.batch * a.g_s[0] + (seq.begin + t) * a.g_s[1] + h * a.g_s[2]);
    bn = gdr_gate_load(a.beta, a.b_dtype, seq.batch * a.b_s[0] + (seq.begin + t) * a.b_s[1] + h * a.b_s[2]);
#pragma unroll
    for (int z = 0; z < KL; ++z) {
      const int r = tid + 256 * z < a.K ? tid + 256 * z : 0;
      kn[z] = k[t * a.k_s[1] + r];
      qn[z] = q[t * a.q_s[1] + r];
    }
    __builtin_memcpy(vn, v + t * a.v_s[1] + (live ? c0 : 0), VW * sizeof(T));
  };
  if (seq.len > 0) load(0);
  for (int64_t t = 0; t < seq.len; ++t) {
    const int b = t & 1;
#pragma unroll
    for (int z = 0; z < KL; ++z)
      if (tid + 256 * z < RG * RPT) {
        kf[b][tid + 256 * z] = tid + 256 * z < a.K ? to_f32(kn[z]) : 0.f;
        qf[b][tid + 256 * z] = tid + 256 * z < a.K ? to_f32(qn[z]) : 0.f;
      }
    const float decay = expf(gdr_gate<T>(gn, a.g_dtype)), beta = gdr_gate<T>(bn, a.b_dtype);
    float vv[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) vv[j] = live ? to_f32(vn[j]) : 0.f;
    load(t + 1 < seq.len ? t + 1 : t);
    __syncthreads();
    float p[W], kq = 0.f;
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] = 0.f;
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const float kr = kf[b][rg + i * RG], qr = qf[b][rg + i * RG];
      kq += kr * qr;
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        p[j] += s[i][j] * kr;
        p[VW + j] += s[i][j] * qr;
      }
    }
#pragma unroll
    for (int off = NV; off < 64; off <<= 1) {
#pragma unroll
      for (int j = 0; j < W; ++j) p[j] += __shfl_xor(p[j], off, 64);
      kq += __shfl_xor(kq, off, 64);
    }
    if (lane < NV) {
#pragma unroll
      for (int j = 0; j < W; ++j) red[b][wave][cg][j] = p[j];
      if (lane == 0) red_kq[b][wave] = kq;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < W; ++j) p[j] = (red[b][0][cg][j] + red[b][1][cg][j]) + (red[b][2][cg][j] + red[b][3][cg][j]);
    kq = (red_kq[b][0] + red_kq[b][1]) + (red_kq[b][2] + red_kq[b][3]);
    float u[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) u[j] = beta * (vv[j] - decay * p[j]);
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const float kr = kf[b][rg + i * RG];
#pragma unroll
      for (int j = 0; j < VW; ++j) s[i][j] = decay * s[i][j] + kr * u[j];
    }
    if (rg == 0 && live) {
#pragma unroll
      for (int j = 0; j < VW; ++j) o[t * a.Hv * (int64_t)a.V + c0 + j] = from_f32<T>(a.scale * (decay * p[VW + j] + kq * u[j]));
    }
    // (the buffers of this token are written again two barriers from here at the earliest)
  }
  if (a.s1) {
#pragma unroll
    for (int i = 0; i < RPT; ++i) {
      const int r = rg + i * RG;
      if (!live || r >= a.K) continue;
      if constexpr (VW == 4) *reinterpret_cast<float4*>(a.s1 + at + (int64_t)r * a.V) = make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
      else a.s1[at + (int64_t)r * a.V] = s[i][0];
    }
  }
  // tokens of a packed row before its first sequence and after its last have an output of zero
  if (a.cu && live && (n == 0 || n == a.n - 1)) {
    T* __restrict__ all = static_cast<T*>(a.o);
    const int64_t from[2] = {n == 0 ? 0 : a.T, n == a.n - 1 ? seq.begin + seq.len : a.T};
    const int64_t to[2] = {n == 0 ? seq.begin : a.T, a.T};
    for (int z = 0; z < 2; ++z)
      for (int64_t i = from[z] + rg; i < to[z]; i += RG)
#pragma unroll
        for (int j = 0; j < VW; ++j) all[(i * a.Hv + h) * (int64_t)a.V + c0 + j] = from_f32<T>(0.f);
  }
}

template <typename T, int VW, int NV, int RPT>
void launch_tokens(const GdrArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.V + NV * VW - 1) / (NV * VW)), (unsigned)a.Hv, (unsigned)a.n);
  hipLaunchKernelGGL((gdr_tokens_kernel<T, VW, NV, RPT>), grid, dim3(256), 0, s, a);
}
template <typename T>
void launch_tokens_typed(const GdrArgs& a, hipStream_t s) {
  if (a.V % 4 || !aligned16(a.s0) || !aligned16(a.s1)) {
    if (a.K <= 64) launch_tokens<T, 1, 64, 16>(a, s);
    else if (a.K <= 128) launch_tokens<T, 1, 64, 32>(a, s);
    else launch_tokens<T, 1, 64, 64>(a, s);
  } else {
    if (a.K <= 64) launch_tokens<T, 4, 8, 2>(a, s);
    else if (a.K <= 128) launch_tokens<T, 4, 8, 4>(a, s);
    else launch_tokens<T, 4, 8, 8>(a, s);
  }
}

}  // namespace

int gdr_tokens(const GdrArgs& a, int dtype, hipStream_t s) {
  if (dtype == ATK_F32) launch_tokens_typed<float>(a, s);
  else if (dtype == ATK_F16) launch_tokens_typed<_Float16>(a, s);
  else launch_tokens_typed<__bf16>(a, s);
  return check_launch("gdr_tokens_kernel");
}

}  // namespace atk

extern "C" int atk_gated_delta_update(const atk_gated_delta_update_args* p) {
  using namespace atk;
  if (!p) return fail(ATK_EINVAL, "gated delta update: null arguments");
  if (!dtype_ok(p->dtype) || !dtype_ok(p->g_dtype) || !dtype_ok(p->beta_dtype))
    return fail(ATK_EINVAL, "gated delta update: unknown dtype code");
  if (!gdr_gate_ok(p->g_dtype, p->dtype) || !gdr_gate_ok(p->beta_dtype, p->dtype))
    return fail(ATK_EINVAL, "gated delta update: g and beta must be of the inputs' type or fp32");
  if (p->N < 0 || p->Hk <= 0 || p->Hv <= 0 || p->K <= 0 || p->V <= 0 || p->slots < 0)
    return fail(ATK_EINVAL, "gated delta update: bad sizes");
  if (p->Hv % p->Hk) return fail(ATK_EINVAL, "gated delta update: value heads must be a multiple of key heads");
  if (p->K > kGdrMaxK || p->Hv > 65535 || p->N > 65535)
    return fail(ATK_UNSUPPORTED, "gated delta update: more than %d key columns, 65535 heads or sequences", kGdrMaxK);
  if (p->N == 0) return ATK_OK;
  if (!p->q || !p->k || !p->v || !p->g || !p->beta || !p->state || !p->out)
    return fail(ATK_EINVAL, "gated delta update: null pointer");
  if (!p->state_indices && p->N > p->slots) return fail(ATK_EINVAL, "gated delta update: fewer states than sequences");
  GdrStepArgs a;
  a.q = p->q; a.k = p->k; a.v = p->v; a.g = p->g; a.beta = p->beta;
  a.state = static_cast<float*>(p->state); a.o = p->out; a.slots = p->state_indices;
  a.n = p->N; a.n_slots = p->slots; a.state_stride = p->state_stride;
  a.q_sb = p->q_stride_n; a.q_sh = p->q_stride_h; a.k_sb = p->k_stride_n; a.k_sh = p->k_stride_h;
  a.v_sb = p->v_stride_n; a.v_sh = p->v_stride_h; a.g_sb = p->g_stride_n; a.g_sh = p->g_stride_h;
  a.b_sb = p->beta_stride_n; a.b_sh = p->beta_stride_h;
  a.Hv = p->Hv; a.group = p->Hv / p->Hk; a.K = p->K; a.V = p->V;
  a.g_dtype = p->g_dtype; a.b_dtype = p->beta_dtype; a.scale = p->scale;
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  if (p->dtype == ATK_F32) launch_step_typed<float>(a, s);
  else if (p->dtype == ATK_F16) launch_step_typed<_Float16>(a, s);
  else launch_step_typed<__bf16>(a, s);
  return check_launch("gdr_step_kernel");
}

// Linear attention with a decay for each head: the decode step over a cache of states, what joins the
// segments of sequences, and the C entries.
//
//   S' = exp(g) S + k v^T;  o = scale S'^T q
#include <math.h>

#include "linear_attn.h"

namespace atk {
namespace {

struct LaStepArgs {
  const void* q; const void* k; const void* v; const void* g;
  float* state; void* o; const int* slots;
  int64_t n, n_slots, state_stride;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, g_sb, g_sh;  // strides in elements: sequence, head
  int Hv, group, K, V, g_dtype;
  float scale;
};

// The decode step is HBM-bound: the state is read and written once, past the caches' replacement
// (nontemporal), since every other layer has gone through them by the next step.  A new element is stored
// as soon as its old one is there; only o waits for a reduction over the rows.
// 64 sequences of 32 heads of 128 x 128: 48.8 us for 270 MB, 5.5 TB/s; one of 16 heads 3.8 us, a launch's own time.
// A workgroup has NV * VW columns of one head's state: NV threads of VW columns side by side, 256 / NV
// groups of rows, RPT rows a thread.
template <typename T, int VW, int NV, int RPT>
__global__ __launch_bounds__(256) void la_step_kernel(LaStepArgs a) {
  constexpr int RG = 256 / NV, KL = (RG * RPT + 255) / 256;
  __shared__ float kf[RG * RPT], qf[RG * RPT];
  __shared__ float red[4][NV][VW];
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
  const T* __restrict__ q = static_cast<const T*>(a.q) + n * a.q_sb + hk * a.q_sh;
  const T* __restrict__ k = static_cast<const T*>(a.k) + n * a.k_sb + hk * a.k_sh;
  const T* __restrict__ v = static_cast<const T*>(a.v) + n * a.v_sb + h * a.v_sh;
  // every load before the first conversion, so that they are in flight together
  T kr[KL], qr[KL], vr[VW];
#pragma unroll
  for (int z = 0; z < KL; ++z) {
    const int r = tid + 256 * z, at = r < a.K ? r : 0;
    kr[z] = k[at];
    qr[z] = q[at];
  }
#pragma unroll
  for (int j = 0; j < VW; ++j) vr[j] = v[c0 + j < a.V ? c0 + j : 0];
  const GdrGate gr = gdr_gate_load(a.g, a.g_dtype, n * a.g_sb + h * a.g_sh);
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
      kf[r] = r < a.K ? to_f32(kr[z]) : 0.f;
      qf[r] = r < a.K ? to_f32(qr[z]) : 0.f;
    }
  }
  const float decay = expf(gdr_gate<T>(gr, a.g_dtype));
  float vv[VW], p[VW];
#pragma unroll
  for (int j = 0; j < VW; ++j) {
    vv[j] = to_f32(vr[j]);
    p[j] = 0.f;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < RPT; ++i) {
    const int r = rg + i * RG;
    const float kk = kf[r], qq = qf[r];
    if (r < a.K && c0 < a.V) {
      float x[VW];
#pragma unroll
      for (int j = 0; j < VW; ++j) {
        x[j] = fmaf(decay, s[i][j], kk * vv[j]);
        p[j] += x[j] * qq;
      }
      if constexpr (VW == 4) st16<true>(S + (int64_t)r * a.V + c0, pack16<float>(x));
      else S[(int64_t)r * a.V + c0] = x[0];
    }
  }
#pragma unroll
  for (int off = NV; off < 64; off <<= 1)
#pragma unroll
    for (int j = 0; j < VW; ++j) p[j] += __shfl_xor(p[j], off, 64);
  if (lane < NV)
#pragma unroll
    for (int j = 0; j < VW; ++j) red[wave][cg][j] = p[j];
  __syncthreads();
  if (rg == 0)
#pragma unroll
    for (int j = 0; j < VW; ++j)
      if (c0 + j < a.V)
        o[c0 + j] = from_f32<T>(a.scale * ((red[0][cg][j] + red[1][cg][j]) + (red[2][cg][j] + red[3][cg][j])));
}

template <typename T, int VW, int NV, int RPT>
void launch_step(const LaStepArgs& a, hipStream_t s) {
  const dim3 grid((unsigned)((a.V + NV * VW - 1) / (NV * VW)), (unsigned)a.Hv, (unsigned)a.n);
  hipLaunchKernelGGL((la_step_kernel<T, VW, NV, RPT>), grid, dim3(256), 0, s, a);
}
template <typename T>
void launch_step_typed(const LaStepArgs& a, hipStream_t s) {
  const bool vec = a.V % 4 == 0 && aligned16(a.state) && a.state_stride % 4 == 0;
  // 128 columns a workgroup where that is one for each CU at least; 32 below, to spread the state over the
  // chip (as for the gated delta rule's step, whose traffic this has)
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

// Segments joined: what each adds to the state becomes the state after it (in reverse, the gradient of the
// state before it), in place.  A thread has VW elements of a state, all segments of a sequence, eight of them in
// flight.  HBM-bound: 15 states of 32 heads of 128 x 128, 12.6 us for 63 MB, 5 TB/s.
template <int VW>
__global__ __launch_bounds__(256) void la_scan_kernel(LaArgs a, float* s0, float* s1, const float* decays, FastDiv per, int first,
                                                      int marks) {
  const uint32_t unit = fdiv(blockIdx.x, per), ih = first + unit, index = fdiv(ih, a.by_hv);
  const int h = (int)(ih - index * a.by_hv.d);
  int n = (int)index;
  LaSeq seq;
  if (marks) {  // the sequence with its first token of those that la_segment_at goes by
    int z;
    if (!la_segment_at(a, (int)index, &n, &seq, &z) || z > 0) return;
  } else {
    seq = la_seq(a, n);
  }
  const int kv = a.K * a.V, segs = seq.segs;
  const bool rev = blockIdx.y;
  if (segs == 1) return;
  for (int i = (int)((blockIdx.x - unit * per.d) * 256 + threadIdx.x) * VW; i < kv; i += (int)per.d * 256 * VW) {
    const float* init = a.role[rev].s_first;
    float run[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) run[j] = init ? init[((int64_t)n * a.Hv + h) * kv + i + j] : 0.f;
    const int64_t step = (int64_t)a.Hv * kv;
    float* __restrict__ p = (rev ? s1 : s0) + (seq.end + (rev ? segs - 2 : 0)) * step + (int64_t)h * kv + i;
    const float* __restrict__ d = decays + ((int64_t)(rev ? a.ends : 0) + seq.end + (rev ? segs - 2 : 0)) * a.Hv + h;
    const int64_t ps = rev ? -step : step, ds = rev ? -a.Hv : a.Hv;
    constexpr int U = 8;  // segments whose loads are in flight together
    for (int z = 0; z + 1 < segs; z += U) {
      float t[U][VW], f[U];
      const int left = segs - 1 - z;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = u < left ? u : 0;
        __builtin_memcpy(t[u], p + at * ps, 4 * VW);
        f[u] = d[at * ds];
      }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (u < left) {
#pragma unroll
          for (int j = 0; j < VW; ++j) run[j] = fmaf(f[u], run[j], t[u][j]);
          __builtin_memcpy(p + u * ps, run, 4 * VW);
        }
      p += U * ps;
      d += U * ds;
    }
  }
}

// Sums of a gradient's parts, over value heads of a key head and tiles of value columns, rounded once.
struct LaSumArgs {
  const float* parts[2]; void* out[2];
  int64_t count;  // elements of the gradient
  int n;          // parts
};
template <typename T, int VW>
__global__ __launch_bounds__(256) void la_sum_kernel(LaSumArgs a) {
  const float* __restrict__ p = a.parts[blockIdx.y];
  T* __restrict__ o = static_cast<T*>(a.out[blockIdx.y]);
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * VW; i < a.count; i += (int64_t)gridDim.x * 256 * VW) {
    float s[VW];
    __builtin_memcpy(s, p + i, 4 * VW);
    for (int k = 1; k < a.n; ++k) {
      float t[VW];
      __builtin_memcpy(t, p + k * a.count + i, 4 * VW);
#pragma unroll
      for (int j = 0; j < VW; ++j) s[j] += t[j];
    }
    T e[VW];
#pragma unroll
    for (int j = 0; j < VW; ++j) e[j] = from_f32<T>(s[j]);
    __builtin_memcpy(o + i, e, VW * sizeof(T));
  }
}

// The gradient of a log decay: q_t . dq_t - k_t . dk_t, both without the token's product with itself, which has no
// decay, summed from t to the end of the segment, and the inner product of the state there with its gradient.  A
// wave for each segment and head.  What is left has the decays as the sum has, but cancels where weak ones stand
// beside strong ones, so the sums are in 64 bits.  Latency of a wave's loads and six steps of its sums for each 64
// tokens: 2 x 2048 tokens of 16 heads, segments of 256, 6.7 us.
struct LaGateArgs {
  const float* qd; const float* kd; const float* x; void* dg; float* seg_sums;
  int tiles;
  uint32_t unit0;  // segments of heads before this launch's
};
template <typename G>
__global__ __launch_bounds__(256) void la_gate_kernel(LaArgs a, LaGateArgs b) {
  const int lane = threadIdx.x & 63;
  const uint32_t unit = b.unit0 + blockIdx.x * 4 + (threadIdx.x >> 6);
  const int slot = (int)fdiv(unit, a.by_hv), h = (int)unit - slot * a.Hv;
  if (slot >= a.slots) return;
  const int n = la_seq_of_slot(a, slot);
  const LaSeq seq = la_seq(a, n);
  const int z = slot - seq.slot, segs = seq.segs;
  const bool live = z >= 0 && z < segs;
  const int64_t BT = a.B * a.T;
  double carry = 0, all = 0;
  if (live) {
    const int t0 = z * a.seg, left = seq.len - t0, len = left < a.seg ? left : a.seg;
    const int64_t first = (int64_t)seq.batch * a.T + seq.begin + t0;
    for (int t = 0; t < b.tiles; ++t) carry += (double)b.x[((int64_t)t * a.slots + slot) * a.Hv + h];
    for (int end = len; end > 0; end -= 64) {
      const int t = end - 1 - lane;  // the lane's token, from the end
      const int64_t at = first + (t > 0 ? t : 0);
      double v = 0;
      for (int i = 0; i < b.tiles; ++i) {
        const int64_t j = ((int64_t)i * a.Hv + h) * BT + at;
        v += (double)b.qd[j] - (double)b.kd[j];
      }
      if (t < 0) v = 0;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double o = __shfl_up(v, off, 64);
        if (lane >= off) v += o;
      }
      const GdrGate gr = gdr_gate_load(a.g, a.g_dtype, seq.batch * a.g_s[0] + (int64_t)(seq.begin + t0 + (t > 0 ? t : 0)) * a.g_s[1] + h * a.g_s[2]);
      const double dg = gdr_gate<G>(gr, a.g_dtype) < -120.f ? 0.0 : carry + v;
      if (t >= 0) {
        if (!a.fixed) static_cast<G*>(b.dg)[at * a.Hv + h] = from_f32<G>((float)dg);
        all += dg;
      }
      carry += __shfl(v, 63, 64);
    }
  }
  if (a.fixed) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) all += __shfl_xor(all, off, 64);
    if (lane == 0) b.seg_sums[(int64_t)h * a.slots + slot] = (float)all;
  } else {
    la_outside(a, slot, [&](int64_t from, int64_t to) {
      for (int64_t t = from + lane; t < to; t += 64) static_cast<G*>(b.dg)[t * a.Hv + h] = from_f32<G>(0.f);
    });
  }
}
// one decay a head: its gradient is the sum over all segments
template <typename G>
__global__ __launch_bounds__(256) void la_gate_sum_kernel(const float* __restrict__ sums, G* __restrict__ dg, int64_t slots) {
  __shared__ double red[256];
  double s = 0;
  for (int64_t i = threadIdx.x; i < slots; i += 256) s += (double)sums[blockIdx.x * slots + i];
  red[threadIdx.x] = s;
  __syncthreads();
  for (int k = 128; k >= 1; k >>= 1) {
    if ((int)threadIdx.x < k) red[threadIdx.x] += red[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) dg[blockIdx.x] = from_f32<G>((float)red[0]);
}

struct LaPlan {
  float* s_fwd; float* s_rev; float* decays; float* parts[2]; float* dots[2]; float* x; float* seg_sums;
  int n_parts, k_tiles, a_tiles;
  bool split;   // more than one segment
  size_t bytes;
};

// Tokens of a segment.  Segments of a sequence run at once, each going through its chunks one after the other,
// for the price of their states.  The length is the one with the least time by a model fitted to what was measured, in
// us, whose workgroups on a CU are three for states of up to 64 rows, two for up to 128 and one above.  (Not of every
// kernel: fp32 outputs of 128 rows and 128 columns have one, gradients of 64 rows two.  That is in the types' factors.)
//   a step of 64 tokens, states and outputs together, takes 5.5 where each CU has half a workgroup (of 128 columns), 7
//   where it has one, 10 where it has two, whatever it holds (bf16, 128 key columns; a state of 256 has one a CU and
//   7.5, one of 64 three and 0.65 of the time; fp16 x 1.75, fp32 x 2.4), more workgroups take turns;
//   + the states, written and read twice, at 4.4 TB/s, and the launches, 5;
// or that of one segment a sequence, with no states between and steps of 4, 5.8 and 8.
//   us a call (C entry, ten calls one after the other, the best of four such) with so many 64 tokens a segment, the one
//   taken in brackets:
//     bf16, 128 x 128: 2 x 2048 tokens of 16 heads 2: 57  [4]: 55  8: 63; 8192 of 32 heads 4: 152  [8]: 132  16: 147
//     16 x 1024 of 16 heads 4: 149  8: 127  [whole]: 104; 256 x 256, 4096 of 8 heads 4: 98  [8]: 90  16: 149
//     fp32, 128 x 128, 2048 of 8 heads [1]: 43  2: 44  4: 64; fp16, 64 x 100, 7 sequences, 4099 of 16 heads 1: 57  [2]: 54  4: 67
// The gradients take the same length: for 2 x 2048 tokens 124, with 8 117; for 2048 in fp32 108, with 2 104; else the least.
// Lengths of packed sequences are on the device.  The longest is taken for two and a half times the average, and
// 0.012 us for each workgroup that finds no segment.  A segment has at most 1024 tokens or four times the average, lest a
// long sequence among short ones be left to a workgroup a head (bf16, 128 x 128, 16 heads: one of 8192 amid 64 of 64
// tokens, whole 756, in segments 187; where all are short that costs, 300 of 64 tokens, 105 and 115).
int64_t la_segment_tokens(const atk_linear_attn_args* p) {
  const double cus = device_cu_count() > 0 ? device_cu_count() : 256, n = (double)(p->N > 0 ? p->N : 1);
  const double chunks = p->cu_seqlens ? (double)p->T / 64 / n : (double)((p->T + 63) / 64);
  const double longest = p->cu_seqlens ? chunks * (n < 2.5 ? n : 2.5) : chunks;
  const int da = la_padded(p->K), w = da <= 128 ? 128 : 64;
  const double type = (p->dtype == ATK_BF16 ? 1 : p->dtype == ATK_F16 ? 1.75 : 2.4) * (da <= 64 ? 0.65 : 1);
  const double work = (double)p->Hv * ((p->V + w - 1) / w) * n, states = (double)p->K * p->V * p->Hv * n * 16 / 4.4e6;
  const auto step = [&](double units, double half, double one, double two) {
    if (da > 128) return 0.75 * two * ceil(units / cus) * type;
    const double turns = units / (cus * (da <= 64 ? 3 : 2));
    return type * (units <= cus / 2 ? half : units <= cus ? one : turns <= 1 ? two : two * (ceil(turns) + turns) / 2);
  };
  const int64_t all = (p->T + 63) / 64 > 0 ? (p->T + 63) / 64 : 1;
  int64_t best = all;
  double least = chunks * step(work, 4, 5.8, 8);
  if (p->cu_seqlens) {
    const double slowest = longest * step(work < 2 * cus ? work : 2 * cus, 4, 5.8, 8);
    if (least < slowest) least = slowest;
  }
  for (int64_t per = 1; per < all && per <= 4096; per += per < 16 ? 1 : per / 8) {
    const double segs = ceil(chunks / (double)per);
    const double units = segs * work, full = units < 2 * cus ? units : 2 * cus, some = (double)per;
    double t = step(units, 5.5, 7, 10) * (some < chunks ? some : chunks) + (segs > 1 ? segs * states : 0) + 5;
    if (p->cu_seqlens) {
      const double slowest = step(full, 5.5, 7, 10) * (some < longest ? some : longest);
      t = (t > slowest ? t : slowest) + 0.012 * work * (chunks / some - (segs - 1));
    }
    if (t < least) {
      least = t;
      best = per;
    }
  }
  if (p->cu_seqlens) {
    const int64_t most = chunks > 4 ? (int64_t)(4 * chunks) : 16;
    if (best > most) best = most;
  }
  return best * 64;
}

// Checks a call and lays out its workspace; *rc says why where it is refused.
LaPlan la_plan(const atk_linear_attn_args* p, bool backward, LaArgs* a, int* rc) {
  LaPlan L = {};
  *rc = ATK_OK;
  if (!p) return *rc = fail(ATK_EINVAL, "linear attention: null arguments"), L;
  if (!dtype_ok(p->dtype) || !dtype_ok(p->g_dtype)) return *rc = fail(ATK_EINVAL, "linear attention: unknown dtype code"), L;
  if (!gdr_gate_ok(p->g_dtype, p->dtype))
    return *rc = fail(ATK_EINVAL, "linear attention: g must be of the inputs' type or fp32"), L;
  if (p->N < 0 || p->T < 0 || p->Hk <= 0 || p->Hv <= 0 || p->K <= 0 || p->V <= 0)
    return *rc = fail(ATK_EINVAL, "linear attention: bad sizes"), L;
  if (p->Hv % p->Hk) return *rc = fail(ATK_EINVAL, "linear attention: value heads must be a multiple of key heads"), L;
  const int vec = 16 / (int)dtype_size(p->dtype);
  if (p->K > kLaMaxK || p->K < vec || p->V < vec || p->V > (1 << 24) || p->Hv > 65535 || p->N > 65535 ||
      p->T >= ((int64_t)1 << 31) - 64)
    return *rc = fail(ATK_UNSUPPORTED, "linear attention: heads of fewer than 16 bytes or more than %d key columns, more than "
                      "65535 heads or sequences, or 2^31 tokens", kLaMaxK), L;
  const int64_t seg = la_segment_tokens(p);
  const double slots = p->cu_seqlens ? (double)(p->T / seg) + (double)p->N
                                     : (double)(p->T > seg ? (p->T + seg - 1) / seg : 1) * (double)p->N;
  if ((double)p->K * p->V >= (double)(1 << 29) || slots * p->Hv > 2147483000.0 || slots > 2147483000.0 || (p->cu_seqlens ? 1.0 : (double)p->N) * (double)p->T > 1e12)
    return *rc = fail(ATK_UNSUPPORTED, "linear attention: a state of 2^29 elements or more, or too many sequences and heads"), L;
  *a = LaArgs{};
  // the kernels' loads of 64 tokens have offsets of 32 bits; of one token there is no offset
  if (p->T > 1) for (const int64_t* st : {p->q_stride, p->k_stride, p->v_stride, p->g_stride})
    if (st[1] < 0 || st[1] >= (1 << 22)) return *rc = fail(ATK_UNSUPPORTED, "linear attention: tokens of 2^22 elements or more apart"), L;
  if ((int64_t)p->Hv * p->V >= (1 << 22) && backward) return *rc = fail(ATK_UNSUPPORTED, "linear attention backward: 2^22 value columns or more"), L;
  a->g = p->g; a->cu = p->cu_seqlens; a->n = (int)p->N; a->T = p->T; a->B = p->cu_seqlens ? 1 : p->N;
  for (int i = 0; i < 3; ++i) a->g_s[i] = p->g_stride[i];
  a->slots = (int)slots; a->seg = (int)seg;
  a->ends = p->cu_seqlens ? (int)((p->T + seg - 1) / seg) : a->slots;
  a->Hk = p->Hk; a->Hv = p->Hv; a->group = p->Hv / p->Hk; a->K = p->K; a->V = p->V;
  a->g_dtype = p->g_dtype; a->fixed = p->fixed_decay; a->scale = p->scale;
  a->by_hk = make_fastdiv((uint32_t)p->Hk); a->by_hv = make_fastdiv((uint32_t)p->Hv); a->by_seg = make_fastdiv((uint32_t)seg);
  a->by_segs = make_fastdiv((uint32_t)(p->T > seg ? (p->T + seg - 1) / seg : 1));
  L.split = p->T > seg;
  char* w = static_cast<char*>(p->workspace);
  auto take = [&](size_t floats) {
    float* q = w ? reinterpret_cast<float*>(w + L.bytes) : nullptr;
    L.bytes += (floats * 4 + 15) / 16 * 16;
    return q;
  };
  const size_t state = (size_t)a->ends * a->Hv * a->K * a->V, tokens = (size_t)a->B * a->T;
  if (L.split) {
    L.s_fwd = take(state);
    L.decays = take((size_t)a->ends * a->Hv * (backward ? 2 : 1));
    if (backward) L.s_rev = take(state);
  }
  if (backward) {
    const int da = la_padded(a->V);
    L.a_tiles = (a->V + da - 1) / da;
    const int w = 64 * la_wide(*a, da, a->K, 3);
    L.k_tiles = (a->K + w - 1) / w;
    L.n_parts = a->group * L.a_tiles;
    if (L.n_parts > 1)
      for (int i = 0; i < 2; ++i) L.parts[i] = take((size_t)L.n_parts * tokens * a->Hk * a->K);
    for (int i = 0; i < 2; ++i) L.dots[i] = take((size_t)L.a_tiles * L.k_tiles * a->Hv * tokens);
    L.x = take((size_t)L.a_tiles * L.k_tiles * a->slots * a->Hv);
    if (a->fixed) L.seg_sums = take((size_t)a->slots * a->Hv);
  }
  return L;
}

void la_copy3(int64_t (&to)[3], const int64_t* from) {
  for (int i = 0; i < 3; ++i) to[i] = from[i];
}

int la_scan(const LaArgs& a, float* s0, float* s1, const float* decays, int roles, hipStream_t s) {
  const int64_t kv = (int64_t)a.K * a.V;
  bool vec = kv % 4 == 0;
  for (int i = 0; i < roles; ++i) vec = vec && aligned16(a.role[i].s_first);
  int64_t per = (kv + (vec ? 1023 : 255)) / (vec ? 1024 : 256);
  const int marks = a.cu && a.ends < a.n ? a.ends : 0;
  const int64_t units = (int64_t)(marks ? marks : a.n) * a.Hv;
  // most sequences of many have one segment: fewer workgroups that find that out
  if (a.cu && units * per > 8192) per = 8192 / units > 0 ? 8192 / units : 1;
  const int64_t most = kLaBlocks / per > 0 ? kLaBlocks / per : 1;
  for (int64_t u = 0; u < units; u += most) {
    const dim3 g((unsigned)((units - u < most ? units - u : most) * per), (unsigned)roles);
    if (vec) hipLaunchKernelGGL((la_scan_kernel<4>), g, dim3(256), 0, s, a, s0, s1, decays, make_fastdiv((uint32_t)per), (int)u, marks);
    else hipLaunchKernelGGL((la_scan_kernel<1>), g, dim3(256), 0, s, a, s0, s1, decays, make_fastdiv((uint32_t)per), (int)u, marks);
    if (int rc = check_launch("la_scan_kernel")) return rc;
  }
  return ATK_OK;
}

template <typename T>
int la_forward(const atk_linear_attn_args* p, LaArgs& a, const LaPlan& L, hipStream_t s) {
  LaRole& r = a.role[0];
  r = LaRole{};
  r.a = p->q; r.b = p->k; r.c = p->v;
  la_copy3(r.a_s, p->q_stride); la_copy3(r.b_s, p->k_stride); la_copy3(r.c_s, p->v_stride);
  r.AD = a.K; r.CD = a.V; r.a_tiles = 1;
  r.s_first = static_cast<const float*>(p->initial_state); r.s_last = static_cast<float*>(p->final_state);
  r.out = p->out;
  if (L.split) {
    r.s_between = L.s_fwd;
    float* to[1] = {L.s_fwd};
    if (int rc = la_launch_states<T>(a, 1, to, L.decays, s)) return rc;
    if (int rc = la_scan(a, L.s_fwd, nullptr, L.decays, 1, s)) return rc;
  }
  return la_launch_out<T>(a, s);
}

template <typename T, typename G>
int la_gates(const LaArgs& a, const LaPlan& L, void* dg, hipStream_t s) {
  LaGateArgs b = {L.dots[0], L.dots[1], L.x, dg, L.seg_sums, L.a_tiles * L.k_tiles, 0};
  const int64_t units = (int64_t)a.slots * a.Hv;
  for (int64_t u = 0; u < units; u += (int64_t)kLaBlocks * 4) {
    b.unit0 = (uint32_t)u;
    const int64_t blocks = (units - u + 3) / 4;
    hipLaunchKernelGGL((la_gate_kernel<G>), dim3((unsigned)(blocks < kLaBlocks ? blocks : kLaBlocks)), dim3(256), 0, s, a, b);
    if (int rc = check_launch("la_gate_kernel")) return rc;
  }
  if (!a.fixed) return ATK_OK;
  hipLaunchKernelGGL((la_gate_sum_kernel<G>), dim3((unsigned)a.Hv), dim3(256), 0, s, L.seg_sums, static_cast<G*>(dg), a.slots);
  return check_launch("la_gate_sum_kernel");
}

template <typename T>
int la_backward(const atk_linear_attn_args* p, LaArgs& a, const LaPlan& L, const void* dout, const float* ds1, void* dq,
                void* dk, void* dv, void* dg, float* ds0, hipStream_t s) {
  const int64_t vs[3] = {a.T * a.Hv * a.V, (int64_t)a.Hv * a.V, a.V};  // dout's strides
  LaArgs b = a;  // states of segments: k, v forward and q, dO in reverse, which is also dv's (k, q, dO)
  LaRole& f = b.role[0];
  LaRole& v = b.role[1];
  f = v = LaRole{};
  f.b = p->k; f.c = p->v;
  la_copy3(f.b_s, p->k_stride); la_copy3(f.c_s, p->v_stride);
  v.a = p->k; v.b = p->q; v.c = dout; v.out = dv;
  la_copy3(v.a_s, p->k_stride); la_copy3(v.b_s, p->q_stride); la_copy3(v.c_s, vs);
  f.AD = v.AD = a.K; f.CD = v.CD = a.V; v.a_tiles = 1;
  f.s_first = static_cast<const float*>(p->initial_state);
  v.s_first = ds1; v.s_between = L.s_rev; v.s_last = ds0;
  if (L.split) {
    float* to[2] = {L.s_fwd, L.s_rev};
    if (int rc = la_launch_states<T>(b, 2, to, L.decays, s)) return rc;
    if (int rc = la_scan(b, L.s_fwd, L.s_rev, L.decays, 2, s)) return rc;
  }
  LaRole& q = a.role[0];
  LaRole& k = a.role[1];
  q = k = LaRole{};
  q.a = dout; q.b = p->v; q.c = p->k; q.e = p->q; q.out = dq;
  la_copy3(q.a_s, vs); la_copy3(q.b_s, p->v_stride); la_copy3(q.c_s, p->k_stride); la_copy3(q.e_s, p->q_stride);
  k.a = p->v; k.b = dout; k.c = p->q; k.e = p->k; k.out = dk;
  la_copy3(k.a_s, p->v_stride); la_copy3(k.b_s, vs); la_copy3(k.c_s, p->q_stride); la_copy3(k.e_s, p->k_stride);
  q.AD = k.AD = a.V; q.CD = k.CD = a.K;
  q.a_tiles = k.a_tiles = L.a_tiles;
  q.s_first = f.s_first; q.s_between = L.s_fwd;
  k.s_first = ds1; k.s_between = L.s_rev;
  q.parts = L.parts[0]; k.parts = L.parts[1];
  q.dots = L.dots[0]; k.dots = L.dots[1];
  q.x_last = ds1; q.x_between = L.s_rev; q.x_out = L.x;
  a.role[2] = v;
  if (int rc = la_launch_grads<T>(a, dg != nullptr, s)) return rc;
  if (L.n_parts > 1 && a.T > 0) {
    LaSumArgs m = {{L.parts[0], L.parts[1]}, {dq, dk}, a.B * a.T * a.Hk * (int64_t)a.K, L.n_parts};
    const bool vec = m.count % 4 == 0;
    int64_t blocks = (m.count + (vec ? 1023 : 255)) / (vec ? 1024 : 256);
    blocks = blocks < 16384 ? blocks : 16384;
    const dim3 g((unsigned)blocks, 2);
    if (vec) hipLaunchKernelGGL((la_sum_kernel<T, 4>), g, dim3(256), 0, s, m);
    else hipLaunchKernelGGL((la_sum_kernel<T, 1>), g, dim3(256), 0, s, m);
    if (int rc = check_launch("la_sum_kernel")) return rc;
  }
  if (!dg) return ATK_OK;
  return a.g_dtype == ATK_F32 ? la_gates<T, float>(a, L, dg, s) : la_gates<T, T>(a, L, dg, s);
}

}  // namespace
}  // namespace atk

extern "C" int atk_linear_attn_update(const atk_linear_attn_update_args* p) {
  using namespace atk;
  if (!p) return fail(ATK_EINVAL, "linear attention update: null arguments");
  if (!dtype_ok(p->dtype) || !dtype_ok(p->g_dtype)) return fail(ATK_EINVAL, "linear attention update: unknown dtype code");
  if (!gdr_gate_ok(p->g_dtype, p->dtype))
    return fail(ATK_EINVAL, "linear attention update: g must be of the inputs' type or fp32");
  if (p->N < 0 || p->slots < 0 || p->Hk <= 0 || p->Hv <= 0 || p->K <= 0 || p->V <= 0)
    return fail(ATK_EINVAL, "linear attention update: bad sizes");
  if (p->Hv % p->Hk) return fail(ATK_EINVAL, "linear attention update: value heads must be a multiple of key heads");
  if (p->K > kLaMaxK || p->Hv > 65535 || p->N > 65535 || p->V > (1 << 24))
    return fail(ATK_UNSUPPORTED, "linear attention update: more than %d key columns, or more than 65535 heads or sequences", kLaMaxK);
  if (p->N == 0) return ATK_OK;
  // (a cache of no slots has no memory; every sequence is padding then)
  if (!p->q || !p->k || !p->v || !p->g || (!p->state && p->slots > 0) || !p->out)
    return fail(ATK_EINVAL, "linear attention update: null pointer");
  if (!p->state_indices && p->slots < p->N) return fail(ATK_EINVAL, "linear attention update: fewer slots than sequences");
  LaStepArgs a = {};
  a.q = p->q; a.k = p->k; a.v = p->v; a.g = p->g;
  a.state = static_cast<float*>(p->state); a.o = p->out; a.slots = p->state_indices;
  a.n = p->N; a.n_slots = p->slots; a.state_stride = p->state_stride;
  a.q_sb = p->q_stride_n; a.q_sh = p->q_stride_h; a.k_sb = p->k_stride_n; a.k_sh = p->k_stride_h;
  a.v_sb = p->v_stride_n; a.v_sh = p->v_stride_h; a.g_sb = p->g_stride_n; a.g_sh = p->g_stride_h;
  a.Hv = p->Hv; a.group = p->Hv / p->Hk; a.K = p->K; a.V = p->V; a.g_dtype = p->g_dtype; a.scale = p->scale;
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  // a launch has fewer than 2^32 threads: so many sequences at a time
  const int64_t blocks = (int64_t)((a.V + 31) / 32) * a.Hv, most = kLaBlocks / blocks > 0 ? kLaBlocks / blocks : 1;
  for (int64_t n = 0; n < p->N; n += most) {
    LaStepArgs b = a;
    const size_t e = dtype_size(p->dtype);
    b.n = p->N - n < most ? p->N - n : most;
    b.q = static_cast<const char*>(a.q) + n * a.q_sb * (int64_t)e;
    b.k = static_cast<const char*>(a.k) + n * a.k_sb * (int64_t)e;
    b.v = static_cast<const char*>(a.v) + n * a.v_sb * (int64_t)e;
    b.g = static_cast<const char*>(a.g) + n * a.g_sb * (int64_t)dtype_size(p->g_dtype);
    b.o = static_cast<char*>(a.o) + n * a.Hv * a.V * (int64_t)e;
    if (a.slots) b.slots = a.slots + n;
    else {
      b.state = a.state + n * a.state_stride;
      b.n_slots = a.n_slots - n;
    }
    if (p->dtype == ATK_F32) launch_step_typed<float>(b, s);
    else if (p->dtype == ATK_F16) launch_step_typed<_Float16>(b, s);
    else launch_step_typed<__bf16>(b, s);
    if (int rc = check_launch("la_step_kernel")) return rc;
  }
  return ATK_OK;
}

extern "C" size_t atk_linear_attn_workspace_bytes(const atk_linear_attn_args* p) {
  atk::LaArgs a;
  int rc;
  return atk::la_plan(p, false, &a, &rc).bytes;
}

extern "C" int atk_linear_attn_fwd(const atk_linear_attn_args* p) {
  using namespace atk;
  LaArgs a;
  int rc;
  const LaPlan L = la_plan(p, false, &a, &rc);
  if (rc) return rc;
  if (p->N == 0 || (p->T == 0 && !p->final_state)) return ATK_OK;
  if (p->T > 0 && (!p->q || !p->k || !p->v || !p->g || !p->out)) return fail(ATK_EINVAL, "linear attention: null pointer");
  if (L.bytes && (!p->workspace || p->workspace_bytes < L.bytes || !aligned16(p->workspace)))
    return fail(ATK_EINVAL, "linear attention: workspace too small or not 16-byte aligned");
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  if (p->dtype == ATK_F32) return la_forward<float>(p, a, L, s);
  if (p->dtype == ATK_F16) return la_forward<_Float16>(p, a, L, s);
  return la_forward<__bf16>(p, a, L, s);
}

extern "C" size_t atk_linear_attn_bwd_workspace_bytes(const atk_linear_attn_args* p) {
  atk::LaArgs a;
  int rc;
  return atk::la_plan(p, true, &a, &rc).bytes;
}

extern "C" int atk_linear_attn_bwd(const atk_linear_attn_args* p, const void* dout, const void* dfinal_state, void* dq, void* dk,
                                   void* dv, void* dg, void* dinitial_state) {
  using namespace atk;
  LaArgs a;
  int rc;
  const LaPlan L = la_plan(p, true, &a, &rc);
  if (rc) return rc;
  if (p->N == 0) return ATK_OK;
  if (p->T > 0 && (!p->q || !p->k || !p->v || !p->g || !dout || !dq || !dk || !dv))
    return fail(ATK_EINVAL, "linear attention backward: null pointer");
  if (L.bytes && (!p->workspace || p->workspace_bytes < L.bytes || !aligned16(p->workspace)))
    return fail(ATK_EINVAL, "linear attention backward: workspace too small or not 16-byte aligned");
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  const float* ds1 = static_cast<const float*>(dfinal_state);
  float* ds0 = static_cast<float*>(dinitial_state);
  if (p->dtype == ATK_F32) return la_backward<float>(p, a, L, dout, ds1, dq, dk, dv, dg, ds0, s);
  if (p->dtype == ATK_F16) return la_backward<_Float16>(p, a, L, dout, ds1, dq, dk, dv, dg, ds0, s);
  return la_backward<__bf16>(p, a, L, dout, ds1, dq, dk, dv, dg, ds0, s);
}

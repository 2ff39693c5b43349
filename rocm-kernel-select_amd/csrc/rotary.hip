// Rotary positions: pairs of columns of each query and key turned by an angle of their token's position.
//
//   (a, b) -> scale (a cos - b sin, a sin + b cos),  angle = position * inv_freq[i], i < rot / 2
// Pair i is columns i and i + rot / 2 (halves) or 2 i and 2 i + 1 (interleaved); columns from rot on are
// copied.  The way back, the gradient, is the same by the opposite angle.
//
// HBM-bound: every element is read once and written once.  The angles are products in 64 bits, with what their
// rounding leaves, brought to a part of a turn there (a position of 10^6 has an error of 0.06 in an fp32 product, one
// of 2^40 7e-5 in a product rounded to 64 bits), and sine and cosine are taken once for each token and pair by a
// workgroup that has all heads of its tokens: the table lies in LDS while they stream through.  8192 tokens of 32 and 16 heads of 128 columns, bf16: 43 us for
// 201 MB, 4.7 TB/s (a large copy reaches 5.05); 64 single tokens 3.5 us, a launch's own time.
#include "atk_common.h"

namespace atk {
namespace {

struct RotaryArgs {
  const void* x[2]; void* y[2];                    // queries and keys
  int64_t sb[2], st[2], sh[2];                     // strides in elements: batch, token, head
  const void* pos; const void* freq;
  int64_t pos_sb, pos_st, offset, rows;            // rows: batch * tokens
  FastDiv T;                                       // tokens of a batch element
  int H[2], D, R, pos64, freq64, interleaved, inverse;
  int tokens;                                      // of a workgroup
  float scale;
};

template <typename T, int V>
struct Pack {
  T e[V];
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) {
  Pack<T, V> r;
  __builtin_memcpy(r.e, p, V * sizeof(T));  // element alignment only
  return r;
}

// position * freq in turns, without whole ones: within 2^-40 of a turn for any position and freq up to 1, 2^-52 of the
// turns of nearer ones.  The position's last 11 bits are apart, so the rest has no rounding in 64 bits; products keep what
// theirs leaves, and 1 / (2 pi) has 107 bits.  (Contracted, a product would be taken with that twice.)
__device__ __forceinline__ double part_of_turn(int64_t pos, double freq) {
#pragma clang fp contract(off)
  constexpr double kTurn = 0.15915494309189535, kTurnRest = -9.839338337591243e-18;
  const int64_t low = pos & 2047;
  const double high = (double)(pos - low), p = high * freq, rest = fma(high, freq, -p) + (double)low * freq;
  const double turns = p * kTurn, left = fma(p, kTurn, -turns) + (p * kTurnRest + rest * kTurn);
  const double part = (turns - rint(turns)) + left;
  return part - rint(part);
}

// V: columns of a vector of pairs (of halves: V of each), CV of one that is copied.  An item is a vector of
// a head: pairs first, then columns to copy.  The last of either ends where they end, so it may repeat some
// columns of the one before it, with the same values.
template <typename T, int V, int CV, bool INTER>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a, int64_t first) {
  extern __shared__ float table[];  // [tokens][2][R]: cosines, sines
  constexpr int PV = INTER ? V / 2 : V;  // pairs of a vector
  const int64_t row0 = first + (int64_t)blockIdx.x * a.tokens;
  const int tokens = (int)(a.rows - row0 < a.tokens ? a.rows - row0 : a.tokens);
  for (int i = threadIdx.x; i < tokens * a.R; i += 256) {
    const int k = i / a.R, j = i - k * a.R;
    const int64_t row = row0 + k;
    const uint32_t b = fdiv((uint32_t)row, a.T);
    const int64_t t = row - (int64_t)b * a.T.d;
    int64_t pos = a.offset + t;
    if (a.pos) {
      const int64_t at = b * a.pos_sb + t * a.pos_st;
      pos = a.pos64 ? static_cast<const int64_t*>(a.pos)[at] : (int64_t)static_cast<const int*>(a.pos)[at];
    }
    const double f = a.freq64 ? static_cast<const double*>(a.freq)[j] : (double)static_cast<const float*>(a.freq)[j];
    // (an angle rounded to fp32 is off by up to 2^-23.3, and what comes of it by more than the fp32 products that follow)
    double s, c;
    sincospi(2. * part_of_turn(pos, f), &s, &c);
    table[k * 2 * a.R + j] = (float)(a.scale * c);
    table[k * 2 * a.R + a.R + j] = (float)(a.scale * (a.inverse ? -s : s));
  }
  __syncthreads();
  const int rot = 2 * a.R, rest = a.D - rot;
  const int nv = (a.R + PV - 1) / PV, nc = (rest + CV - 1) / CV, n = nv + nc, heads = a.H[0] + a.H[1];
  for (int i = threadIdx.x; i < tokens * heads * n; i += 256) {
    const int u = i / n, k = u / heads;
    int j = i - u * n, h = u - k * heads;
    const int64_t row = row0 + k;
    const uint32_t b = fdiv((uint32_t)row, a.T);
    const int64_t t = row - (int64_t)b * a.T.d;
    const int key = h >= a.H[0];
    if (key) h -= a.H[0];
    const T* __restrict__ x = static_cast<const T*>(a.x[key]) + (int64_t)b * a.sb[key] + t * a.st[key] + h * a.sh[key];
    T* __restrict__ y = static_cast<T*>(a.y[key]) + (row * a.H[key] + h) * a.D;
    if (j >= nv) {
      j = (j - nv) * CV;
      j = rot + (j + CV <= rest ? j : rest - CV);
      const Pack<T, CV> p = load_pack<T, CV>(x + j);
      __builtin_memcpy(y + j, p.e, CV * sizeof(T));
      continue;
    }
    j = j * PV + PV <= a.R ? j * PV : a.R - PV;
    const float* __restrict__ c = table + k * 2 * a.R + j;
    const float* __restrict__ s = c + a.R;
    if constexpr (INTER) {
      Pack<T, V> p = load_pack<T, V>(x + 2 * j);
#pragma unroll
      for (int e = 0; e < PV; ++e) {
        const float u0 = to_f32(p.e[2 * e]), u1 = to_f32(p.e[2 * e + 1]);
        p.e[2 * e] = from_f32<T>(u0 * c[e] - u1 * s[e]);
        p.e[2 * e + 1] = from_f32<T>(u0 * s[e] + u1 * c[e]);
      }
      __builtin_memcpy(y + 2 * j, p.e, V * sizeof(T));
    } else {
      Pack<T, V> p = load_pack<T, V>(x + j), q = load_pack<T, V>(x + a.R + j);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float u0 = to_f32(p.e[e]), u1 = to_f32(q.e[e]);
        p.e[e] = from_f32<T>(u0 * c[e] - u1 * s[e]);
        q.e[e] = from_f32<T>(u0 * s[e] + u1 * c[e]);
      }
      __builtin_memcpy(y + j, p.e, V * sizeof(T));
      __builtin_memcpy(y + a.R + j, q.e, V * sizeof(T));
    }
  }
}

template <typename T>
int launch_rotary(RotaryArgs a, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const int rest = a.D - 2 * a.R;
  const bool wide = (a.R == 0 || (a.interleaved ? 2 * a.R : a.R) >= V) && (rest == 0 || rest >= V);
  const int items = (a.H[0] + a.H[1]) * ((a.D + V - 1) / V);
  // Tokens of a workgroup: enough for two vectors a thread, within 32 KB of tables.
  const int64_t cus = device_cu_count() > 0 ? device_cu_count() : 256;
  int tokens = 1;
  while (tokens * items < 512 && a.rows > 4 * cus * tokens && tokens * 2 * a.R * 8 <= 32768) tokens *= 2;
  a.tokens = tokens;
  const size_t lds = (size_t)tokens * 2 * a.R * sizeof(float);
  const int64_t most = (int64_t)tokens << 23;  // (a launch has fewer than 2^32 threads)
  for (int64_t first = 0; first < a.rows; first += most) {
    const int64_t rows = a.rows - first < most ? a.rows - first : most;
    const dim3 g((unsigned)((rows + tokens - 1) / tokens)), b(256);
    if (a.interleaved && wide) hipLaunchKernelGGL((rotary_kernel<T, V, V, true>), g, b, lds, s, a, first);
    else if (a.interleaved) hipLaunchKernelGGL((rotary_kernel<T, 2, 1, true>), g, b, lds, s, a, first);
    else if (wide) hipLaunchKernelGGL((rotary_kernel<T, V, V, false>), g, b, lds, s, a, first);
    else hipLaunchKernelGGL((rotary_kernel<T, 1, 1, false>), g, b, lds, s, a, first);
    if (int rc = check_launch("rotary_kernel")) return rc;
  }
  return ATK_OK;
}

}  // namespace
}  // namespace atk

extern "C" int atk_rotary(const atk_rotary_args* p) {
  using namespace atk;
  if (!p) return fail(ATK_EINVAL, "rotary: null arguments");
  if (!dtype_ok(p->dtype)) return fail(ATK_EINVAL, "rotary: unknown dtype code %d", p->dtype);
  if (p->N < 0 || p->T < 0 || p->Hq < 0 || p->Hk < 0 || p->D < 0 || p->rot < 0 || p->rot % 2 || p->rot > p->D)
    return fail(ATK_EINVAL, "rotary: bad sizes");
  if (p->D > 4096 || p->Hq > 65535 || p->Hk > 65535 || (double)p->N * (double)p->T > 2147483647.0)
    return fail(ATK_UNSUPPORTED, "rotary: heads of more than 4096 columns, more than 65535 heads, or 2^31 tokens");
  const int64_t rows = p->N * p->T;
  if (rows == 0 || p->D == 0 || p->Hq + p->Hk == 0) return ATK_OK;
  if ((p->Hq && (!p->q || !p->q_out)) || (p->Hk && (!p->k || !p->k_out)) || (p->rot && !p->inv_freq))
    return fail(ATK_EINVAL, "rotary: null pointer");
  RotaryArgs a = {};
  a.x[0] = p->q; a.x[1] = p->k; a.y[0] = p->q_out; a.y[1] = p->k_out;
  for (int i = 0; i < 2; ++i) {
    const int64_t* st = i ? p->k_stride : p->q_stride;
    a.sb[i] = st[0]; a.st[i] = st[1]; a.sh[i] = st[2];
  }
  a.pos = p->positions; a.freq = p->inv_freq;
  a.pos_sb = p->pos_stride[0]; a.pos_st = p->pos_stride[1]; a.offset = p->offset; a.rows = rows;
  a.T = make_fastdiv((uint32_t)p->T);
  a.H[0] = p->Hq; a.H[1] = p->Hk; a.D = p->D; a.R = p->rot / 2;
  a.pos64 = p->pos64; a.freq64 = p->freq64; a.interleaved = p->interleaved; a.inverse = p->inverse; a.scale = p->scale;
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  if (p->dtype == ATK_F32) return launch_rotary<float>(a, s);
  if (p->dtype == ATK_F16) return launch_rotary<_Float16>(a, s);
  return launch_rotary<__bf16>(a, s);
}

// Gradients of the gated delta rule over whole sequences.
//
// With the names of the forward (per chunk: S the state before it, e the errors, U = beta e, P =
// lower(Q K^T * D), T = (1 + diag(beta) W)^-1, E = exp(G_63 - G)) and dS' the gradient of the state
// after the chunk:
//   dU = scale P^T dO + E (K dS');   dR = T^T dU           the gradients of u_t, all paths together
//   dS = exp(G_63) dS' + Q^T (scale exp(G) dO) - K^T (beta exp(G) dR)
// which only passes dS' on: a chain from the last chunk to the first, like the forward's and with no
// need of S or e.  The forward's chain is run again beside it for those (nothing of a chunk is kept
// from the forward).  Everything else is one chunk's alone:
//   dV = beta dR;  dbeta_i = dR_i . e_i
//   N = scale lower(dO U^T * D);   M = -diag(beta) strictlower(dR U^T * D)
//   dQ = N K + scale exp(G) dO S^T
//   dK = [M K - beta exp(G) dR S^T] + [M^T K + N^T Q + (E U) dS'^T]      (k_t read, and written)
//   dG_i = q_i . dq_i + k_i . (read part - written part)_i, and for the chunk's last token also
//          exp(G_63) <S, dS'> + sum_j k_j . ((E U) dS'^T)_j;   dg = sums of dG from the chunk's end
// Key heads that several value heads share get the sum over them in a fixed order: one workgroup has
// a key head's whole group.
#include "gated_delta.h"

namespace atk {
namespace {

constexpr int LD = 68;

// The chain of dS'.  Distribution as in the forward's chain.
template <typename T, int KP>
__global__ __launch_bounds__(256) void gdr_bwd_chain_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32, MT = KP / 64, BV = 16;
  constexpr int SP = KP + 8, UP = 64 + 8;
  // 8 of 32 rows in gdr_at's order
  auto frag = [](const __bf16* p, int g) {
    const uint2 lo = *reinterpret_cast<const uint2*>(p + 4 * g), hi = *reinterpret_cast<const uint2*>(p + 16 + 4 * g);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  __shared__ __align__(16) __bf16 sl[3][BV][SP], dl[NP][BV][UP], gl[3][BV][UP], ul[3][BV][UP], rl[3][BV][UP];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
  const int h = blockIdx.y, hk = h / a.group;
  const int64_t n = blockIdx.z;
  const int col = blockIdx.x * BV + c;
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  f32x4 S[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = 16 * (wave * MT + m) + 4 * g + r;
      S[m][r] = a.ds1 && row < a.K && col < a.V ? a.ds1[((n * a.Hv + h) * a.K + row) * a.V + col] : 0.f;
    }
  auto put_state = [&]() {
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      bf16x4 parts[3];
      const float x[4] = {S[m][0], S[m][1], S[m][2], S[m][3]};
      split_parts<3, 4>(x, parts);
#pragma unroll
      for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x4*>(&sl[p][c][16 * (wave * MT + m) + 4 * g]) = parts[p];
    }
  };
  auto put_rows = [&](const float* x, auto& to) {  // this lane's 4 tokens of one column
    constexpr int P = sizeof(to) / sizeof(to[0]);
    bf16x4 parts[P];
    split_parts<P, 4>(x, parts);
#pragma unroll
    for (int p = 0; p < P; ++p) *reinterpret_cast<bf16x4*>(&to[p][c][16 * wave + 4 * g]) = parts[p];
  };
  put_state();
  const int64_t chunks = (seq.len + kGdrC - 1) / kGdrC;
  for (int64_t ch = chunks - 1; ch >= 0; --ch) {
    const int64_t slot = seq.slot + ch;
    const int64_t left = seq.len - ch * kGdrC;
    const int rows = (int)(left < kGdrC ? left : kGdrC);
    const int64_t t0 = seq.begin + ch * kGdrC;
    const int64_t kbase = (hk * a.slots + slot) * (int64_t)(KS * 4 * NP * 64);
    const int64_t tbase = (h * a.slots + slot) * (int64_t)(kTri * 3 * 64);
    const float* __restrict__ row = a.row + (h * a.slots + slot) * 192;
    const float all = row[63];
    float rest[4], bg[4], x[4], y[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wave + 4 * g + r;
      const float grown = row[i];
      rest[r] = row[64 + i];
      bg[r] = -row[128 + i] * grown;
      x[r] = i < rows && col < a.V
                 ? to_f32(static_cast<const T*>(a.dout)[((seq.batch * a.T + t0 + i) * a.Hv + h) * (int64_t)a.V + col])
                 : 0.f;
      y[r] = a.scale * grown * x[r];
    }
    put_rows(x, dl);
    put_rows(y, gl);
    __syncthreads();
    float* __restrict__ dsc = a.dsc + (h * a.slots + slot) * (int64_t)KP * a.VP;
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) dsc[(int64_t)(16 * (wave * MT + m) + 4 * g + r) * a.VP + col] = S[m][r];
    f32x4 ks = {0.f, 0.f, 0.f, 0.f}, pd = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      uint4 ka[NP], b[3];
#pragma unroll
      for (int p = 0; p < NP; ++p) ka[p] = a.kf[kbase + ((s * 4 + wave) * NP + p) * 64 + lane];
#pragma unroll
      for (int p = 0; p < 3; ++p) b[p] = frag(&sl[p][c][32 * s], g);
      ks = mma_parts<NP, 3>(ka, b, ks);
    }
    for (int s = wave >> 1; s < 2; ++s) {
      uint4 pa[3], b[NP];
#pragma unroll
      for (int p = 0; p < 3; ++p) pa[p] = a.ptf[tbase + (tri_upper(wave, s) * 3 + p) * 64 + lane];
#pragma unroll
      for (int p = 0; p < NP; ++p) b[p] = frag(&dl[p][c][32 * s], g);
      pd = mma_parts<3, NP>(pa, b, pd);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) x[r] = a.scale * pd[r] + rest[r] * ks[r];
    put_rows(x, ul);
    __syncthreads();
    f32x4 dr = {0.f, 0.f, 0.f, 0.f};
    for (int s = wave >> 1; s < 2; ++s) {
      uint4 ta[3], b[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) ta[p] = a.ttf[tbase + (tri_upper(wave, s) * 3 + p) * 64 + lane];
#pragma unroll
      for (int p = 0; p < 3; ++p) b[p] = frag(&ul[p][c][32 * s], g);
      dr = mma_parts<3, 3>(ta, b, dr);
    }
    float* __restrict__ drc = a.drc + (h * a.slots + slot) * (int64_t)64 * a.VP;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      drc[(int64_t)(16 * wave + 4 * g + r) * a.VP + col] = dr[r];
      x[r] = bg[r] * dr[r];
    }
    put_rows(x, rl);
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) S[m] *= all;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      uint4 bq[3], bk[3];
#pragma unroll
      for (int p = 0; p < 3; ++p) {
        bq[p] = frag(&gl[p][c][32 * s], g);
        bk[p] = frag(&rl[p][c][32 * s], g);
      }
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        uint4 qa[NP], ka[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          qa[p] = a.qtf[kbase + (((wave * MT + m) * 2 + s) * NP + p) * 64 + lane];
          ka[p] = a.ktf[kbase + (((wave * MT + m) * 2 + s) * NP + p) * 64 + lane];
        }
        S[m] = mma_parts<NP, 3>(qa, bq, S[m]);
        S[m] = mma_parts<NP, 3>(ka, bk, S[m]);
      }
    }
    put_state();  // read after the next chunk's first barrier; its last readers are two barriers back
    __syncthreads();
  }
  if (a.ds0) {
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = 16 * (wave * MT + m) + 4 * g + r;
        if (row < a.K && col < a.V) a.ds0[((n * a.Hv + h) * a.K + row) * a.V + col] = S[m][r];
      }
  }
}

__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == ATK_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == ATK_F16) static_cast<_Float16*>(p)[i] = from_f32<_Float16>(v);
  else static_cast<__bf16*>(p)[i] = from_f32<__bf16>(v);
}

// (row, column) tile t of the ten of a lower triangle of 16 x 16 tiles
__device__ __forceinline__ void tri_tile(int t, int* i, int* j) {
  *i = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
  *j = t - *i * (*i + 1) / 2;
}

// What one chunk's gradients need of that chunk, for one key head and all of its value heads.  Wave w
// has key columns w KP / 4 .. of dq and dk for all 64 tokens.  The value columns are walked 32 at a
// time: the waves bring 16 tokens each of dO, dR and e into LDS as fragments, and every wave
// multiplies all of them with its own rows of S and dS', which it splits itself.
template <typename T, int KP>
__global__ __launch_bounds__(256) void gdr_grads_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32, NT = KP / 64;
  constexpr int STAGE = 4 * (NP + 6) * 64;                       // fragments of 32 value columns
  constexpr int FRAGS = 2 * kTri * 3 * 64;                       // a triangle's and its transpose's
  __shared__ uint4 fr[STAGE > FRAGS ? STAGE : FRAGS];
  __shared__ __align__(16) float nm[64 * LD], mm[64 * LD];
  __shared__ float2 gs[64];
  __shared__ float grown[64], rest[64], beta[64], dg_part[4][64], dots[4];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
  const int64_t slot = blockIdx.x;
  const int hk = blockIdx.y;
  const int64_t n = gdr_seq_of_slot(a.cu, a.T, a.n, slot);
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t at = (slot - seq.slot) * kGdrC;
  if (at < 0 || at >= seq.len) return;
  const int rows = (int)(seq.len - at < kGdrC ? seq.len - at : kGdrC);
  const int64_t t0 = seq.begin + at, token = seq.batch * a.T + t0;
  const int64_t kbase = (hk * a.slots + slot) * (int64_t)(KS * 4 * NP * 64);
  const T* __restrict__ qp = static_cast<const T*>(a.q) + seq.batch * a.q_s[0] + t0 * a.q_s[1] + hk * a.q_s[2];
  const T* __restrict__ kp = static_cast<const T*>(a.k) + seq.batch * a.k_s[0] + t0 * a.k_s[1] + hk * a.k_s[2];
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  f32x4 dqs[4][NT], dks[4][NT];  // sums over the group
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) dqs[m][t] = dks[m][t] = zero;
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    const int64_t hs = h * a.slots + slot;
    const float* __restrict__ sc = a.sc + hs * KP * a.VP;
    const float* __restrict__ dsc = a.dsc + hs * KP * a.VP;
    const float* __restrict__ ec = a.ec + hs * 64 * a.VP;
    const float* __restrict__ drc = a.drc + hs * 64 * a.VP;
    if (tid < 64) {
      gs[tid] = a.gsum[hs * 64 + tid];
      grown[tid] = a.row[hs * 192 + tid];
      rest[tid] = a.row[hs * 192 + 64 + tid];
      beta[tid] = a.row[hs * 192 + 128 + tid];
    }
    f32x4 dq[4][NT], dr[4][NT], dw[4][NT];  // dq, and dk as it is read and as it is written
    f32x4 ne[3], me[3];                     // dO e^T and dR e^T, tiles wave, wave + 4, wave + 8 of the ten
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t) dq[m][t] = dr[m][t] = dw[m][t] = zero;
#pragma unroll
    for (int t = 0; t < 3; ++t) ne[t] = me[t] = zero;
    float dot = 0.f;  // <S, dS'>
    for (int v0 = 0; v0 < a.VP; v0 += 32) {
      __syncthreads();  // fr's readers are past it
      {
        const int i = 16 * wave + c, col = v0 + 8 * g;  // a token, 8 columns
        float x[8];
        bf16x8 parts[3];
        const T* __restrict__ d = static_cast<const T*>(a.dout) + ((token + (i < rows ? i : 0)) * a.Hv + h) * (int64_t)a.V;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[j] = i < rows && col + j < a.V ? to_f32(d[col + j]) : 0.f;
        bf16x8 exact[NP];
        split_parts<NP, 8>(x, exact);
#pragma unroll
        for (int p = 0; p < NP; ++p) fr[(wave * (NP + 6) + p) * 64 + lane] = __builtin_bit_cast(uint4, exact[p]);
        split_parts<3, 8>(drc + (int64_t)i * a.VP + col, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) fr[(wave * (NP + 6) + NP + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
        split_parts<3, 8>(ec + (int64_t)i * a.VP + col, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) fr[(wave * (NP + 6) + NP + 3 + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
      }
      __syncthreads();
      uint4 sb[NT][3], db[NT][3];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int64_t o = (int64_t)(16 * (wave * NT + t) + c) * a.VP + v0 + 8 * g;
        float x[8], y[8];
        bf16x8 parts[3];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = sc[o + j];
          y[j] = dsc[o + j];
          dot += x[j] * y[j];
        }
        split_parts<3, 8>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) sb[t][p] = __builtin_bit_cast(uint4, parts[p]);
        split_parts<3, 8>(y, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) db[t][p] = __builtin_bit_cast(uint4, parts[p]);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        uint4 da[NP], ra[3], ea[3];
#pragma unroll
        for (int p = 0; p < NP; ++p) da[p] = fr[(m * (NP + 6) + p) * 64 + lane];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          ra[p] = fr[(m * (NP + 6) + NP + p) * 64 + lane];
          ea[p] = fr[(m * (NP + 6) + NP + 3 + p) * 64 + lane];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          dq[m][t] = mma_parts<NP, 3>(da, sb[t], dq[m][t]);
          dr[m][t] = mma_parts<3, 3>(ra, sb[t], dr[m][t]);
          dw[m][t] = mma_parts<3, 3>(ea, db[t], dw[m][t]);
        }
      }
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        if (wave + 4 * t < 10) {
          int i, j;
          tri_tile(wave + 4 * t, &i, &j);
          uint4 da[NP], ra[3], ea[3];
#pragma unroll
          for (int p = 0; p < NP; ++p) da[p] = fr[(i * (NP + 6) + p) * 64 + lane];
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            ra[p] = fr[(i * (NP + 6) + NP + p) * 64 + lane];
            ea[p] = fr[(j * (NP + 6) + NP + 3 + p) * 64 + lane];
          }
          ne[t] = mma_parts<NP, 3>(da, ea, ne[t]);
          me[t] = mma_parts<3, 3>(ra, ea, me[t]);
        }
      }
    }
    // N and M, row i, column j
#pragma unroll
    for (int t = 0; t < 3; ++t) {
      if (wave + 4 * t < 10) {
        int it, jt;
        tri_tile(wave + 4 * t, &it, &jt);
        const int j = 16 * jt + c;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * it + 4 * g + r;
          const float d = j <= i ? beta[j] * gdr_decay(gs[i], gs[j]) : 0.f;
          nm[i * LD + j] = j <= i ? a.scale * d * ne[t][r] : 0.f;
          mm[i * LD + j] = j < i ? -beta[i] * d * me[t][r] : 0.f;
          if (i == j && i < rows) store_param(a.dbeta, a.b_dtype, (token + i) * a.Hv + h, me[t][r]);
        }
      }
    }
    // tiles above the diagonal that fragments of 32 columns reach into: (0, 1) and (2, 3)
    for (int z = tid; z < 512; z += 256) {
      const int i = (z >> 8) * 32 + ((z >> 4) & 15), j = (z >> 8) * 32 + 16 + (z & 15);
      nm[i * LD + j] = 0.f;
      mm[i * LD + j] = 0.f;
    }
    float last = 0.f;  // sum of k . ((E U) dS'^T): this lane's share
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * m + 4 * g + r;
        const float sg = a.scale * grown[i], bg = -beta[i] * grown[i], eb = rest[i] * beta[i];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int col = 16 * (wave * NT + t) + c;
          dq[m][t][r] *= sg;
          dr[m][t][r] *= bg;
          dw[m][t][r] *= eb;
          if (i < rows && col < a.K) last += to_f32(kp[i * a.k_s[1] + col]) * dw[m][t][r];
        }
      }
    last += grown[63] * dot;
    last = wave_sum(last);
    if (lane == 0) dots[wave] = last;
    __syncthreads();
    // dV = beta dR
    for (int i = tid >> 5; i < rows; i += 8) {
      const float b = beta[i];
      T* __restrict__ d = static_cast<T*>(a.dv) + ((token + i) * a.Hv + h) * (int64_t)a.V;
      for (int col = tid & 31; col < a.V; col += 32) d[col] = from_f32<T>(b * drc[(int64_t)i * a.VP + col]);
    }
#pragma unroll
    for (int which = 0; which < 2; ++which) {  // N, then M: the products with K and Q
      const float* __restrict__ X = which ? mm : nm;
      for (int f = wave; f < kTri; f += 4) {
        const int ml = f < 2 ? f : f / 2 + 1, sl = f < 2 ? 0 : f & 1, mu = f < 4 ? f / 2 : f - 2, su = f < 4 ? f & 1 : 1;
        float v[8];
        bf16x8 parts[3];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = X[(16 * ml + c) * LD + 32 * sl + gdr_at(g, i)];
        split_parts<3, 8>(v, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) fr[(f * 3 + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = X[(32 * su + gdr_at(g, i)) * LD + 16 * mu + c];
        split_parts<3, 8>(v, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) fr[((kTri + f) * 3 + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
      }
      __syncthreads();
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint4 kb[NT][NP], qb[NT][NP];
#pragma unroll
        for (int t = 0; t < NT; ++t)
#pragma unroll
          for (int p = 0; p < NP; ++p) {
            kb[t][p] = a.ktf[kbase + (((wave * NT + t) * 2 + s) * NP + p) * 64 + lane];
            if (!which) qb[t][p] = a.qtf[kbase + (((wave * NT + t) * 2 + s) * NP + p) * 64 + lane];
          }
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          uint4 xa[3];
          if (s == 0 || m >= 2) {
#pragma unroll
            for (int p = 0; p < 3; ++p) xa[p] = fr[(tri_lower(m, s) * 3 + p) * 64 + lane];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              if (!which) dq[m][t] = mma_parts<3, NP>(xa, kb[t], dq[m][t]);
              else dr[m][t] = mma_parts<3, NP>(xa, kb[t], dr[m][t]);
            }
          }
          if (s == 1 || m < 2) {
#pragma unroll
            for (int p = 0; p < 3; ++p) xa[p] = fr[((kTri + tri_upper(m, s)) * 3 + p) * 64 + lane];
#pragma unroll
            for (int t = 0; t < NT; ++t) dw[m][t] = mma_parts<3, NP>(xa, which ? kb[t] : qb[t], dw[m][t]);
          }
        }
      }
      __syncthreads();
    }
    // dG, 16 tokens of this wave's columns at a time
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      float x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * m + 4 * g + r;
        x[r] = 0.f;
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          const int col = 16 * (wave * NT + t) + c;
          if (i < rows && col < a.K)
            x[r] += to_f32(qp[i * a.q_s[1] + col]) * dq[m][t][r] +
                    to_f32(kp[i * a.k_s[1] + col]) * (dr[m][t][r] - dw[m][t][r]);
        }
      }
#pragma unroll
      for (int off = 8; off >= 1; off >>= 1)
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] += __shfl_xor(x[r], off, 64);
      if (c == 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r) dg_part[wave][16 * m + 4 * g + r] = x[r];
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        dqs[m][t] += dq[m][t];
        dks[m][t] += dr[m][t] + dw[m][t];
      }
    }
    __syncthreads();
    if (wave == 0) {
      double s = (double)((dg_part[0][lane] + dg_part[1][lane]) + (dg_part[2][lane] + dg_part[3][lane]));
      if (lane == 63) s += (double)((dots[0] + dots[1]) + (dots[2] + dots[3]));
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double t = __shfl_down(s, off, 64);
        if (lane + off < 64) s += t;
      }
      if (lane < rows) store_param(a.dg, a.g_dtype, (token + lane) * a.Hv + h, (float)s);
    }
    // (the next head's first barrier comes before anything that is read here is written)
  }
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * m + 4 * g + r;
      if (i >= rows) continue;
      const int64_t o = ((token + i) * a.Hk + hk) * (int64_t)a.K;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int col = 16 * (wave * NT + t) + c;
        if (col < a.K) {
          static_cast<T*>(a.dq)[o + col] = from_f32<T>(dqs[m][t][r]);
          static_cast<T*>(a.dk)[o + col] = from_f32<T>(dks[m][t][r]);
        }
      }
    }
}

template <typename T, int KP>
int launch(const GdrArgs& a, hipStream_t s) {
  hipLaunchKernelGGL((gdr_bwd_chain_kernel<T, KP>), dim3((unsigned)(a.VP / 16), (unsigned)a.Hv, (unsigned)a.n), dim3(256), 0, s, a);
  if (int rc = check_launch("gdr_bwd_chain_kernel")) return rc;
  if (a.T == 0) return ATK_OK;
  hipLaunchKernelGGL((gdr_grads_kernel<T, KP>), dim3((unsigned)a.slots, (unsigned)a.Hk), dim3(256), 0, s, a);
  return check_launch("gdr_grads_kernel");
}
template <typename T>
int launch_sized(const GdrArgs& a, hipStream_t s) {
  switch (gdr_padded_k(a.K)) {
    case 64: return launch<T, 64>(a, s);
    case 128: return launch<T, 128>(a, s);
    default: return launch<T, 256>(a, s);
  }
}

}  // namespace
}  // namespace atk

extern "C" size_t atk_gated_delta_bwd_workspace_bytes(const atk_gated_delta_args* p) {
  atk::GdrArgs a;
  int rc;
  return atk::gdr_plan(p, true, &a, &rc);
}

extern "C" int atk_gated_delta_bwd(const atk_gated_delta_args* p, const void* dout, const void* dfinal_state, void* dq,
                                   void* dk, void* dv, void* dg, void* dbeta, void* dinitial_state) {
  using namespace atk;
  GdrArgs a;
  int rc;
  const size_t need = gdr_plan(p, true, &a, &rc);
  if (rc) return rc;
  if (p->N == 0) return ATK_OK;
  if (p->T > 0 && (!p->q || !p->k || !p->v || !p->g || !p->beta || !dout || !dq || !dk || !dv || !dg || !dbeta))
    return fail(ATK_EINVAL, "gated delta backward: null pointer");
  if (need && (!p->workspace || p->workspace_bytes < need || !aligned16(p->workspace)))
    return fail(ATK_EINVAL, "gated delta backward: workspace too small or not 16-byte aligned");
  a.s1 = nullptr;
  a.dout = dout; a.ds1 = static_cast<const float*>(dfinal_state); a.ds0 = static_cast<float*>(dinitial_state);
  a.dq = dq; a.dk = dk; a.dv = dv; a.dg = dg; a.dbeta = dbeta;
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  if (p->T > 0) {
    if (int r = gdr_prepare(a, p->dtype, true, s)) return r;
    if (int r = gdr_chain(a, p->dtype, true, s)) return r;
  }
  if (p->dtype == ATK_F32) return launch_sized<float>(a, s);
  if (p->dtype == ATK_F16) return launch_sized<_Float16>(a, s);
  return launch_sized<__bf16>(a, s);
}

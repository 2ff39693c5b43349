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

// The chain of dS', built as the forward's: four waves pass the state's gradient on, 16 value columns
// of it; four more make what needs dO alone, a chunk ahead: scale P^T dO and Q^T (scale exp(G) dO).
// FULL as there.
template <typename T, int KP, bool FULL>
__global__ __launch_bounds__(512) void gdr_bwd_chain_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32, MT = KP / 64, KW = MT > 1 ? MT / 2 : 1;
  constexpr int KF = KS * 4 * NP * 64;
  __shared__ f32x4 kp[4][4][64];                            // partial sums of K dS'
  __shared__ uint2 ul[2][3][64][2], rl[2][3][64][2];        // dU, and -beta exp(G) dR
  __shared__ uint2 dl[2][NP][64][2], gl[2][3][64][2];       // dO, and scale exp(G) dO
  __shared__ f32x4 pl[4][64];                               // scale P^T dO
  __shared__ f32x4 ql[2][KP / 16][64];                      // Q^T (scale exp(G) dO), two chunks'
  __shared__ f32x4 tl[4][64];                               // dO on its way from rows to columns
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile, h;
  int64_t n;
  if (!gdr_chain_place(a, a.VP / 16, &tile, &h, &n)) return;
  const int hk = h / a.group, col = tile * 16 + c;
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t chunks = (seq.len + kGdrC - 1) / kGdrC, end = seq.slot + chunks - 1;  // from the last chunk down
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (wave < 4) {
    const int s0 = MT == 1 ? wave / 2 : wave * KW;
    const uint4* __restrict__ kf = a.kf + (hk * a.slots + end) * KF + s0 * 4 * NP * 64;
    const uint4* __restrict__ ktf = a.ktf + (hk * a.slots + end) * KF + wave * MT * 2 * NP * 64;
    const bool two = wave < 2;  // column halves of this wave's rows of T^T
    const uint4* __restrict__ tf = a.ttf + (h * a.slots + end) * (int64_t)(kTri * 3 * 64) + tri_upper(wave, wave >> 1) * 3 * 64;
    const float* __restrict__ row = a.row + (h * a.slots + end) * 192;
    float* __restrict__ dsc = a.dsc + (h * a.slots + end) * (int64_t)KP * a.VP + col;
    float* __restrict__ drc = a.drc + (h * a.slots + end) * (int64_t)64 * a.VP + (16 * wave + 4 * g) * (int64_t)a.VP + col;
    f32x4 S[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * (wave * MT + m) + 4 * g + r;
        S[m][r] = a.ds1 && i < a.K && col < a.V ? a.ds1[((n * a.Hv + h) * a.K + i) * a.V + col] : 0.f;
      }
    // here, and not in every pass of the loop, the compiler waits for these loads
#pragma unroll
    for (int m = 0; m < MT; ++m) asm volatile("" : "+v"(S[m]));
    uint4 ka[KW][4][NP], ta[2][3], kta[2][MT][NP];
    f32x4 grown, rest, beta;
    float all;
    int lane63 = 63;
    asm("" : "+v"(lane63));  // a vector address: a scalar load would be waited for at the next barrier
    auto load_k = [&]() {
#pragma unroll
      for (int s = 0; s < KW; ++s)
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int p = 0; p < NP; ++p) ka[s][m][p] = kf[((s * 4 + m) * NP + p) * 64 + lane];
    };
    auto load_t = [&]() {
#pragma unroll
      for (int p = 0; p < 3; ++p) ta[0][p] = tf[p * 64 + lane];
#pragma unroll
      for (int p = 0; p < 3; ++p) ta[1][p] = tf[((two ? 3 : 0) + p) * 64 + lane];
    };
    auto load_kt = [&]() {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int p = 0; p < NP; ++p) kta[s][m][p] = ktf[((m * 2 + s) * NP + p) * 64 + lane];
    };
    auto load_rows = [&]() {
      grown = *reinterpret_cast<const f32x4*>(row + 16 * wave + 4 * g);
      rest = *reinterpret_cast<const f32x4*>(row + 64 + 16 * wave + 4 * g);
      beta = *reinterpret_cast<const f32x4*>(row + 128 + 16 * wave + 4 * g);
      all = row[lane63];
    };
    if (chunks > 0) {
      load_k();
      load_rows();
      load_t();
      load_kt();
    }
    __syncthreads();  // the helpers' dO of the last chunk
    __syncthreads();  // and what they make of it
    for (int64_t ch = chunks - 1; ch >= 0; --ch) {
      const bool more = ch > 0;
      kf -= more ? KF : 0;
      ktf -= more ? KF : 0;
      tf -= more ? kTri * 3 * 64 : 0;
      row -= more ? 192 : 0;
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) dsc[(int64_t)(16 * (wave * MT + m) + 4 * g + r) * a.VP] = S[m][r];
      dsc -= (int64_t)KP * a.VP;
      f32x4 y[4] = {zero, zero, zero, zero};
#pragma unroll
      for (int s = 0; s < KW; ++s) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = MT > 1 ? S[MT > 1 ? 2 * s : 0][r] : (wave & 1) ? 0.f : S[0][r];
          x[4 + r] = MT > 1 ? S[MT > 1 ? 2 * s + 1 : 0][r] : (wave & 1) ? S[0][r] : 0.f;
        }
        bf16x8 parts[3];
        uint4 sp[3];
        split_parts<3, 8>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) sp[p] = __builtin_bit_cast(uint4, parts[p]);
        mma_tiles<4, NP, 3>(ka[s], sp, y);
      }
      load_k();
#pragma unroll
      for (int m = 0; m < 4; ++m) kp[wave][m][lane] = y[m];
      __syncthreads();
      {
        const f32x4 y0 = kp[0][wave][lane], y1 = kp[1][wave][lane], y2 = kp[2][wave][lane], y3 = kp[3][wave][lane];
        const f32x4 z = (y0 + y1) + (y2 + y3), pd = pl[wave][lane];
        float x[4];
        bf16x4 parts[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = pd[r] + rest[r] * z[r];
        split_parts<3, 4>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) ul[wave >> 1][p][lane][wave & 1] = __builtin_bit_cast(uint2, parts[p]);
      }
      __syncthreads();
      f32x4 dr;
      {
        f32x4 part[3] = {zero, zero, zero};  // three sums, so that no product waits for the one before it
        uint4 b[2][3];
#pragma unroll
        for (int p = 0; p < 3; ++p) b[0][p] = *reinterpret_cast<const uint4*>(&ul[wave >> 1][p][lane]);
        if (two)
#pragma unroll
          for (int p = 0; p < 3; ++p) b[1][p] = *reinterpret_cast<const uint4*>(&ul[1][p][lane]);
        auto half = [&](int s) {
          part[0] = mma(ta[s][2], b[s][0], part[0]);
          part[1] = mma(ta[s][1], b[s][1], part[1]);
          part[2] = mma(ta[s][0], b[s][2], part[2]);
          __builtin_amdgcn_sched_barrier(0);
          part[0] = mma(ta[s][1], b[s][0], part[0]);
          part[1] = mma(ta[s][0], b[s][1], part[1]);
          part[2] = mma(ta[s][0], b[s][0], part[2]);
        };
        half(0);
        if (two) half(1);
        dr = (part[0] + part[1]) + part[2];
      }
      {
        float x[4];
        bf16x4 parts[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = -beta[r] * grown[r] * dr[r];
        split_parts<3, 4>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) rl[wave >> 1][p][lane][wave & 1] = __builtin_bit_cast(uint2, parts[p]);
      }
#pragma unroll
      for (int r = 0; r < 4; ++r) drc[r * (int64_t)a.VP] = dr[r];
      drc -= (int64_t)64 * a.VP;
      load_t();
      __syncthreads();
      {
        f32x4 z[MT];
        uint4 b[2][3];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int p = 0; p < 3; ++p) b[s][p] = *reinterpret_cast<const uint4*>(&rl[s][p][lane]);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          S[m] = S[m] * all + ql[ch & 1][wave * MT + m][lane];
          z[m] = zero;
        }
        __builtin_amdgcn_sched_barrier(0);
        mma_tiles<MT, NP, 3>(kta[1], b[1], z);
        mma_tiles<MT, NP, 3>(kta[0], b[0], S);
#pragma unroll
        for (int m = 0; m < MT; ++m) S[m] += z[m];
      }
      load_rows();
      load_kt();
    }
    if (a.ds0) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * (wave * MT + m) + 4 * g + r;
          if (i < a.K && col < a.V) a.ds0[((n * a.Hv + h) * a.K + i) * a.V + col] = S[m][r];
        }
    }
  } else {
    const int m = wave - 4;
    const int tok = 16 * m + (lane >> 2);
    const bool dead = tile * 16 >= a.V;  // a tile of padding: dO of zeros
    const int c4 = FULL && !dead ? (tile * 16 + 4 * (lane & 3) + 4 <= a.V ? 4 * (lane & 3) : a.V - 4 - tile * 16) : 4 * (lane & 3);
    const int64_t os = (int64_t)a.Hv * a.V, last = (chunks - 1) * kGdrC;
    const T* __restrict__ op = static_cast<const T*>(a.dout) + ((seq.batch * a.T + seq.begin + last) * a.Hv + h) * (int64_t)a.V +
                               (dead ? 0 : tile * 16 + (FULL ? c4 : 0));
    const bool two = m < 2;
    const float* __restrict__ row = a.row + (h * a.slots + end) * 192 + 16 * m + 4 * g;
    const uint4* __restrict__ pf = a.ptf + (h * a.slots + end) * (int64_t)(kTri * 3 * 64) + tri_upper(m, m >> 1) * 3 * 64;
    const uint4* __restrict__ qtf = a.qtf + (hk * a.slots + end) * KF + m * MT * 2 * NP * 64;
    T oa[4];
    bool gone;
    f32x4 grown;
    uint4 pa[2][3], qa[2][MT][NP];
    auto load_o = [&](int64_t left) {
      gone = dead || tok >= left;
      const T* __restrict__ p = op + (tok < left ? tok * os : 0);
      if constexpr (FULL) {
        __builtin_memcpy(oa, p, 4 * sizeof(T));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) oa[j] = p[tile * 16 + c4 + j < a.V ? c4 + j : 0];
      }
      grown = *reinterpret_cast<const f32x4*>(row);
    };
    auto load_p = [&]() {
#pragma unroll
      for (int p = 0; p < 3; ++p) pa[0][p] = pf[p * 64 + lane];
#pragma unroll
      for (int p = 0; p < 3; ++p) pa[1][p] = pf[((two ? 3 : 0) + p) * 64 + lane];
    };
    auto load_q = [&]() {
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int p = 0; p < NP; ++p) qa[s][t][p] = qtf[((t * 2 + s) * NP + p) * 64 + lane];
    };
    auto put_o = [&]() {  // this wave's 16 tokens, through LDS from rows to columns
#pragma unroll
      for (int j = 0; j < 4; ++j)
        tl[m][16 * (lane >> 4) + c4 + j][(lane >> 2) & 3] =
            gone || (!FULL && tile * 16 + c4 + j >= a.V) ? 0.f : to_f32(oa[j]);
      __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses keep their order)
      const f32x4 x = tl[m][lane], y = a.scale * grown * x;
      bf16x4 exact[NP], parts[3];
      const float xs[4] = {x[0], x[1], x[2], x[3]}, ys[4] = {y[0], y[1], y[2], y[3]};
      split_parts<NP, 4>(xs, exact);
      split_parts<3, 4>(ys, parts);
#pragma unroll
      for (int p = 0; p < NP; ++p) dl[m >> 1][p][lane][m & 1] = __builtin_bit_cast(uint2, exact[p]);
#pragma unroll
      for (int p = 0; p < 3; ++p) gl[m >> 1][p][lane][m & 1] = __builtin_bit_cast(uint2, parts[p]);
      __builtin_amdgcn_wave_barrier();
    };
    auto products = [&](int buffer) {
      f32x4 y = zero, z = zero, q[MT];
      uint4 b[NP], d[2][3];
#pragma unroll
      for (int p = 0; p < NP; ++p) b[p] = *reinterpret_cast<const uint4*>(&dl[m >> 1][p][lane]);
      y = mma_parts<3, NP>(pa[0], b, y);
      if (two) {
#pragma unroll
        for (int p = 0; p < NP; ++p) b[p] = *reinterpret_cast<const uint4*>(&dl[1][p][lane]);
        z = mma_parts<3, NP>(pa[1], b, z);
      }
      pl[m][lane] = a.scale * (y + z);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int p = 0; p < 3; ++p) d[s][p] = *reinterpret_cast<const uint4*>(&gl[s][p][lane]);
#pragma unroll
      for (int t = 0; t < MT; ++t) q[t] = zero;
      mma_tiles<MT, NP, 3>(qa[0], d[0], q);
      mma_tiles<MT, NP, 3>(qa[1], d[1], q);
#pragma unroll
      for (int t = 0; t < MT; ++t) ql[buffer][m * MT + t][lane] = q[t];
    };
    tl[m][lane] = zero;  // columns past V keep it
    __builtin_amdgcn_wave_barrier();
    // Rows past the end of a sequence's last chunk are zeros; the chunks before it are whole.
    auto next = [&](bool more) {
      op -= more ? kGdrC * os : 0;
      row -= more ? 192 : 0;
      pf -= more ? kTri * 3 * 64 : 0;
      qtf -= more ? KF : 0;
    };
    if (chunks > 0) {
      load_o(seq.len - last);
      put_o();
      load_p();
      load_q();
    }
    __syncthreads();
    if (chunks > 0) {
      products((chunks - 1) & 1);
      next(chunks > 1);
      load_o(chunks > 1 ? kGdrC : seq.len - last);
      load_p();
      load_q();
    }
    __syncthreads();
    for (int64_t ch = chunks - 1; ch >= 0; --ch) {
      // beside chunk ch: the products of the chunk before it (at the end the first one's again, unread)
      __syncthreads();
      put_o();
      __syncthreads();
      products((ch - 1) & 1);
      next(ch > 1);
      load_o(ch > 0 ? kGdrC : seq.len);
      load_p();
      load_q();
      __syncthreads();
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
  const int64_t grid = (a.n * a.Hv + 7) / 8 * 8 * (a.VP / 16);
  if (grid > 0x7fffffff) return fail(ATK_UNSUPPORTED, "gated delta backward: too many heads, sequences and value columns");
  if (a.V % 16 == 0 || a.V % 16 >= 4) hipLaunchKernelGGL((gdr_bwd_chain_kernel<T, KP, true>), dim3((unsigned)grid), dim3(512), 0, s, a);
  else hipLaunchKernelGGL((gdr_bwd_chain_kernel<T, KP, false>), dim3((unsigned)grid), dim3(512), 0, s, a);
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

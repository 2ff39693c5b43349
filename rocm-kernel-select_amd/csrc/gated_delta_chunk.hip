// The gated delta rule over whole sequences, in chunks of 64 tokens.
//
// Within a chunk, with G the running sum of the log decays, D_ij = exp(G_i - G_j), S the state before
// it and W the strictly lower part of K K^T * D:
//   X  = V - exp(G) (K S)
//   e  = (1 + W diag(beta))^-1 X        the errors v_t - S~^T k_t of the chunk's tokens
//   U  = beta e
//   O  = scale (exp(G) (Q S) + lower(Q K^T * D) U)
//   S' = exp(G_63) S + K^T (exp(G_63 - G) U)
// The inverse and lower(Q K^T * D) depend on one chunk alone: the prepare kernel computes them for all
// chunks at once and writes everything a product needs in the order in which MFMA lanes read it.
// The chain kernel then passes the state from chunk to chunk, a workgroup for each sequence, head
// and tile of value columns.
#include "gated_delta.h"

namespace atk {
namespace {

constexpr int LD = 68;  // row pitch of the fp32 64 x 64 tiles in LDS: 16-byte rows, 4 banks apart

// 4 consecutive elements of a row of N, zeros past its end
template <typename T>
__device__ __forceinline__ void load4(const T* __restrict__ p, int c, int N, bool live, float* o) {
  if (live && c + 4 <= N) {
    T e[4];
    __builtin_memcpy(e, p + c, 4 * sizeof(T));  // element alignment only
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = to_f32(e[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) o[i] = live && c + i < N ? to_f32(p[c + i]) : 0.f;
  }
}

// T = (1 + A)^-1 for the strictly lower A (LDS, 64 x LD; read below the diagonal only).  Each wave
// inverts one 16 x 16 diagonal block by forward substitution, a column a lane; the blocks below follow
// by distance from the diagonal, T_ij = -T_ii sum_k A_ik T_kj, on fp32 MFMA.  All of Tm's upper part
// is zeroed.  Ends with a barrier.
__device__ void invert_unit_lower(const float* __restrict__ A, float* __restrict__ Tm, int wave, int lane) {
  const int c = lane & 15, g = lane >> 4;
  {
    float x[16];
    const float* a = A + (16 * wave) * LD + 16 * wave;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float s = i == c ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) s -= a[i * LD + j] * x[j];
      x[i] = s;
    }
    if (g == 0) {
#pragma unroll
      for (int i = 0; i < 16; ++i) Tm[(16 * wave + i) * LD + 16 * wave + c] = x[i];
    } else {  // the blocks right of the diagonal: wave w has 3 - w of them
      for (int b = wave + g; b < 4; b += 3)
#pragma unroll
        for (int i = 0; i < 16; ++i) Tm[(16 * wave + i) * LD + 16 * b + c] = 0.f;
    }
  }
  __syncthreads();
#pragma unroll
  for (int d = 1; d < 4; ++d) {
    const int j = wave, i = wave + d;
    if (i < 4) {
      f32x4 s = {0.f, 0.f, 0.f, 0.f};
      for (int k = j; k < i; ++k) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(A + (16 * i + c) * LD + 16 * k + 4 * g);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          s = __builtin_amdgcn_mfma_f32_16x16x4f32(a[r], Tm[(16 * k + 4 * g + r) * LD + 16 * j + c], s, 0, 0, 0);
      }
      const f32x4 t = *reinterpret_cast<const f32x4*>(Tm + (16 * i + c) * LD + 16 * i + 4 * g);
      f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int r = 0; r < 4; ++r) o = __builtin_amdgcn_mfma_f32_16x16x4f32(t[r], s[r], o, 0, 0, 0);
#pragma unroll
      for (int r = 0; r < 4; ++r) Tm[(16 * i + 4 * g + r) * LD + 16 * j + c] = -o[r];
    }
    __syncthreads();
  }
}

// The rows of a lower triangular 64 x 64 matrix (LDS) as fragments in three parts.
__device__ __forceinline__ void write_lower(const float* __restrict__ M, uint4* __restrict__ out, int wave, int lane) {
  const int c = lane & 15, g = lane >> 4;
  for (int f = wave; f < kTri; f += 4) {
    const int m = f < 2 ? f : f / 2 + 1, s = f < 2 ? 0 : f & 1;
    float v[8];
    bf16x8 parts[3];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = M[(16 * m + c) * LD + 32 * s + gdr_at(g, i)];
    split_parts<3, 8>(v, parts);
#pragma unroll
    for (int p = 0; p < 3; ++p) out[(f * 3 + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
  }
}

// Its columns: the rows of the transpose, an upper triangular matrix.
__device__ __forceinline__ void write_transposed(const float* __restrict__ M, uint4* __restrict__ out, int wave, int lane) {
  const int c = lane & 15, g = lane >> 4;
  for (int f = wave; f < kTri; f += 4) {
    const int m = f < 4 ? f / 2 : f - 2, s = f < 4 ? f & 1 : 1;
    float v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = M[(32 * s + gdr_at(g, i)) * LD + 16 * m + c];
    bf16x8 parts[3];
    split_parts<3, 8>(v, parts);
#pragma unroll
    for (int p = 0; p < 3; ++p) out[(f * 3 + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
  }
}

// The transpose of 64 tokens' fragments in LDS: 8 tokens of one column a lane.
template <int KP, int NP>
__device__ __forceinline__ void write_columns(const uint4* __restrict__ frags, uint4* __restrict__ out, int wave, int lane) {
  const __bf16* b = reinterpret_cast<const __bf16*>(frags);
  const int c = lane & 15, g = lane >> 4;
  for (int f = wave; f < (KP / 16) * 2; f += 4) {
    const int m = f >> 1, s = f & 1, col = 16 * m + c;
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      bf16x8 v;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int tok = 32 * s + gdr_at(g, i);
        v[i] = b[((((col >> 5) * 4 + (tok >> 4)) * NP + p) * 64 + (tok & 15) + 16 * ((col >> 2) & 3)) * 8 + (col & 3) + 4 * ((col >> 4) & 1)];
      }
      out[(f * NP + p) * 64 + lane] = __builtin_bit_cast(uint4, v);
    }
  }
}

// A workgroup for each (chunk, value head); the first value head of a key head's group also writes
// that key head's K, Q and K^T.
template <typename T, int KP, bool BWD>
__global__ __launch_bounds__(256) void gdr_prepare_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32;
  __shared__ uint4 kl[KS * 4 * NP * 64];  // K's fragments
  __shared__ __align__(16) float wm[64 * LD], tm[64 * LD];
  __shared__ double gd[64];
  __shared__ float bs[64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, c = lane & 15, g = lane >> 4;
  const int64_t slot = blockIdx.x;
  const int h = blockIdx.y, hk = h / a.group;
  const int64_t n = gdr_seq_of_slot(a.cu, a.T, a.n, slot);
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t at = (slot - seq.slot) * kGdrC;  // the chunk's first token within the sequence
  if (at < 0 || at >= seq.len) return;
  const int rows = (int)(seq.len - at < kGdrC ? seq.len - at : kGdrC);
  const int64_t t0 = seq.begin + at;
  const bool owner = h % a.group == 0;
  const int64_t kbase = (slot * a.Hk + hk) * (int64_t)(KS * 4 * NP * 64);
  const int64_t tbase = (slot * a.Hv + h) * (int64_t)(kTri * 3 * 64);
  if (wave == 0) {
    float gv = 0.f, bv = 0.f;
    if (lane < rows) {
      gv = load_param(a.g, a.g_dtype, seq.batch * a.g_s[0] + (t0 + lane) * a.g_s[1] + h * a.g_s[2]);
      bv = load_param(a.beta, a.b_dtype, seq.batch * a.b_s[0] + (t0 + lane) * a.b_s[1] + h * a.b_s[2]);
    }
    gv = gv < -120.f ? -120.f : gv;  // exp of either is 0 in fp32, and sums with -inf have no differences
    double s = gv;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
      const double t = __shfl_up(s, off, 64);
      if (lane >= off) s += t;
    }
    const double last = __shfl(s, 63, 64);
    gd[lane] = s;
    bs[lane] = bv;
    if constexpr (BWD) a.gsum[(slot * a.Hv + h) * 64 + lane] = s;
    float* __restrict__ row = a.row + (slot * a.Hv + h) * 192;
    row[lane] = expf((float)s);
    row[64 + lane] = expf((float)(last - s));
    row[128 + lane] = bv;
  }
  uint4 qr[KS][NP], kr[KS][NP];  // this wave's 16 tokens
  {
    const int64_t tok = t0 + 16 * wave + c;
    const bool live = 16 * wave + c < rows;
    const T* __restrict__ q = static_cast<const T*>(a.q) + (live ? seq.batch * a.q_s[0] + tok * a.q_s[1] + hk * a.q_s[2] : 0);
    const T* __restrict__ k = static_cast<const T*>(a.k) + (live ? seq.batch * a.k_s[0] + tok * a.k_s[1] + hk * a.k_s[2] : 0);
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float v[8];
      bf16x8 parts[NP];
      load4(q, 32 * s + 4 * g, a.K, live, v);
      load4(q, 32 * s + 16 + 4 * g, a.K, live, v + 4);
      split_parts<NP, 8>(v, parts);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        qr[s][p] = __builtin_bit_cast(uint4, parts[p]);
        if (owner) a.qf[kbase + ((s * 4 + wave) * NP + p) * 64 + lane] = qr[s][p];
      }
      load4(k, 32 * s + 4 * g, a.K, live, v);
      load4(k, 32 * s + 16 + 4 * g, a.K, live, v + 4);
      split_parts<NP, 8>(v, parts);
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        kr[s][p] = __builtin_bit_cast(uint4, parts[p]);
        kl[((s * 4 + wave) * NP + p) * 64 + lane] = kr[s][p];
        if (owner) a.kf[kbase + ((s * 4 + wave) * NP + p) * 64 + lane] = kr[s][p];
      }
    }
  }
  __syncthreads();
  if (owner) write_columns<KP, NP>(kl, a.ktf + kbase, wave, lane);
  // rows 16 wave .. of K K^T * D (strict) into wm, and of Q K^T * D into tm
  float w[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    f32x4 kk = {0.f, 0.f, 0.f, 0.f}, qk = {0.f, 0.f, 0.f, 0.f};
    if (j <= wave) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 b[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) b[p] = kl[((s * 4 + j) * NP + p) * 64 + lane];
        kk = mma_parts<NP, NP>(kr[s], b, kk);
        qk = mma_parts<NP, NP>(qr[s], b, qk);
      }
    }
    const int cj = 16 * j + c;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * wave + 4 * g + r;
      const float d = cj <= i ? expf((float)(gd[i] - gd[cj])) : 0.f;
      w[j][r] = cj < i ? kk[r] * d : 0.f;
      wm[i * LD + cj] = w[j][r] * bs[cj];
      tm[i * LD + cj] = cj <= i ? qk[r] * d : 0.f;
    }
  }
  __syncthreads();
  if constexpr (BWD) {
    write_transposed(tm, a.ptf + tbase, wave, lane);
    if (owner) {  // Q in K's place: every wave is past its products
#pragma unroll
      for (int s = 0; s < KS; ++s)
#pragma unroll
        for (int p = 0; p < NP; ++p) kl[((s * 4 + wave) * NP + p) * 64 + lane] = qr[s][p];
      __syncthreads();
      write_columns<KP, NP>(kl, a.qtf + kbase, wave, lane);
    }
  } else {
    write_lower(tm, a.pf + tbase, wave, lane);
  }
  __syncthreads();
  invert_unit_lower(wm, tm, wave, lane);
  write_lower(tm, a.tf + tbase, wave, lane);
  if constexpr (BWD) {  // and (1 + diag(beta) W)^-1, transposed
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * g + r;
        wm[i * LD + 16 * j + c] = bs[i] * w[j][r];
      }
    __syncthreads();
    invert_unit_lower(wm, tm, wave, lane);
    write_transposed(tm, a.ttf + tbase, wave, lane);
  }
}

// Workgroup -> (value tile, head, sequence).  Workgroups are dealt to the 8 XCDs in turn; all value
// tiles of a head and sequence get the same one, since they read the same fragments through its L2.
__device__ __forceinline__ bool chain_place(const GdrArgs& a, int tiles, int* tile, int* h, int64_t* n) {
  const int64_t j = blockIdx.x / 8, unit = j / tiles * 8 + blockIdx.x % 8;
  *tile = (int)(j % tiles);
  *h = (int)(unit % a.Hv);
  *n = unit / a.Hv;
  return *n < a.n;
}

// The state's chain: 16 value columns of one head's state, all of its key rows, from chunk to chunk.
//
// What bounds it is the time of one step, since a step needs the one before it: three products that
// follow each other (K S, T X, K^T E U).  Four waves share them: wave w has the state's row tiles
// w MT .. in its accumulators, multiplies them as they are (their layout is B's) with the K of all 64
// tokens, and the four partial sums meet in LDS; then it has the tokens 16 w .. for X and e.  So the
// state itself never leaves the registers.  Fragments are loaded right after their last use, for the
// next chunk: a load has most of a step to arrive.  Four more waves make the outputs of the chunk
// before, off the chain.  A barrier orders LDS only; loads stay in flight across it.
template <typename T, int KP, bool KEEP>
__global__ __launch_bounds__(KEEP ? 256 : 512) void gdr_chain_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32, MT = KP / 64, KW = MT > 1 ? MT / 2 : 1;
  constexpr int KF = KS * 4 * NP * 64;
  __shared__ f32x4 kp[4][4][64], qp[KEEP ? 1 : 4][4][64];  // partial sums [state wave][token tile][lane]
  __shared__ uint2 xl[2][3][64][2], el[2][3][64][2];       // X and E U in parts, as B is read
  __shared__ f32x4 ul[KEEP ? 1 : 4][64];                   // U, fp32
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile, h;
  int64_t n;
  if (!chain_place(a, KEEP ? a.VP / 16 : (a.V + 15) / 16, &tile, &h, &n)) return;
  const int hk = h / a.group, col = tile * 16 + c;
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t chunks = (seq.len + kGdrC - 1) / kGdrC;
  const uint4* __restrict__ kf = a.kf + (seq.slot * a.Hk + hk) * KF;
  const uint4* __restrict__ qf = a.qf + (seq.slot * a.Hk + hk) * KF;
  const uint4* __restrict__ ktf = a.ktf + (seq.slot * a.Hk + hk) * KF;
  const uint4* __restrict__ tf = a.tf + (seq.slot * a.Hv + h) * (int64_t)(kTri * 3 * 64);
  const uint4* __restrict__ pf = a.pf + (seq.slot * a.Hv + h) * (int64_t)(kTri * 3 * 64);
  const float* __restrict__ row = a.row + (seq.slot * a.Hv + h) * 192;
  const int64_t kstep = (int64_t)a.Hk * KF, tstep = (int64_t)a.Hv * (kTri * 3 * 64), rstep = (int64_t)a.Hv * 192;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (wave < 4) {
    f32x4 S[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * (wave * MT + m) + 4 * g + r;
        S[m][r] = a.s0 && i < a.K && col < a.V ? a.s0[((n * a.Hv + h) * a.K + i) * a.V + col] : 0.f;
      }
    const int s0 = MT == 1 ? wave / 2 : wave * KW;  // this wave's first 32 key columns
    uint4 ka[KW][4][NP], qa[KW][4][NP], ta[2][3], kta[MT][2][NP];
    T va[4];
    f32x4 grown, eb, beta;
    float all;
    auto load_k = [&](int64_t ch) {
#pragma unroll
      for (int s = 0; s < KW; ++s)
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
          for (int p = 0; p < NP; ++p) ka[s][m][p] = kf[ch * kstep + (((s0 + s) * 4 + m) * NP + p) * 64 + lane];
    };
    auto load_q = [&](int64_t ch) {
      if constexpr (!KEEP) {
#pragma unroll
        for (int s = 0; s < KW; ++s)
#pragma unroll
          for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int p = 0; p < NP; ++p) qa[s][m][p] = qf[ch * kstep + (((s0 + s) * 4 + m) * NP + p) * 64 + lane];
      }
    };
    auto load_rows = [&](int64_t ch) {
      const float* __restrict__ rw = row + ch * rstep;
      grown = *reinterpret_cast<const f32x4*>(rw + 16 * wave + 4 * g);
      const f32x4 rest = *reinterpret_cast<const f32x4*>(rw + 64 + 16 * wave + 4 * g);
      beta = *reinterpret_cast<const f32x4*>(rw + 128 + 16 * wave + 4 * g);
      eb = rest * beta;
      all = rw[63];
      const int64_t left = seq.len - ch * kGdrC;
      const int64_t t0 = seq.begin + ch * kGdrC;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * g + r;
        va[r] = i < left && col < a.V
                    ? static_cast<const T*>(a.v)[seq.batch * a.v_s[0] + (t0 + i) * a.v_s[1] + h * a.v_s[2] + col]
                    : from_f32<T>(0.f);
      }
    };
    auto load_t = [&](int64_t ch) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= wave >> 1)
#pragma unroll
          for (int p = 0; p < 3; ++p) ta[s][p] = tf[ch * tstep + (tri_lower(wave, s) * 3 + p) * 64 + lane];
    };
    auto load_kt = [&](int64_t ch) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int p = 0; p < NP; ++p) kta[m][s][p] = ktf[ch * kstep + (((wave * MT + m) * 2 + s) * NP + p) * 64 + lane];
    };
    if (chunks > 0) {
      load_k(0);
      load_rows(0);
      load_q(0);
      load_t(0);
      load_kt(0);
    }
    for (int64_t ch = 0; ch < chunks; ++ch) {
      const int64_t next = ch + 1 < chunks ? ch + 1 : ch;  // (the last chunk's again at the end)
      if constexpr (KEEP) {
        float* __restrict__ sc = a.sc + ((seq.slot + ch) * a.Hv + h) * (int64_t)KP * a.VP;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[(int64_t)(16 * (wave * MT + m) + 4 * g + r) * a.VP + col] = S[m][r];
      }
      uint4 sp[KW][3];
#pragma unroll
      for (int s = 0; s < KW; ++s) {
        float x[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          x[r] = MT > 1 ? S[MT > 1 ? 2 * s : 0][r] : (wave & 1) ? 0.f : S[0][r];
          x[4 + r] = MT > 1 ? S[MT > 1 ? 2 * s + 1 : 0][r] : (wave & 1) ? S[0][r] : 0.f;
        }
        bf16x8 parts[3];
        split_parts<3, 8>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) sp[s][p] = __builtin_bit_cast(uint4, parts[p]);
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        f32x4 y = zero;
#pragma unroll
        for (int s = 0; s < KW; ++s) y = mma_parts<NP, 3>(ka[s][m], sp[s], y);
        kp[wave][m][lane] = y;
      }
      load_k(next);
      __syncthreads();
      const f32x4 y = (kp[0][wave][lane] + kp[1][wave][lane]) + (kp[2][wave][lane] + kp[3][wave][lane]);
      {
        float x[4];
        bf16x4 parts[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = to_f32(va[r]) - grown[r] * y[r];
        split_parts<3, 4>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) xl[wave >> 1][p][lane][wave & 1] = __builtin_bit_cast(uint2, parts[p]);
      }
      if constexpr (!KEEP) {
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          f32x4 z = zero;
#pragma unroll
          for (int s = 0; s < KW; ++s) z = mma_parts<NP, 3>(qa[s][m], sp[s], z);
          qp[wave][m][lane] = z;
        }
        load_q(next);
      }
      __syncthreads();
      f32x4 e = zero;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= wave >> 1) {
          uint4 b[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) b[p] = *reinterpret_cast<const uint4*>(&xl[s][p][lane]);
          e = mma_parts<3, 3>(ta[s], b, e);
        }
      load_t(next);
      {
        float x[4];
        bf16x4 parts[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = eb[r] * e[r];
        split_parts<3, 4>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) el[wave >> 1][p][lane][wave & 1] = __builtin_bit_cast(uint2, parts[p]);
        if constexpr (KEEP) {
          float* __restrict__ ec = a.ec + ((seq.slot + ch) * a.Hv + h) * (int64_t)64 * a.VP;
#pragma unroll
          for (int r = 0; r < 4; ++r) ec[(int64_t)(16 * wave + 4 * g + r) * a.VP + col] = e[r];
        } else {
          ul[wave][lane] = beta * e;
        }
      }
      const float decay = all;
      load_rows(next);
      __syncthreads();
#pragma unroll
      for (int m = 0; m < MT; ++m) S[m] *= decay;
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        uint4 b[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) b[p] = *reinterpret_cast<const uint4*>(&el[s][p][lane]);
#pragma unroll
        for (int m = 0; m < MT; ++m) S[m] = mma_parts<NP, 3>(kta[m][s], b, S[m]);
      }
      load_kt(next);
    }
    if (a.s1) {
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * (wave * MT + m) + 4 * g + r;
          if (i < a.K && col < a.V) a.s1[((n * a.Hv + h) * a.K + i) * a.V + col] = S[m][r];
        }
    }
  } else if constexpr (!KEEP) {
    const int m = wave - 4;
    T* __restrict__ o = static_cast<T*>(a.o);
    uint4 pa[2][3];
    f32x4 grown;
    auto load = [&](int64_t ch) {
      grown = *reinterpret_cast<const f32x4*>(row + ch * rstep + 16 * m + 4 * g);
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= m >> 1)
#pragma unroll
          for (int p = 0; p < 3; ++p) pa[s][p] = pf[ch * tstep + (tri_lower(m, s) * 3 + p) * 64 + lane];
    };
    if (chunks > 0) load(0);
    for (int64_t ch = 0; ch < chunks; ++ch) {
      __syncthreads();
      __syncthreads();
      __syncthreads();
      // from here to the state waves' next barrier but one, qp and ul are this chunk's
      f32x4 y = (qp[0][m][lane] + qp[1][m][lane]) + (qp[2][m][lane] + qp[3][m][lane]);
      y *= grown;
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (s <= m >> 1) {
          float x[8];
          bf16x8 parts[3];
          uint4 b[3];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            x[r] = ul[2 * s][lane][r];
            x[4 + r] = ul[2 * s + 1][lane][r];
          }
          split_parts<3, 8>(x, parts);
#pragma unroll
          for (int p = 0; p < 3; ++p) b[p] = __builtin_bit_cast(uint4, parts[p]);
          y = mma_parts<3, 3>(pa[s], b, y);
        }
      load(ch + 1 < chunks ? ch + 1 : ch);
      const int64_t left = seq.len - ch * kGdrC, t0 = seq.begin + ch * kGdrC;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * m + 4 * g + r;
        if (i < left && col < a.V) o[((seq.batch * a.T + t0 + i) * a.Hv + h) * (int64_t)a.V + col] = from_f32<T>(a.scale * y[r]);
      }
    }
    // tokens of a packed row before its first sequence and after its last have an output of zero
    if (a.cu && (n == 0 || n == a.n - 1)) {
      const int64_t from[2] = {n == 0 ? 0 : a.T, n == a.n - 1 ? seq.begin + seq.len : a.T};
      const int64_t to[2] = {n == 0 ? seq.begin : a.T, a.T};
      for (int z = 0; z < 2; ++z)
        for (int64_t i = from[z] + 4 * m + g; i < to[z]; i += 16)
          if (col < a.V) o[(i * a.Hv + h) * (int64_t)a.V + col] = from_f32<T>(0.f);
    }
  }
}

template <typename T, int KP>
int launch_prepare(const GdrArgs& a, bool backward, hipStream_t s) {
  const dim3 grid((unsigned)a.slots, (unsigned)a.Hv);
  if (backward) hipLaunchKernelGGL((gdr_prepare_kernel<T, KP, true>), grid, dim3(256), 0, s, a);
  else hipLaunchKernelGGL((gdr_prepare_kernel<T, KP, false>), grid, dim3(256), 0, s, a);
  return check_launch("gdr_prepare_kernel");
}
template <typename T, int KP>
int launch_chain(const GdrArgs& a, bool keep, hipStream_t s) {
  const int64_t units = (a.n * a.Hv + 7) / 8 * 8, grid = units * (keep ? a.VP / 16 : (a.V + 15) / 16);
  if (grid > 0x7fffffff) return fail(ATK_UNSUPPORTED, "gated delta: too many heads, sequences and value columns");
  if (keep) hipLaunchKernelGGL((gdr_chain_kernel<T, KP, true>), dim3((unsigned)grid), dim3(256), 0, s, a);
  else hipLaunchKernelGGL((gdr_chain_kernel<T, KP, false>), dim3((unsigned)grid), dim3(512), 0, s, a);
  return check_launch("gdr_chain_kernel");
}

}  // namespace

#define ATK_GDR_TYPED(FN, ...)                                            \
  [&]() {                                                                 \
    const int kp = gdr_padded_k(a.K);                                     \
    if (dtype == ATK_F32) return kp == 64 ? FN<float, 64>(__VA_ARGS__) : kp == 128 ? FN<float, 128>(__VA_ARGS__) : FN<float, 256>(__VA_ARGS__); \
    if (dtype == ATK_F16) return kp == 64 ? FN<_Float16, 64>(__VA_ARGS__) : kp == 128 ? FN<_Float16, 128>(__VA_ARGS__) : FN<_Float16, 256>(__VA_ARGS__); \
    return kp == 64 ? FN<__bf16, 64>(__VA_ARGS__) : kp == 128 ? FN<__bf16, 128>(__VA_ARGS__) : FN<__bf16, 256>(__VA_ARGS__); \
  }()

int gdr_prepare(const GdrArgs& a, int dtype, bool backward, hipStream_t s) {
  return ATK_GDR_TYPED(launch_prepare, a, backward, s);
}
int gdr_chain(const GdrArgs& a, int dtype, bool keep, hipStream_t s) { return ATK_GDR_TYPED(launch_chain, a, keep, s); }

// Checks a call and lays out its workspace: the bytes it takes, or 0 with *rc set.
size_t gdr_plan(const atk_gated_delta_args* p, bool backward, GdrArgs* a, int* rc) {
  *rc = ATK_OK;
  if (!p) return *rc = fail(ATK_EINVAL, "gated delta: null arguments"), 0;
  if (!dtype_ok(p->dtype) || !dtype_ok(p->g_dtype) || !dtype_ok(p->beta_dtype))
    return *rc = fail(ATK_EINVAL, "gated delta: unknown dtype code"), 0;
  if (p->N < 0 || p->T < 0 || p->Hk <= 0 || p->Hv <= 0 || p->K <= 0 || p->V <= 0)
    return *rc = fail(ATK_EINVAL, "gated delta: bad sizes"), 0;
  if (p->Hv % p->Hk) return *rc = fail(ATK_EINVAL, "gated delta: value heads must be a multiple of key heads"), 0;
  const int64_t per = (p->T + kGdrC - 1) / kGdrC;
  if (p->K > kGdrMaxK || p->Hv > 65535 || p->N > 65535 || p->T >= ((int64_t)1 << 31) - 64 ||
      (double)per * (double)p->N >= 2147483648.0 || p->V > (1 << 24))
    return *rc = fail(ATK_UNSUPPORTED, "gated delta: more than %d key columns, 65535 heads or sequences, or 2^31 tokens", kGdrMaxK), 0;
  *a = GdrArgs{};
  a->q = p->q; a->k = p->k; a->v = p->v; a->g = p->g; a->beta = p->beta; a->o = p->out;
  a->s0 = static_cast<const float*>(p->initial_state); a->s1 = static_cast<float*>(p->final_state); a->cu = p->cu_seqlens;
  for (int i = 0; i < 3; ++i) {
    a->q_s[i] = p->q_stride[i]; a->k_s[i] = p->k_stride[i]; a->v_s[i] = p->v_stride[i];
    a->g_s[i] = p->g_stride[i]; a->b_s[i] = p->beta_stride[i];
  }
  a->n = p->N; a->T = p->T; a->slots = p->cu_seqlens ? p->T / kGdrC + p->N : p->N * per;
  a->Hk = p->Hk; a->Hv = p->Hv; a->group = p->Hv / p->Hk; a->K = p->K; a->V = p->V;
  a->VP = (a->V + 31) / 32 * 32;
  a->g_dtype = p->g_dtype; a->b_dtype = p->beta_dtype; a->scale = p->scale;
  // (16-byte pieces throughout, so each part of the workspace is aligned as its start is)
  const int np = p->dtype == ATK_F32 ? 3 : p->dtype == ATK_F16 ? 2 : 1;
  const size_t kb = (size_t)a->slots * a->Hk * gdr_padded_k(a->K) * 64 * 2 * np, tb = (size_t)a->slots * a->Hv * kTri * 3 * 1024;
  char* w = static_cast<char*>(p->workspace);
  size_t off = 0;
  auto take = [&](size_t bytes) { char* q = w + off; off += bytes; return q; };
  a->kf = reinterpret_cast<uint4*>(take(kb)); a->qf = reinterpret_cast<uint4*>(take(kb));
  a->ktf = reinterpret_cast<uint4*>(take(kb)); a->tf = reinterpret_cast<uint4*>(take(tb));
  a->row = reinterpret_cast<float*>(take((size_t)a->slots * a->Hv * 768));
  if (!backward) {
    a->pf = reinterpret_cast<uint4*>(take(tb));
    return off;
  }
  const size_t state = (size_t)a->slots * a->Hv * gdr_padded_k(a->K) * a->VP * 4, row = (size_t)a->slots * a->Hv * 64 * a->VP * 4;
  a->qtf = reinterpret_cast<uint4*>(take(kb)); a->ttf = reinterpret_cast<uint4*>(take(tb));
  a->ptf = reinterpret_cast<uint4*>(take(tb));
  a->gsum = reinterpret_cast<double*>(take((size_t)a->slots * a->Hv * 512));
  a->sc = reinterpret_cast<float*>(take(state)); a->dsc = reinterpret_cast<float*>(take(state));
  a->ec = reinterpret_cast<float*>(take(row)); a->drc = reinterpret_cast<float*>(take(row));
  return off;
}

}  // namespace atk

extern "C" size_t atk_gated_delta_workspace_bytes(const atk_gated_delta_args* p) {
  atk::GdrArgs a;
  int rc;
  return atk::gdr_plan(p, false, &a, &rc);
}

extern "C" int atk_gated_delta_fwd(const atk_gated_delta_args* p) {
  using namespace atk;
  GdrArgs a;
  int rc;
  const size_t need = gdr_plan(p, false, &a, &rc);
  if (rc) return rc;
  if (p->N == 0 || (p->T == 0 && !p->final_state)) return ATK_OK;
  if (p->T > 0 && (!p->q || !p->k || !p->v || !p->g || !p->beta || !p->out))
    return fail(ATK_EINVAL, "gated delta: null pointer");
  if (need && (!p->workspace || p->workspace_bytes < need || !aligned16(p->workspace)))
    return fail(ATK_EINVAL, "gated delta: workspace too small or not 16-byte aligned");
  hipStream_t s = reinterpret_cast<hipStream_t>(p->stream);
  if (p->T > 0)
    if (int r = gdr_prepare(a, p->dtype, false, s)) return r;
  return gdr_chain(a, p->dtype, false, s);
}

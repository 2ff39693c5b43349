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
// What is not finite leaves no gradient finite that the recurrence spoils, but may spoil others of its chunk
// (dg is a sum from the chunk's end).  Key heads that several value heads share get the sum over them in a fixed order: one workgroup has
// a key head's whole group.
#include "gated_delta_chain.h"

namespace atk {
namespace {

__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == ATK_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == ATK_F16) static_cast<_Float16*>(p)[i] = from_f32<_Float16>(v);
  else static_cast<__bf16*>(p)[i] = from_f32<__bf16>(v);
}

// The chain of dS', built as the forward's: four waves pass the state's gradient on, 16 value columns
// of it; four more make what needs dO alone, a chunk ahead: scale P^T dO and Q^T (scale exp(G) dO).
// Bound by a step's time too, with the forward chain after it: 2048 tokens, 2 x 16 heads of 128 x 128 bf16,
// twice 32 steps in 160 to 166 us, matrix units 12 % busy, 84 MB read and 197 MB written.
// FULL as there.
template <typename T, int KP>
struct GdrBwdLds {
  static constexpr int NP = kParts<T>;
  f32x4 kp[4][4][64];                            // partial sums of K dS'
  uint2 ul[2][3][64][2], rl[2][3][64][2];        // dU, and -beta exp(G) dR
  uint2 dl[2][NP][64][2], gl[2][3][64][2];       // dO, and scale exp(G) dO
  f32x4 pl[4][64];                               // scale P^T dO
  f32x4 ql[2][KP / 16][64];                      // Q^T (scale exp(G) dO), two chunks'
  f32x4 tl[4][64];                               // dO on its way from rows to columns
};
template <typename T, int KP, bool FULL>
__device__ __forceinline__ void gdr_bwd_chain(const GdrArgs& a, char* lds, int64_t block) {
  constexpr int NP = kParts<T>, KS = KP / 32, MT = KP / 64, KW = MT > 1 ? MT / 2 : 1;
  constexpr int KF = KS * 4 * NP * 64;
  GdrBwdLds<T, KP>& L = *reinterpret_cast<GdrBwdLds<T, KP>*>(lds);
  auto& kp = L.kp;
  auto& ul = L.ul;
  auto& rl = L.rl;
  auto& dl = L.dl;
  auto& gl = L.gl;
  auto& pl = L.pl;
  auto& ql = L.ql;
  auto& tl = L.tl;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile, h;
  int64_t n;
  if (!gdr_chain_place(a, block, a.VP / 16, &tile, &h, &n)) return;
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
    float* __restrict__ dsc = a.dsc + (h * a.slots + end) * (int64_t)KP * a.VP + gdr_kept(tile, KP / 16, c, g);
    float* __restrict__ drc = a.drc + (h * a.slots + end) * (int64_t)64 * a.VP + gdr_kept(tile, 4, c, g) + wave * 512;
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
        for (int r = 0; r < 4; ++r) dsc[(wave * MT + m) * 512 + r * 8] = S[m][r];
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
      for (int r = 0; r < 4; ++r) drc[r * 8] = dr[r];
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
    // tokens of a packed row before its first sequence and after its last have gradients of zero
    if (a.cu && (n == 0 || n == a.n - 1)) {
      const int64_t from[2] = {n == 0 ? 0 : a.T, n == a.n - 1 ? seq.begin + seq.len : a.T};
      const int64_t to[2] = {n == 0 ? seq.begin : a.T, a.T};
      for (int z = 0; z < 2; ++z)
        for (int64_t i = from[z] + 4 * m + g; i < to[z]; i += 16) {
          const int64_t at = i * a.Hv + h;
          if (col < a.V) static_cast<T*>(a.dv)[at * a.V + col] = from_f32<T>(0.f);
          if (tile > 0) continue;
          if (c == 0) {
            store_param(a.dg, a.g_dtype, at, 0.f);
            store_param(a.dbeta, a.b_dtype, at, 0.f);
          }
          if (h % a.group == 0)
            for (int d = c; d < a.K; d += 16) {
              static_cast<T*>(a.dq)[(i * a.Hk + hk) * a.K + d] = from_f32<T>(0.f);
              static_cast<T*>(a.dk)[(i * a.Hk + hk) * a.K + d] = from_f32<T>(0.f);
            }
        }
    }
  }
}

// Both chains in one launch, the longer one's workgroups first: neither needs the other, and where there
// are fewer tiles than CUs they run side by side (1021 tokens, 4 heads of 64 x 64 fp32: 38 -> 24 us).
// Two to a CU gained nothing for 256 tiles of 128 x 128 in bf16 (168 us, one after the other 156): their
// loads then wait for each other.
template <typename T, int KP, bool FULL>
__global__ __launch_bounds__(512) void gdr_chains_kernel(GdrArgs a, int64_t first) {
  constexpr size_t A = sizeof(GdrChainLds<T, KP, true>), B = sizeof(GdrBwdLds<T, KP>);
  __shared__ __align__(16) char lds[A > B ? A : B];
  const int64_t half = gridDim.x / 2;
  if (blockIdx.x >= half) gdr_chain<T, KP, true, FULL>(a, lds, first + blockIdx.x - half);
  else gdr_bwd_chain<T, KP, FULL>(a, lds, first + blockIdx.x);
}

// (row, column) tile t of the ten of a lower triangle of 16 x 16 tiles
__device__ __forceinline__ void tri_tile(int t, int* i, int* j) {
  *i = t < 1 ? 0 : t < 3 ? 1 : t < 6 ? 2 : 3;
  *j = t - *i * (*i + 1) / 2;
}

// sum over each 16 lanes, in all of them
__device__ __forceinline__ float row16_sum(float v) {
  v += dpp_mov<0xB1>(v);
  v += dpp_mov<0x4E>(v);
  v += dpp_mov<0x141>(v);
  return v + dpp_mov<0x140>(v);
}

// What one chunk's gradients need of that chunk, for one key head and all of its value heads.  Each of
// eight waves has 16 NT key columns of dq and dk, for all 64 tokens or (64 columns) for 32.  The value columns are walked 32 at a
// time: the waves bring dO, dR and e of all tokens into LDS as fragments (the next 32 columns on their
// way meanwhile), and every wave multiplies them with its own rows of S and dS', which it splits
// itself.  The 16 x 16 tiles of dO e^T and dR e^T on and below the diagonal are shared out among the
// waves; a result's layout is that of the transpose's rows, so N and M leave the accumulators as
// fragments of their transposes, and, element by element, as their own.  K^T's and Q^T's fragments
// hold for each lane the elements that its accumulators have, so the row products of dG need no more
// loads.  V8: value columns come in eights, so a lane's are all there or all not.
// Bound by latency, one workgroup a CU and waves that wait about half of their time: 64 chunks, 8 and 16
// heads of 128 x 128, bf16, in 93 to 96 us, 126 MB read and 40 MB written, matrix units 24 % busy.  (With four
// waves, and S and dS' through LDS, 257 us.)
template <typename T, int KP, bool V8>
__global__ __launch_bounds__(512) void gdr_grads_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32, W = 8, NT = KP > 128 ? KP / 128 : 1;
  constexpr int CW = KP / 16 / NT, MR = 4 * CW / W;  // waves side by side over the key columns; row tiles of each
  constexpr int TILES = 2;                 // of the ten, this wave's: wave, and wave + 8 for the first two
  constexpr int UNIT = NP + 6;             // fragments of 16 tokens: dO, dR, e
  __shared__ uint4 st[4 * UNIT * 64];
  __shared__ uint2 nf[2][kTri * 3 * 64][2], mf[2][kTri * 3 * 64][2];  // N and M, their transposes
  __shared__ float2 gs[64];
  __shared__ float grown[64], rest[64], beta[64], dg_part[CW][64], dots[W], db[64];
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int cw = wave % CW, m0 = wave / CW * MR;
  const int64_t slot = blockIdx.x;
  const int hk = blockIdx.y;
  const int64_t n = gdr_seq_of_slot(a.cu, a.T, a.n, slot);
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t at = (slot - seq.slot) * kGdrC;
  if (at < 0 || at >= seq.len) return;
  const int rows = (int)(seq.len - at < kGdrC ? seq.len - at : kGdrC);
  const int64_t token = seq.batch * a.T + seq.begin + at;
  const int64_t kbase = (hk * a.slots + slot) * (int64_t)(KS * 4 * NP * 64);
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  // halves of fragments that lie beyond the diagonal: (row tile, column half, half) of N and of its transpose
  for (int z = tid; z < 4 * 3 * 64; z += 64 * W) {
    const int p = z / 64 % 3, l = z % 64, q = z / 192;
    const int f = q == 0 ? tri_lower(0, 0) : q == 1 ? tri_lower(2, 1) : q == 2 ? tri_upper(1, 0) : tri_upper(3, 1);
    nf[q >> 1][(f * 3 + p) * 64 + l][q < 2] = mf[q >> 1][(f * 3 + p) * 64 + l][q < 2] = make_uint2(0, 0);
  }
  f32x4 dqs[MR][NT], dks[MR][NT];  // sums over the group
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int t = 0; t < NT; ++t) dqs[m][t] = dks[m][t] = zero;
  int it[TILES], jt[TILES];
#pragma unroll
  for (int x = 0; x < TILES; ++x) {
    tri_tile(wave + W * x < 10 ? wave + W * x : 0, &it[x], &jt[x]);
    if (wave + W * x >= 10) it[x] = -1;
  }
  // one unit of 16 tokens a wave and turn: 0..3 dR (and dV), 4..7 e and dO
  constexpr int UNITS = 8 / W;
  for (int h = hk * a.group; h < (hk + 1) * a.group; ++h) {
    // (opaque to the compiler, which would keep the addresses of every access in registers for the next head)
    int lane = tid & 63;
    asm volatile("" : "+v"(lane));
    const int c = lane & 15, g = lane >> 4;
    const int64_t hs = h * a.slots + slot;
    const float* __restrict__ sc = a.sc + hs * KP * a.VP + cw * NT * 512 + 8 * lane;
    const float* __restrict__ dsc = a.dsc + hs * KP * a.VP + cw * NT * 512 + 8 * lane;
    const float* __restrict__ ec = a.ec + hs * 64 * a.VP + 8 * lane;
    const float* __restrict__ drc = a.drc + hs * 64 * a.VP + 8 * lane;
    f32x4 rs[NT][2], rd[NT][2], ru[UNITS][2];
    T ro[8];
    auto load = [&](int v0) {
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int z = 0; z < 2; ++z) {
          rs[t][z] = *reinterpret_cast<const f32x4*>(sc + v0 * KP + t * 512 + 4 * z);
          rd[t][z] = *reinterpret_cast<const f32x4*>(dsc + v0 * KP + t * 512 + 4 * z);
        }
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int unit = wave + W * u;
        const float* __restrict__ p = (unit < 4 ? drc : ec) + v0 * 64 + (unit & 3) * 512;
        ru[u][0] = *reinterpret_cast<const f32x4*>(p);
        ru[u][1] = *reinterpret_cast<const f32x4*>(p + 4);
      }
      const int i = 16 * (wave & 3) + c, col = v0 + 8 * g;
      const T* __restrict__ p = static_cast<const T*>(a.dout) + ((token + (i < rows ? i : 0)) * a.Hv + h) * (int64_t)a.V;
      if constexpr (V8) {
        __builtin_memcpy(ro, p + (col < a.V ? col : 0), 8 * sizeof(T));
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) ro[j] = p[col + j < a.V ? col + j : 0];
      }
    };
    load(0);
    if (tid < 64) {
      gs[tid] = a.gsum[hs * 64 + tid];
      grown[tid] = a.row[hs * 192 + tid];
      rest[tid] = a.row[hs * 192 + 64 + tid];
      beta[tid] = a.row[hs * 192 + 128 + tid];
    }
    f32x4 dq[MR][NT], dr[MR][NT], dw[MR][NT];  // dq, and dk as it is read and as it is written
    f32x4 ne[TILES], me[TILES];
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int t = 0; t < NT; ++t) dq[m][t] = dr[m][t] = dw[m][t] = zero;
#pragma unroll
    for (int x = 0; x < TILES; ++x) ne[x] = me[x] = zero;
    float dot = 0.f;  // <S, dS'>
    for (int v0 = 0; v0 < a.VP; v0 += 32) {
      __syncthreads();  // st's readers are past it
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int unit = wave + W * u, m = unit & 3, i = 16 * m + c, col = v0 + 8 * g;
        const float x[8] = {ru[u][0][0], ru[u][0][1], ru[u][0][2], ru[u][0][3], ru[u][1][0], ru[u][1][1], ru[u][1][2], ru[u][1][3]};
        bf16x8 parts[3];
        split_parts<3, 8>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) st[(m * UNIT + NP + (unit < 4 ? 0 : 3) + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
        if (unit < 4) {  // dV = beta dR
          if (i < rows) {
            const float b = beta[i];
            T* __restrict__ d = static_cast<T*>(a.dv) + ((token + i) * a.Hv + h) * (int64_t)a.V + col;
            T z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = from_f32<T>(b * x[j]);
            if constexpr (V8) {
              if (col < a.V) __builtin_memcpy(d, z, 8 * sizeof(T));
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (col + j < a.V) d[j] = z[j];
            }
          }
        } else {
          float y[8];
          bf16x8 exact[NP];
#pragma unroll
          for (int j = 0; j < 8; ++j) y[j] = i < rows && col + j < a.V ? to_f32(ro[j]) : 0.f;
          split_parts<NP, 8>(y, exact);
#pragma unroll
          for (int p = 0; p < NP; ++p) st[(m * UNIT + p) * 64 + lane] = __builtin_bit_cast(uint4, exact[p]);
        }
      }
      uint4 sb[NT][3], db[NT][3];
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float x[8], y[8];
        bf16x8 parts[3];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] = rs[t][j >> 2][j & 3];
          y[j] = rd[t][j >> 2][j & 3];
          dot += x[j] * y[j];
        }
        split_parts<3, 8>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) sb[t][p] = __builtin_bit_cast(uint4, parts[p]);
        split_parts<3, 8>(y, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) db[t][p] = __builtin_bit_cast(uint4, parts[p]);
      }
      load(v0 + 32 < a.VP ? v0 + 32 : v0);
      __syncthreads();
      uint4 et[TILES][3];  // e of this wave's tiles' columns
#pragma unroll
      for (int x = 0; x < TILES; ++x)
#pragma unroll
        for (int p = 0; p < 3; ++p) et[x][p] = st[(jt[x] * UNIT + NP + 3 + p) * 64 + lane];
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        uint4 da[NP], ra[3], ea[3];
        const uint4* from = st + (m0 + m) * UNIT * 64 + lane;
#pragma unroll
        for (int p = 0; p < NP; ++p) da[p] = from[p * 64];
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          ra[p] = from[(NP + p) * 64];
          ea[p] = from[(NP + 3 + p) * 64];
        }
#pragma unroll
        for (int t = 0; t < NT; ++t)  // the three in turn, so that none waits for its own last product
#pragma unroll
          for (int z = 2; z >= 0; --z)
#pragma unroll
            for (int p = 0; p <= z; ++p) {
              dr[m][t] = mma(ra[p], sb[t][z - p], dr[m][t]);
              if (p < NP) dq[m][t] = mma(da[p], sb[t][z - p], dq[m][t]);
              dw[m][t] = mma(ea[p], db[t][z - p], dw[m][t]);
            }
        if constexpr (MR == 4) {
#pragma unroll
          for (int x = 0; x < TILES; ++x)
            if (it[x] == m)
#pragma unroll
              for (int z = 2; z >= 0; --z)
#pragma unroll
                for (int p = 0; p <= z; ++p) {
                  me[x] = mma(ra[p], et[x][z - p], me[x]);
                  if (p < NP) ne[x] = mma(da[p], et[x][z - p], ne[x]);
                }
        }
        __builtin_amdgcn_sched_barrier(0);  // (all tiles' operands at once would not fit the registers)
      }
      if constexpr (MR < 4) {
#pragma unroll
        for (int x = 0; x < TILES; ++x)
          if (it[x] >= 0) {
            uint4 da[NP], ra[3];
            const uint4* from = st + it[x] * UNIT * 64 + lane;
#pragma unroll
            for (int p = 0; p < NP; ++p) da[p] = from[p * 64];
#pragma unroll
            for (int p = 0; p < 3; ++p) ra[p] = from[(NP + p) * 64];
#pragma unroll
            for (int z = 2; z >= 0; --z)
#pragma unroll
              for (int p = 0; p <= z; ++p) {
                me[x] = mma(ra[p], et[x][z - p], me[x]);
                if (p < NP) ne[x] = mma(da[p], et[x][z - p], ne[x]);
              }
          }
      }
    }
    // N and M, row i and column j
#pragma unroll
    for (int x = 0; x < TILES; ++x) {
      if (it[x] >= 0) {
        const int j = 16 * jt[x] + c;
        const float2 gj = gs[j];
        const float bj = beta[j];
        float nv[4], mv[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * it[x] + 4 * g + r;
          const float d = j <= i ? bj * gdr_decay(gs[i], gj) : 0.f;
          nv[r] = j <= i ? a.scale * d * ne[x][r] : 0.f;
          mv[r] = j < i ? -beta[i] * d * me[x][r] : 0.f;
          if (it[x] == jt[x] && i == j) db[i] = me[x][r];
        }
        const int up = tri_upper(jt[x], it[x] >> 1) * 3 * 64 + lane, low = tri_lower(it[x], jt[x] >> 1) * 3 * 64;
        const int to = 4 * g + 16 * (c >> 2), at = (c & 3) + 4 * (jt[x] & 1);  // of element r = 0 among N's own
        bf16x4 parts[3];
        split_parts<3, 4>(nv, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          nf[1][up + p * 64][it[x] & 1] = __builtin_bit_cast(uint2, parts[p]);
#pragma unroll
          for (int r = 0; r < 4; ++r) reinterpret_cast<__bf16*>(&nf[0][low + p * 64 + to + r])[at] = parts[p][r];
        }
        split_parts<3, 4>(mv, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) {
          mf[1][up + p * 64][it[x] & 1] = __builtin_bit_cast(uint2, parts[p]);
#pragma unroll
          for (int r = 0; r < 4; ++r) reinterpret_cast<__bf16*>(&mf[0][low + p * 64 + to + r])[at] = parts[p][r];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    uint4 kb[2][NT][NP], qb[2][NT][NP];
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          kb[s][t][p] = a.ktf[kbase + (((cw * NT + t) * 2 + s) * NP + p) * 64 + lane];
          qb[s][t][p] = a.qtf[kbase + (((cw * NT + t) * 2 + s) * NP + p) * 64 + lane];
        }
    auto element = [&](const uint4 (&x)[NP], int i) {  // of a fragment, all parts
      float v = 0.f;
#pragma unroll
      for (int p = NP - 1; p >= 0; --p) v += static_cast<float>(__builtin_bit_cast(bf16x8, x[p])[i]);
      return v;
    };
    float last = m0 ? 0.f : grown[63] * dot;  // and the sum of k . ((E U) dS'^T): this lane's share
#pragma unroll
    for (int m = 0; m < MR; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * (m0 + m) + 4 * g + r;
        const float sg = a.scale * grown[i], bg = -beta[i] * grown[i], eb = rest[i] * beta[i];
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          dq[m][t][r] *= sg;
          dr[m][t][r] *= bg;
          dw[m][t][r] *= eb;
          last += element(MR == 4 ? kb[m >> 1][t] : m0 ? kb[1][t] : kb[0][t], 4 * (m & 1) + r) * dw[m][t][r];
        }
      }
    last = wave_sum_rows(last);
    if (lane == 0) dots[wave] = last;
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        const int mt = m0 + m;
        uint4 xa[3], ya[3];
        if (s == 0 || mt >= 2) {
          const int f = tri_lower(mt, s) * 3 * 64 + lane;
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            xa[p] = *reinterpret_cast<const uint4*>(&nf[0][f + p * 64]);
            ya[p] = *reinterpret_cast<const uint4*>(&mf[0][f + p * 64]);
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            dq[m][t] = mma_parts<3, NP>(xa, kb[s][t], dq[m][t]);
            dr[m][t] = mma_parts<3, NP>(ya, kb[s][t], dr[m][t]);
          }
        }
        if (s == 1 || mt < 2) {
          const int f = tri_upper(mt, s) * 3 * 64 + lane;
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            xa[p] = *reinterpret_cast<const uint4*>(&nf[1][f + p * 64]);
            ya[p] = *reinterpret_cast<const uint4*>(&mf[1][f + p * 64]);
          }
#pragma unroll
          for (int t = 0; t < NT; ++t) {
            dw[m][t] = mma_parts<3, NP>(xa, qb[s][t], dw[m][t]);
            dw[m][t] = mma_parts<3, NP>(ya, kb[s][t], dw[m][t]);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    // dG over this wave's columns
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      float x[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int t = 0; t < NT; ++t)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int half = MR == 4 ? m >> 1 : m0 >> 1;
          x[r] += element(half ? qb[1][t] : qb[0][t], 4 * (m & 1) + r) * dq[m][t][r] +
                  element(half ? kb[1][t] : kb[0][t], 4 * (m & 1) + r) * (dr[m][t][r] - dw[m][t][r]);
          dqs[m][t][r] += dq[m][t][r];
          dks[m][t][r] += dr[m][t][r] + dw[m][t][r];
        }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        x[r] = row16_sum(x[r]);
        if (c == 0) dg_part[cw][16 * (m0 + m) + 4 * g + r] = x[r];
      }
    }
    __syncthreads();
    if (wave == 0) {
      double s = 0.;
#pragma unroll
      for (int w = 0; w < CW; ++w) s += (double)dg_part[w][lane];
      // after a token whose e is not finite later ones may be finite here, where the recurrence's are not; their
      // dq is not, so neither is dG
      const float dbeta = db[lane] + (float)s * 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) s += lane == 63 ? (double)dots[w] : 0.;
#pragma unroll
      for (int off = 1; off < 64; off <<= 1) {
        const double t = __shfl_down(s, off, 64);
        if (lane + off < 64) s += t;
      }
      if (lane < rows) {
        store_param(a.dg, a.g_dtype, (token + lane) * a.Hv + h, (float)s);
        store_param(a.dbeta, a.b_dtype, (token + lane) * a.Hv + h, dbeta);
      }
    }
    // (the next head's gs, grown .. are wave 0's to write and read after its first barrier; what else is
    // written then has no readers left, or comes after two barriers)
  }
  const int c = tid & 15, g = (tid & 63) >> 4;
#pragma unroll
  for (int m = 0; m < MR; ++m)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * (m0 + m) + 4 * g + r;
      if (i >= rows) continue;
      const int64_t o = ((token + i) * a.Hk + hk) * (int64_t)a.K;
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        const int col = 16 * (cw * NT + t) + c;
        if (col < a.K) {
          static_cast<T*>(a.dq)[o + col] = from_f32<T>(dqs[m][t][r]);
          static_cast<T*>(a.dk)[o + col] = from_f32<T>(dks[m][t][r]);
        }
      }
    }
}

template <typename T, int KP>
int launch(const GdrArgs& a, hipStream_t s) {
  const int64_t grid = (a.n * a.Hv + 7) / 8 * 8 * (a.VP / 16);  // of each chain
  for (int64_t first = 0; first < grid; first += kGdrBlocks) {
    const dim3 c(2 * (unsigned)(grid - first < kGdrBlocks ? grid - first : kGdrBlocks));
    if (a.V % 16 == 0 || a.V % 16 >= 4) hipLaunchKernelGGL((gdr_chains_kernel<T, KP, true>), c, dim3(512), 0, s, a, first);
    else hipLaunchKernelGGL((gdr_chains_kernel<T, KP, false>), c, dim3(512), 0, s, a, first);
    if (int rc = check_launch("gdr_chains_kernel")) return rc;
  }
  if (a.T == 0) return ATK_OK;
  const dim3 g((unsigned)a.slots, (unsigned)a.Hk);
  if (a.V % 8 == 0) hipLaunchKernelGGL((gdr_grads_kernel<T, KP, true>), g, dim3(512), 0, s, a);
  else hipLaunchKernelGGL((gdr_grads_kernel<T, KP, false>), g, dim3(512), 0, s, a);
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
  if (p->T > 0)
    if (int r = gdr_prepare(a, p->dtype, true, s)) return r;
  if (p->dtype == ATK_F32) return launch_sized<float>(a, s);
  if (p->dtype == ATK_F16) return launch_sized<_Float16>(a, s);
  return launch_sized<__bf16>(a, s);
}

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

// Running sum over the wave of v / ln 2 in 64 bits, as two floats each; lane 63's sum in *last.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
  const uint64_t u = __builtin_bit_cast(uint64_t, v);
  const uint32_t lo = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)u, CTRL, ROWS, 0xF, false);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)(uint32_t)(u >> 32), CTRL, ROWS, 0xF, false);
  return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ float2 running_sum(float v, float2* last) {
  double s = (double)v * 1.4426950408889634;
  s += dpp_f64<0x111, 0xF>(s);  // row_shr 1, 2, 4, 8: sums within 16 lanes
  s += dpp_f64<0x112, 0xF>(s);
  s += dpp_f64<0x114, 0xF>(s);
  s += dpp_f64<0x118, 0xF>(s);
  s += dpp_f64<0x142, 0xA>(s);  // row_bcast 15 into rows 1 and 3
  s += dpp_f64<0x143, 0xC>(s);  // row_bcast 31 into rows 2 and 3
  const float2 r = make_float2((float)s, (float)(s - (double)(float)s));
  last->x = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, r.x), 63));
  last->y = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, r.y), 63));
  return r;
}

// element J of each row of 16 lanes, in all of the row's lanes
template <int J>
__device__ __forceinline__ float row_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + J, 0xF, 0xF, false));
}
template <int I, int J>
__device__ __forceinline__ void substitute(const float (&a)[16], float (&x)[16], float s) {
  if constexpr (J < I) substitute<I, J + 1>(a, x, s - row_lane<J>(a[I]) * x[J]);
  else x[I] = s;
}
template <int I>
__device__ __forceinline__ void substitute_rows(const float (&a)[16], float (&x)[16], int c) {
  if constexpr (I < 16) {
    substitute<I, 0>(a, x, I == c ? 1.f : 0.f);
    substitute_rows<I + 1>(a, x, c);
  }
}

// T = (1 + A)^-1 in the place of the strictly lower A (LDS, 64 x LD; read below the diagonal only), in
// three steps with a barrier after each.  First the four 16 x 16 diagonal blocks, by one wave: forward
// substitution, which is stable whatever A holds; 16 lanes have a block, a column of T each, and a row
// of A at a time, whose elements a lane takes from its neighbours.
__device__ __forceinline__ void invert_diagonal(float* A, int lane) {
  const int c = lane & 15, g = lane >> 4;
  const int at = 16 * g * LD + 16 * g + c;
  float a[16], x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) a[i] = A[at + i * LD];
  substitute_rows<0>(a, x, c);
#pragma unroll
  for (int i = 0; i < 16; ++i) A[at + i * LD] = x[i];
  if (!(g & 1)) {  // the tiles right of the first and third, which fragments of 32 columns take with them
#pragma unroll
    for (int i = 0; i < 16; ++i) A[at + i * LD + 16] = 0.f;
  }
}
// tile (i, k) times tile (k, j), or times a result already in registers
__device__ __forceinline__ f32x4 tile_mul(const float* A, int i, int k, int j, f32x4 s, int lane) {
  const int c = lane & 15, g = lane >> 4;
  const f32x4 x = *reinterpret_cast<const f32x4*>(A + (16 * i + c) * LD + 16 * k + 4 * g);
#pragma unroll
  for (int r = 0; r < 4; ++r)
    s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], A[(16 * k + 4 * g + r) * LD + 16 * j + c], s, 0, 0, 0);
  return s;
}
__device__ __forceinline__ f32x4 tile_mul(const float* A, int i, int k, f32x4 y, f32x4 s, int lane) {
  const int c = lane & 15, g = lane >> 4;
  const f32x4 x = *reinterpret_cast<const f32x4*>(A + (16 * i + c) * LD + 16 * k + 4 * g);
#pragma unroll
  for (int r = 0; r < 4; ++r) s = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r], y[r], s, 0, 0, 0);
  return s;
}
__device__ __forceinline__ void tile_put(float* Tm, int i, int j, f32x4 v, int lane) {
  const int c = lane & 15, g = lane >> 4;
#pragma unroll
  for (int r = 0; r < 4; ++r) Tm[(16 * i + 4 * g + r) * LD + 16 * j + c] = -v[r];
}
// Then blocks of 32 from blocks of 16, and 64 from 32, on fp32 MFMA: the lower left is
// -T22 A21 T11.  All four waves call it; barriers inside and at the end.
__device__ __forceinline__ void invert_below(float* A, int wave, int lane) {
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (wave < 2) {
    const int i = 2 * wave + 1, j = 2 * wave;
    tile_put(A, i, j, tile_mul(A, i, i, tile_mul(A, i, j, j, zero, lane), zero, lane), lane);
  }
  __syncthreads();
  const int i = 2 + (wave >> 1), j = wave & 1;
  f32x4 y = zero, t = zero;
  for (int k = 2; k <= i; ++k) {
    y = tile_mul(A, k, 1, j, zero, lane);  // (tile (0, 1) of T is zero)
    if (j == 0) y = tile_mul(A, k, 0, j, y, lane);
    t = tile_mul(A, i, k, y, t, lane);
  }
  __syncthreads();  // the lower left is still A's until every wave is past it
  tile_put(A, i, j, t, lane);
  __syncthreads();
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

// 32 rows' worth of a product's results, scaled, as one fragment of the transposed product
template <int P>
__device__ __forceinline__ void write_products(const f32x4& lo, const f32x4& hi, uint4* __restrict__ out, int lane) {
  const float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  bf16x8 parts[P];
  split_parts<P, 8>(v, parts);
#pragma unroll
  for (int p = 0; p < P; ++p) out[p * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
}

// A workgroup for each (chunk, value head); the first value head of a key head's group also writes
// that key head's K and K^T (and Q^T).  The masked products leave the registers as fragments: a
// product's result has the layout of its transpose's rows, so Q K^T comes out of K Q^T.
template <typename T, int KP, bool BWD>
__global__ __launch_bounds__(256) void gdr_prepare_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32, PP = BWD ? 3 : kOutParts<T>;
  __shared__ uint4 kl[KS * 4 * NP * 64];  // K's fragments, then Q's
  __shared__ __align__(16) float wm[64 * LD];
  __shared__ float2 gd[64];
  __shared__ float bs[64];
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t slot = blockIdx.x;
  const int h = blockIdx.y, hk = h / a.group;
  const int64_t n = gdr_seq_of_slot(a.cu, a.T, a.n, slot);
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t at = (slot - seq.slot) * kGdrC;  // the chunk's first token within the sequence
  if (at < 0 || at >= seq.len) return;
  const int rows = (int)(seq.len - at < kGdrC ? seq.len - at : kGdrC);
  const int64_t t0 = seq.begin + at;
  const bool owner = h % a.group == 0;
  const int64_t kbase = (hk * a.slots + slot) * (int64_t)(KS * 4 * NP * 64);
  const int64_t tbase = (h * a.slots + slot) * (int64_t)(kTri * 3 * 64);
  float gv = 0.f, bv = 0.f;
  if (wave == 0 && lane < rows) {
    gv = load_param(a.g, a.g_dtype, seq.batch * a.g_s[0] + (t0 + lane) * a.g_s[1] + h * a.g_s[2]);
    bv = load_param(a.beta, a.b_dtype, seq.batch * a.b_s[0] + (t0 + lane) * a.b_s[1] + h * a.b_s[2]);
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
      load4(k, 32 * s + 4 * g, a.K, live, v);
      load4(k, 32 * s + 16 + 4 * g, a.K, live, v + 4);
      split_parts<NP, 8>(v, parts);
#pragma unroll
      for (int p = 0; p < NP; ++p) kr[s][p] = __builtin_bit_cast(uint4, parts[p]);
      load4(q, 32 * s + 4 * g, a.K, live, v);
      load4(q, 32 * s + 16 + 4 * g, a.K, live, v + 4);
      split_parts<NP, 8>(v, parts);
#pragma unroll
      for (int p = 0; p < NP; ++p) qr[s][p] = __builtin_bit_cast(uint4, parts[p]);
    }
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        kl[((s * 4 + wave) * NP + p) * 64 + lane] = kr[s][p];
        if (owner) a.kf[kbase + ((s * 4 + wave) * NP + p) * 64 + lane] = kr[s][p];
        if (!BWD && owner) a.qf[kbase + ((s * 4 + wave) * NP + p) * 64 + lane] = qr[s][p];
      }
  }
  if (wave == 0) {
    float2 last;
    // below -120 the decay is 0 in fp32 whatever follows, and sums with -inf have no differences
    const float2 s = running_sum(gv < -120.f ? -120.f : gv, &last);
    gd[lane] = s;
    bs[lane] = bv;
    if constexpr (BWD) a.gsum[(h * a.slots + slot) * 64 + lane] = s;
    float* __restrict__ row = a.row + (h * a.slots + slot) * 192;
    row[lane] = gdr_decay(s, make_float2(0.f, 0.f));
    row[64 + lane] = gdr_decay(last, s);
    row[128 + lane] = bv;
  }
  __syncthreads();
  // rows 16 wave .. of W = strictly lower K K^T * D, its columns times beta, into wm
  f32x4 w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    w[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (j <= wave) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 b[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) b[p] = kl[((s * 4 + j) * NP + p) * 64 + lane];
        w[j] = mma_parts<NP, NP>(kr[s], b, w[j]);
      }
      const int cj = 16 * j + c;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * wave + 4 * g + r;
        w[j][r] = cj < i ? w[j][r] * gdr_decay(gd[i], gd[cj]) : 0.f;
        wm[i * LD + cj] = w[j][r] * bs[cj];
      }
    }
  }
  if (owner) write_columns<KP, NP>(kl, a.ktf + kbase, wave, lane);
  __syncthreads();
  if constexpr (BWD) {  // Q in K's place
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int p = 0; p < NP; ++p) kl[((s * 4 + wave) * NP + p) * 64 + lane] = qr[s][p];
    __syncthreads();
  }
  if (wave == 0) invert_diagonal(wm, lane);
  {
    // forward: (Q K^T)^T = K Q^T, columns 16 wave .., row tiles up to the diagonal; backward: Q K^T,
    // columns 16 wave .., row tiles from the diagonal on
    const int col = 16 * wave + c;
    const float2 gc = gd[col];
    for (int s = BWD ? wave >> 1 : 0; s < (BWD ? 2 : (wave >> 1) + 1); ++s) {
      f32x4 y[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int j = 2 * s + u;
        y[u] = f32x4{0.f, 0.f, 0.f, 0.f};
        if (BWD ? j >= wave : j <= wave) {
#pragma unroll
          for (int z = 0; z < KS; ++z) {
            uint4 b[NP];
#pragma unroll
            for (int p = 0; p < NP; ++p) b[p] = kl[((z * 4 + j) * NP + p) * 64 + lane];
            y[u] = mma_parts<NP, NP>(b, BWD ? kr[z] : qr[z], y[u]);
          }
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 16 * j + 4 * g + r;
            if constexpr (BWD) y[u][r] = i >= col ? y[u][r] * gdr_decay(gd[i], gc) : 0.f;
            else y[u][r] = i <= col ? y[u][r] * gdr_decay(gc, gd[i]) : 0.f;
          }
        }
      }
      write_products<PP>(y[0], y[1], (BWD ? a.ptf + tbase + tri_upper(wave, s) * PP * 64
                                          : a.pf + (h * a.slots + slot) * (int64_t)(kTri * PP * 64) + tri_lower(wave, s) * PP * 64), lane);
    }
    if constexpr (BWD)
      if (owner) write_columns<KP, NP>(kl, a.qtf + kbase, wave, lane);
  }
  __syncthreads();
  invert_below(wm, wave, lane);
  write_lower(wm, a.tf + tbase, wave, lane);
  if constexpr (BWD) {  // and (1 + diag(beta) W)^-1, transposed
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j <= wave)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * wave + 4 * g + r;
          wm[i * LD + 16 * j + c] = bs[i] * w[j][r];
        }
    __syncthreads();
    if (wave == 0) invert_diagonal(wm, lane);
    __syncthreads();
    invert_below(wm, wave, lane);
    write_transposed(wm, a.ttf + tbase, wave, lane);
  }
}

// The state's chain: 16 value columns of one head's state, all of its key rows, from chunk to chunk.
//
// What bounds it is the time of one step, since a step needs the one before it: three products that
// follow each other (K S, T X, K^T E U).  Four waves share them: wave w has the state's row tiles
// w MT .. in its accumulators, multiplies them as they are (their layout is B's) with the K of all 64
// tokens, and the four partial sums meet in LDS; then it has the tokens 16 w .. for X and e.  So the
// state itself never leaves the registers.  Fragments are loaded right after their last use, for the
// next chunk: a load has most of a step to arrive.  Four more waves bring V into LDS a chunk ahead and
// make the chunk's outputs, off the chain.  A barrier orders LDS only; loads stay in flight across it.
// All value tiles of a head read the same fragments, so each brings its share of the lines of the chunk
// after next into their L2 (a word of each): what the next chunk's loads then find there took a step
// longer than they have.
// FULL: no tile of value columns ends in one of fewer than 4, so a lane has 4 columns of a token in one
// load or store (the last of a tile that V ends in overlap).
template <typename T, int KP, bool KEEP, bool FULL>
__global__ __launch_bounds__(512) void gdr_chain_kernel(GdrArgs a) {
  constexpr int NP = kParts<T>, KS = KP / 32, MT = KP / 64, KW = MT > 1 ? MT / 2 : 1, OP = kOutParts<T>;
  constexpr int KF = KS * 4 * NP * 64;
  __shared__ f32x4 kp[4][4][64];                      // partial sums [state wave][token tile][lane]
  __shared__ uint2 xl[2][3][64][2], el[2][3][64][2];  // X and E U in parts, as B is read
  __shared__ f32x4 vl[4][64];                         // V
  __shared__ __align__(16) float rl[192];             // the chunk's decays and betas
  __shared__ T ol[KEEP ? 1 : 4][16][20];              // an output tile on its way to rows
  __shared__ uint4 sl[KEEP ? 1 : KS][3][64];          // the state in parts, for the outputs
  __shared__ f32x4 ul[KEEP ? 1 : 4][64];              // U, fp32
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile, h;
  int64_t n;
  const int tiles = KEEP ? a.VP / 16 : (a.V + 15) / 16;
  if (!gdr_chain_place(a, tiles, &tile, &h, &n)) return;
  const int hk = h / a.group, col = tile * 16 + c;
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t chunks = (seq.len + kGdrC - 1) / kGdrC;
  constexpr int rstep = 192;
  const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
  if (wave < 4) {
    const int s0 = MT == 1 ? wave / 2 : wave * KW;  // this wave's first 32 key columns
    const uint4* __restrict__ kf = a.kf + (hk * a.slots + seq.slot) * KF + s0 * 4 * NP * 64;
    const uint4* __restrict__ ktf = a.ktf + (hk * a.slots + seq.slot) * KF + wave * MT * 2 * NP * 64;
    const uint4* __restrict__ tf = a.tf + (h * a.slots + seq.slot) * (int64_t)(kTri * 3 * 64) + tri_lower(wave, 0) * 3 * 64;
    constexpr int kstep = KF, tstep = kTri * 3 * 64;
    const bool two = wave >= 2;  // column halves of this wave's rows of T
    f32x4 S[MT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * (wave * MT + m) + 4 * g + r;
        S[m][r] = a.s0 && i < a.K && col < a.V ? a.s0[((n * a.Hv + h) * a.K + i) * a.V + col] : 0.f;
      }
    // here, and not in every pass of the loop, the compiler waits for these loads
#pragma unroll
    for (int m = 0; m < MT; ++m) asm volatile("" : "+v"(S[m]));
    uint4 ka[KW][4][NP], ta[2][3], kta[2][MT][NP];
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
    if (chunks > 0) {
      load_k();
      load_t();
      load_kt();
    }
    __syncthreads();  // the first V and decays
    for (int64_t ch = 0; ch < chunks; ++ch) {
      // No branches around loads: where paths with and without them meet, the compiler waits for all.
      // (At the end the last chunk's are loaded again.)
      const bool more = ch + 1 < chunks;
      kf += more ? kstep : 0;
      ktf += more ? kstep : 0;
      tf += more ? tstep : 0;
      if constexpr (KEEP) {
        float* __restrict__ sc = a.sc + (h * a.slots + seq.slot + ch) * (int64_t)KP * a.VP + gdr_kept(tile, KP / 16, c, g);
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int r = 0; r < 4; ++r) sc[(wave * MT + m) * 512 + r * 8] = S[m][r];
      }
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
        if constexpr (!KEEP) {
#pragma unroll
          for (int p = 0; p < 3; ++p) {
            if (MT > 1) sl[s0 + s][p][lane] = sp[p];
            else reinterpret_cast<uint2*>(&sl[s0][p][lane])[wave & 1] = (wave & 1) ? make_uint2(sp[p].z, sp[p].w) : make_uint2(sp[p].x, sp[p].y);
          }
        }
        mma_tiles<4, NP, 3>(ka[s], sp, y);
      }
      load_k();
#pragma unroll
      for (int m = 0; m < 4; ++m) kp[wave][m][lane] = y[m];
      __syncthreads();
      {
        const f32x4 v = vl[wave][lane], y0 = kp[0][wave][lane], y1 = kp[1][wave][lane], y2 = kp[2][wave][lane], y3 = kp[3][wave][lane];
        const f32x4 grown = *reinterpret_cast<const f32x4*>(&rl[16 * wave + 4 * g]);
        const f32x4 z = (y0 + y1) + (y2 + y3);
        float x[4];
        bf16x4 parts[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = v[r] - grown[r] * z[r];
        split_parts<3, 4>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) xl[wave >> 1][p][lane][wave & 1] = __builtin_bit_cast(uint2, parts[p]);
      }
      const f32x4 rest = *reinterpret_cast<const f32x4*>(&rl[64 + 16 * wave + 4 * g]);
      const f32x4 beta = *reinterpret_cast<const f32x4*>(&rl[128 + 16 * wave + 4 * g]);
      const float all = rl[63];
      __syncthreads();
      f32x4 e;
      {
        f32x4 part[3] = {zero, zero, zero};  // three sums, so that no product waits for the one before it
        uint4 b[2][3];
#pragma unroll
        for (int p = 0; p < 3; ++p) b[0][p] = *reinterpret_cast<const uint4*>(&xl[0][p][lane]);
        if (two)
#pragma unroll
          for (int p = 0; p < 3; ++p) b[1][p] = *reinterpret_cast<const uint4*>(&xl[1][p][lane]);
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
        e = (part[0] + part[1]) + part[2];
      }
      {
        float x[4];
        bf16x4 parts[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = rest[r] * beta[r] * e[r];
        split_parts<3, 4>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) el[wave >> 1][p][lane][wave & 1] = __builtin_bit_cast(uint2, parts[p]);
        if constexpr (KEEP) {
          float* __restrict__ ec = a.ec + (h * a.slots + seq.slot + ch) * (int64_t)64 * a.VP + gdr_kept(tile, 4, c, g);
#pragma unroll
          for (int r = 0; r < 4; ++r) ec[wave * 512 + r * 8] = e[r];
        } else {
          ul[wave][lane] = beta * e;
        }
      }
      load_t();
      __syncthreads();
      {
        f32x4 z[MT];
        uint4 b[2][3];
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
          for (int p = 0; p < 3; ++p) b[s][p] = *reinterpret_cast<const uint4*>(&el[s][p][lane]);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int m = 0; m < MT; ++m) {
          S[m] *= all;
          z[m] = zero;
        }
        // (the second half first: the decayed state is not needed yet)
        mma_tiles<MT, NP, 3>(kta[1], b[1], z);
        mma_tiles<MT, NP, 3>(kta[0], b[0], S);
#pragma unroll
        for (int m = 0; m < MT; ++m) S[m] += z[m];
      }
      load_kt();
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
  } else {
    const int m = wave - 4;
    // V and the outputs by rows: this lane's token of a chunk, and its 4 columns of the tile
    const int tok = 16 * m + (lane >> 2);
    const bool dead = KEEP && tile * 16 >= a.V;  // a tile of padding: V of zeros
    const int c4 = FULL && !dead ? (tile * 16 + 4 * (lane & 3) + 4 <= a.V ? 4 * (lane & 3) : a.V - 4 - tile * 16) : 4 * (lane & 3);
    const T* __restrict__ vp = static_cast<const T*>(a.v) + seq.batch * a.v_s[0] + seq.begin * a.v_s[1] + h * a.v_s[2] +
                               (dead ? 0 : tile * 16 + (FULL ? c4 : 0));
    const int64_t vlane = tok * a.v_s[1], vstep = kGdrC * a.v_s[1];
    const float* __restrict__ row = a.row + (h * a.slots + seq.slot) * 192 + (m < 3 ? m : 0) * 64 + lane;
    T va[4];
    float ra;
    // Tokens past the end: the chunk's first instead (their beta is 0, and they are not stored).
    auto load_v = [&](int64_t left) {
      const T* __restrict__ p = vp + (tok < left ? vlane : 0);
      if constexpr (FULL) {
        __builtin_memcpy(va, p, 4 * sizeof(T));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) va[j] = p[tile * 16 + c4 + j < a.V ? c4 + j : 0];
      }
      ra = *row;
    };
    auto load_next_v = [&](int64_t left) {  // from a chunk with `left` tokens to go; the last one's again
      vp += left > kGdrC ? vstep : 0;
      row += left > kGdrC ? rstep : 0;
      load_v(left > kGdrC ? left - kGdrC : left);
    };
    auto put_v = [&]() {
#pragma unroll
      for (int j = 0; j < 4; ++j) vl[m][16 * (lane >> 4) + c4 + j][(lane >> 2) & 3] = dead ? 0.f : to_f32(va[j]);
      if (m < 3) rl[64 * m + lane] = ra;
    };
    vl[m][lane] = zero;  // columns past V keep it
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses keep their order)
    if (chunks > 0) {
      load_v(seq.len);
      put_v();
      load_next_v(seq.len);
    }
    if constexpr (KEEP) {
      __syncthreads();
      for (int64_t ch = 0; ch < chunks; ++ch) {
        __syncthreads();
        __syncthreads();
        put_v();  // the next chunk's: this one's was read before this barrier
        __syncthreads();
        load_next_v(seq.len - (ch + 1) * kGdrC);
      }
    } else {
      const uint4* __restrict__ qf = a.qf + (hk * a.slots + seq.slot) * KF + m * NP * 64;
      const uint4* __restrict__ pf = a.pf + (h * a.slots + seq.slot) * (int64_t)(kTri * OP * 64) + tri_lower(m, 0) * OP * 64;
      constexpr int qstep = KF, pstep = kTri * OP * 64;
      const bool two = m >= 2;
      const int64_t os = (int64_t)a.Hv * a.V;
      T* __restrict__ o = static_cast<T*>(a.o) + ((seq.batch * a.T + seq.begin + tok) * a.Hv + h) * (int64_t)a.V + tile * 16 + c4;
      T* __restrict__ dump = reinterpret_cast<T*>(a.dump) + 4 * lane;
      uint4 pa[2][OP], qa[KS][NP];
      auto load_q = [&]() {
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int p = 0; p < NP; ++p) qa[s][p] = qf[(s * 4 * NP + p) * 64 + lane];
      };
      // the lines of K, Q, K^T, T and P in turn; this lane's among them, if there is one left for it
      constexpr int LK = KF / 8, LT = kTri * 3 * 8, LP = kTri * OP * 8, LINES = 3 * LK + LT + LP;
      int line = (tile * 4 + m) * 64 + lane;
      line = line < LINES ? line : LINES - 1;
      const uint4* ahead = line < LK       ? a.kf + (hk * a.slots + seq.slot) * KF + line * 8
                           : line < 2 * LK ? a.qf + (hk * a.slots + seq.slot) * KF + (line - LK) * 8
                           : line < 3 * LK ? a.ktf + (hk * a.slots + seq.slot) * KF + (line - 2 * LK) * 8
                           : line < 3 * LK + LT ? a.tf + (h * a.slots + seq.slot) * (int64_t)(kTri * 3 * 64) + (line - 3 * LK) * 8
                                                : a.pf + (h * a.slots + seq.slot) * (int64_t)(kTri * OP * 64) + (line - 3 * LK - LT) * 8;
      const int ahead_step = line < 3 * LK ? KF : line < 3 * LK + LT ? kTri * 3 * 64 : kTri * OP * 64;
      ahead += (chunks > 2 ? 2 : 0) * ahead_step;
      uint32_t seen = 0;
      auto touch = [&](bool another) {
        asm volatile("" ::"v"(seen));  // (the load before this one has arrived by now)
        ahead += another ? ahead_step : 0;
        seen = *reinterpret_cast<const uint32_t*>(ahead);
      };
      auto load_p = [&]() {
#pragma unroll
        for (int p = 0; p < OP; ++p) pa[0][p] = pf[p * 64 + lane];
#pragma unroll
        for (int p = 0; p < OP; ++p) pa[1][p] = pf[((two ? OP : 0) + p) * 64 + lane];
      };
      f32x4 y, z;
      auto q_s = [&](int from, int to) {  // Q S over key columns 32 from .. 32 to
#pragma unroll
        for (int s = from; s < to; ++s) {
          uint4 b[3];
#pragma unroll
          for (int p = 0; p < 3; ++p) b[p] = sl[s][p][lane];
          if (s & 1) z = mma_parts<NP, 3>(qa[s], b, z);
          else y = mma_parts<NP, 3>(qa[s], b, y);
        }
      };
      if (chunks > 0) {
        load_q();
        load_p();
      }
      __syncthreads();
      for (int64_t ch = 0; ch < chunks; ++ch) {
        const int64_t left = seq.len - ch * kGdrC;
        const bool more = left > kGdrC;
        __syncthreads();
        // sl is this chunk's for two barriers
        y = z = zero;
        q_s(0, KS / 2);
        const f32x4 grown = *reinterpret_cast<const f32x4*>(&rl[16 * m + 4 * g]);
        __syncthreads();
        put_v();  // the next chunk's: vl's and rl's readers are past this barrier
        q_s(KS / 2, KS);
        qf += more ? qstep : 0;
        load_q();
        load_next_v(more ? left - kGdrC : left);
        touch(ch + 3 < chunks);
        __syncthreads();
        // ul is this chunk's for two barriers
        y = (y + z) * grown;
        z = zero;
        auto half = [&](int s, f32x4 w) {
          bf16x8 parts[OP];
          uint4 b[OP];
          const f32x4 lo = ul[2 * s][lane], hi = ul[2 * s + 1][lane];
          const float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          split_parts<OP, 8>(x, parts);
#pragma unroll
          for (int p = 0; p < OP; ++p) b[p] = __builtin_bit_cast(uint4, parts[p]);
          return mma_parts<OP, OP>(pa[s], b, w);
        };
        y = half(0, y);
        if (two) z = half(1, z);
        y += z;
        // loads before the store: what waits for them would wait for a store in front of them too
        pf += more ? pstep : 0;
        load_p();
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int r = 0; r < 4; ++r) ol[m][4 * g + r][c] = from_f32<T>(a.scale * y[r]);
        __builtin_amdgcn_wave_barrier();
        T out[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) out[j] = ol[m][lane >> 2][c4 + j];
        // a lane with nothing to store has a place in the workspace for it, rather than a branch
        T* __restrict__ at = tok < left ? o : dump;
        if constexpr (FULL) {
          __builtin_memcpy(at, out, 4 * sizeof(T));
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) *(tile * 16 + c4 + j < a.V ? at + j : dump + j) = out[j];
        }
        o += kGdrC * os;
        __builtin_amdgcn_wave_barrier();
      }
      // tokens of a packed row before its first sequence and after its last have an output of zero
      if (a.cu && (n == 0 || n == a.n - 1)) {
        T* __restrict__ all = static_cast<T*>(a.o);
        const int64_t from[2] = {n == 0 ? 0 : a.T, n == a.n - 1 ? seq.begin + seq.len : a.T};
        const int64_t to[2] = {n == 0 ? seq.begin : a.T, a.T};
        for (int z = 0; z < 2; ++z)
          for (int64_t i = from[z] + 4 * m + g; i < to[z]; i += 16)
            if (col < a.V) all[(i * a.Hv + h) * (int64_t)a.V + col] = from_f32<T>(0.f);
      }
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
  const bool full = a.V % 16 == 0 || a.V % 16 >= 4;
  const dim3 g((unsigned)grid), b(512);
  if (keep && full) hipLaunchKernelGGL((gdr_chain_kernel<T, KP, true, true>), g, b, 0, s, a);
  else if (keep) hipLaunchKernelGGL((gdr_chain_kernel<T, KP, true, false>), g, b, 0, s, a);
  else if (full) hipLaunchKernelGGL((gdr_chain_kernel<T, KP, false, true>), g, b, 0, s, a);
  else hipLaunchKernelGGL((gdr_chain_kernel<T, KP, false, false>), g, b, 0, s, a);
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
  a->kf = reinterpret_cast<uint4*>(take(kb)); a->ktf = reinterpret_cast<uint4*>(take(kb));
  a->tf = reinterpret_cast<uint4*>(take(tb));
  a->dump = take(1024);
  a->row = reinterpret_cast<float*>(take((size_t)a->slots * a->Hv * 768));
  if (!backward) {
    a->qf = reinterpret_cast<uint4*>(take(kb));
    a->pf = reinterpret_cast<uint4*>(take(tb));
    return off;
  }
  const size_t state = (size_t)a->slots * a->Hv * gdr_padded_k(a->K) * a->VP * 4, row = (size_t)a->slots * a->Hv * 64 * a->VP * 4;
  a->qtf = reinterpret_cast<uint4*>(take(kb)); a->ttf = reinterpret_cast<uint4*>(take(tb));
  a->ptf = reinterpret_cast<uint4*>(take(tb));
  a->gsum = reinterpret_cast<float2*>(take((size_t)a->slots * a->Hv * 512));
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
  // A token at a time takes 1.4 us for each, two launches on a chunk 13 to 20 us whatever it holds (1
  // sequence, 16 heads, 128 x 128: 8 tokens 14.0 us against 15.9, 16 tokens 25.3 against 15.1; 16
  // sequences, 32 heads: 8 tokens 43.7 us against 82.0, 16 tokens 80.2 against 81.0).
  if (p->T <= 8) return gdr_tokens(a, p->dtype, s);
  if (int r = gdr_prepare(a, p->dtype, false, s)) return r;
  return gdr_chain(a, p->dtype, false, s);
}

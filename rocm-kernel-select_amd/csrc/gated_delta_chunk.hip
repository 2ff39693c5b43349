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
#include "gated_delta_chain.h"

namespace atk {
namespace {

constexpr int LD = 68;  // row pitch of the fp32 64 x 64 tiles in LDS: 16-byte rows, 4 banks apart

// This lane's elements of a row of K, in gdr_at's order for each 32, and all of its loads at once: with
// a branch around each the compiler waits for each (20 000 of a workgroup's 40 000 cycles, when it did).
template <typename T, int KP, bool FULL>
__device__ __forceinline__ void load_row(const T* __restrict__ p, int K, int g, T (&o)[KP / 32][8]) {
#pragma unroll
  for (int s = 0; s < KP / 32; ++s) {
    if constexpr (FULL) {
      __builtin_memcpy(o[s], p + 32 * s + 4 * g, 4 * sizeof(T));  // element alignment only
      __builtin_memcpy(o[s] + 4, p + 32 * s + 16 + 4 * g, 4 * sizeof(T));
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int d = 32 * s + gdr_at(g, i);
        o[s][i] = p[d < K ? d : 0];
      }
    }
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

// The same row by row, a column of T a lane, for an A that is not finite or whose T is not: there the blocks
// would multiply zeros with what is not, and spoil rows before the first.  One wave; slow, and hardly ever run.
__device__ __forceinline__ void invert_by_rows(float* A) {
  const int lane = gdr_lane();
#pragma nounroll
  for (int i = 0; i < kGdrC; ++i) {
    float t = lane == i ? 1.f : 0.f;
#pragma nounroll
    for (int j = 0; j < i; ++j) t -= A[i * LD + j] * A[j * LD + lane];
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS accesses keep their order)
    A[i * LD + lane] = t;
    __builtin_amdgcn_wave_barrier();
  }
}

// The rows of a lower triangular 64 x 64 matrix (LDS) as fragments in three parts; whether any is not finite.
__device__ __forceinline__ bool write_lower(const float* __restrict__ M, uint4* __restrict__ out, int wave, int lane) {
  const int c = lane & 15, g = lane >> 4;
  bool spoilt = false;
  for (int f = wave; f < kTri; f += 4) {
    const int m = f < 2 ? f : f / 2 + 1, s = f < 2 ? 0 : f & 1;
    float v[8];
    bf16x8 parts[3];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = M[(16 * m + c) * LD + 32 * s + gdr_at(g, i)];
    spoilt |= gdr_spoilt<8>(v);
    split_parts<3, 8>(v, parts);
#pragma unroll
    for (int p = 0; p < 3; ++p) out[(f * 3 + p) * 64 + lane] = __builtin_bit_cast(uint4, parts[p]);
  }
  return spoilt;
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

// A workgroup for each chunk and `heads` value heads of one key head (one or two); the first of a key
// head's group also writes that key head's K, Q and K^T (or K, K^T and Q^T).  K K^T and Q K^T are
// computed once for both.  The masked products leave the registers as fragments: a product's result has
// the layout of its transpose's rows, so Q K^T comes out of K Q^T.  FULL: K is KP.
// Bound by latency: loads, then the products, then the inverse's three dependent steps, then stores
// (bf16, 8192 tokens, 16 and 32 heads of 128: 69 to 74 us for 224 MB written and 35 read, 3.6 TB/s; one
// chunk each of 16 heads: 11 us).
template <typename T, int KP, bool BWD, bool FULL>
__global__ __launch_bounds__(256, (KP * kParts<T> <= 128 ? 4 : 1)) void gdr_prepare_kernel(GdrArgs a, int heads) {
  constexpr int NP = kParts<T>, KS = KP / 32, PP = BWD ? 3 : kOutParts<T>;
  __shared__ uint4 kl[KS * 4 * NP * 64];  // K's fragments, then Q's
  __shared__ __align__(16) float wm[64 * LD];
  __shared__ float2 gd[2][64];
  __shared__ float bs[2][64];
  __shared__ int spoilt[2];  // whether a head's T is not finite
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t slot = blockIdx.x;
  const int h0 = blockIdx.y * heads, hk = h0 / a.group;
  const int64_t n = gdr_seq_of_slot(a.cu, a.T, a.n, slot);
  const GdrSeq seq = gdr_seq(a.cu, a.T, n);
  const int64_t at = (slot - seq.slot) * kGdrC;  // the chunk's first token within the sequence
  if (at < 0 || at >= seq.len) return;
  const int rows = (int)(seq.len - at < kGdrC ? seq.len - at : kGdrC);
  const int64_t t0 = seq.begin + at;
  const bool owner = h0 % a.group == 0;
  const int64_t kbase = (hk * a.slots + slot) * (int64_t)(KS * 4 * NP * 64);
  if (tid < 2) spoilt[tid] = 0;
  uint4 qr[KS][NP], kr[KS][NP];  // this wave's 16 tokens
  {
    const bool live = 16 * wave + c < rows;
    const int64_t tok = t0 + (live ? 16 * wave + c : 0);
    const T* __restrict__ q = static_cast<const T*>(a.q) + seq.batch * a.q_s[0] + tok * a.q_s[1] + hk * a.q_s[2];
    const T* __restrict__ k = static_cast<const T*>(a.k) + seq.batch * a.k_s[0] + tok * a.k_s[1] + hk * a.k_s[2];
    // wave w has the decays of head w
    const int h = h0 + (wave < heads ? wave : 0);
    const int64_t i = t0 + (lane < rows ? lane : 0);
    const GdrGate gr = gdr_gate_load(a.g, a.g_dtype, seq.batch * a.g_s[0] + i * a.g_s[1] + h * a.g_s[2]);
    const GdrGate br = gdr_gate_load(a.beta, a.b_dtype, seq.batch * a.b_s[0] + i * a.b_s[1] + h * a.b_s[2]);
    T kv[KS][8], qv[KS][8];
    load_row<T, KP, FULL>(k, a.K, g, kv);
    load_row<T, KP, FULL>(q, a.K, g, qv);
    if (wave < heads) {
      const float gv = lane < rows ? gdr_gate<T>(gr, a.g_dtype) : 0.f;
      const float bv = lane < rows ? gdr_gate<T>(br, a.b_dtype) : 0.f;
      float2 last;
      // below -120 the decay is 0 in fp32 whatever follows, and sums with -inf have no differences
      const float2 s = running_sum(gv < -120.f ? -120.f : gv, &last);
      gd[wave][lane] = s;
      bs[wave][lane] = bv;
      if constexpr (BWD) a.gsum[(h * a.slots + slot) * 64 + lane] = s;
      float* __restrict__ row = a.row + (h * a.slots + slot) * 192;
      row[lane] = gdr_decay(s, make_float2(0.f, 0.f));
      row[64 + lane] = gdr_decay(last, s);
      row[128 + lane] = bv;
    }
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      float x[8], y[8];
      bf16x8 parts[NP];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool in = live && (FULL || 32 * s + gdr_at(g, i) < a.K);
        x[i] = in ? to_f32(kv[s][i]) : 0.f;
        y[i] = in ? to_f32(qv[s][i]) : 0.f;
      }
      split_parts<NP, 8>(x, parts);
#pragma unroll
      for (int p = 0; p < NP; ++p) kr[s][p] = __builtin_bit_cast(uint4, parts[p]);
      split_parts<NP, 8>(y, parts);
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
  __syncthreads();
  // K K^T, rows 16 wave ..
  f32x4 kk[4], qk[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    kk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (j <= wave) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 b[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) b[p] = kl[((s * 4 + j) * NP + p) * 64 + lane];
        kk[j] = mma_parts<NP, NP>(kr[s], b, kk[j]);
      }
    }
  }
  if (owner) write_columns<KP, NP>(kl, a.ktf + kbase, wave, lane);
  if constexpr (BWD) {  // Q in K's place
    __syncthreads();
#pragma unroll
    for (int s = 0; s < KS; ++s)
#pragma unroll
      for (int p = 0; p < NP; ++p) kl[((s * 4 + wave) * NP + p) * 64 + lane] = qr[s][p];
    __syncthreads();
  }
  // forward: (Q K^T)^T = K Q^T, columns 16 wave .., row tiles up to the diagonal; backward: Q K^T,
  // columns 16 wave .., row tiles from the diagonal on
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    qk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (BWD ? j >= wave : j <= wave) {
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        uint4 b[NP];
#pragma unroll
        for (int p = 0; p < NP; ++p) b[p] = kl[((s * 4 + j) * NP + p) * 64 + lane];
        qk[j] = mma_parts<NP, NP>(b, BWD ? kr[s] : qr[s], qk[j]);
      }
    }
  }
  if constexpr (BWD)
    if (owner) write_columns<KP, NP>(kl, a.qtf + kbase, wave, lane);
  for (int x = 0; x < heads; ++x) {
    const int h = h0 + x;
    const int64_t tbase = (h * a.slots + slot) * (int64_t)(kTri * 3 * 64);
    // W = strictly lower K K^T * D, its columns times beta
    f32x4 w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j <= wave) {
        const int cj = 16 * j + c;
        const float2 gj = gd[x][cj];
        const float bj = bs[x][cj];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int i = 16 * wave + 4 * g + r;
          w[j][r] = cj < i ? kk[j][r] * gdr_decay(gd[x][i], gj) : 0.f;
          wm[i * LD + cj] = w[j][r] * bj;
        }
      }
    __syncthreads();
    if (wave == 0) invert_diagonal(wm, lane);
    {
      const int col = 16 * wave + c;
      const float2 gc = gd[x][col];
#pragma unroll
      for (int s = 0; s < 2; ++s)
        if (BWD ? s >= wave >> 1 : s <= wave >> 1) {
          f32x4 y[2];
#pragma unroll
          for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int i = 16 * (2 * s + u) + 4 * g + r;
              if constexpr (BWD) y[u][r] = i >= col ? qk[2 * s + u][r] * gdr_decay(gd[x][i], gc) : 0.f;
              else y[u][r] = i <= col ? qk[2 * s + u][r] * gdr_decay(gc, gd[x][i]) : 0.f;
            }
          write_products<PP>(y[0], y[1], (BWD ? a.ptf + tbase + tri_upper(wave, s) * PP * 64
                                              : a.pf + (h * a.slots + slot) * (int64_t)(kTri * PP * 64) + tri_lower(wave, s) * PP * 64), lane);
        }
    }
    __syncthreads();
    invert_below(wm, wave, lane);
    if (write_lower(wm, a.tf + tbase, wave, lane)) spoilt[x] = 1;
    __syncthreads();
    if (spoilt[x]) {
      const int l = gdr_lane(), cl = l & 15, gl = l >> 4;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j <= wave)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * gl + r, cj = 16 * j + cl;
            if (cj < i) wm[i * LD + cj] = kk[j][r] * gdr_decay(gd[x][i], gd[x][cj]) * bs[x][cj];
          }
      __syncthreads();
      if (wave == 0) invert_by_rows(wm);
      __syncthreads();
      write_lower(wm, a.tf + tbase, wave, l);
      __syncthreads();
    }
    if constexpr (BWD) {  // and (1 + diag(beta) W)^-1, transposed
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j <= wave)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int i = 16 * wave + 4 * g + r;
            wm[i * LD + 16 * j + c] = bs[x][i] * w[j][r];
          }
      __syncthreads();
      if (wave == 0) invert_diagonal(wm, lane);
      __syncthreads();
      invert_below(wm, wave, lane);
      write_transposed(wm, a.ttf + tbase, wave, lane);
      __syncthreads();
    }
  }
}

template <typename T, int KP, bool FULL>
__global__ __launch_bounds__(512, (kChainWaves<T, KP>)) void gdr_chain_kernel(GdrArgs a, int64_t first) {
  __shared__ __align__(16) char lds[sizeof(GdrChainLds<T, KP, false>)];
  gdr_chain<T, KP, false, FULL>(a, lds, first + blockIdx.x);
}

template <typename T, int KP>
int launch_prepare(const GdrArgs& a, bool backward, hipStream_t s) {
  // Two heads of a group to a workgroup where that still leaves four for each CU; one, for their latency,
  // where it does not (bf16, K 128, one and two: 16 chunks of 16 heads 15.9 and 19.4 us, 32 of 32 22.0
  // and 21.0, 64 of 32 36.9 and 32.0, 128 of 32 74.8 and 68.6).
  const int64_t cus = device_cu_count() > 0 ? device_cu_count() : 256;
  const int heads = a.group % 2 == 0 && a.slots * a.Hv >= 8 * cus ? 2 : 1;
  const dim3 grid((unsigned)a.slots, (unsigned)(a.Hv / heads)), b(256);
  const bool full = a.K == KP;
  if (backward && full) hipLaunchKernelGGL((gdr_prepare_kernel<T, KP, true, true>), grid, b, 0, s, a, heads);
  else if (backward) hipLaunchKernelGGL((gdr_prepare_kernel<T, KP, true, false>), grid, b, 0, s, a, heads);
  else if (full) hipLaunchKernelGGL((gdr_prepare_kernel<T, KP, false, true>), grid, b, 0, s, a, heads);
  else hipLaunchKernelGGL((gdr_prepare_kernel<T, KP, false, false>), grid, b, 0, s, a, heads);
  return check_launch("gdr_prepare_kernel");
}
template <typename T, int KP>
int launch_chain(const GdrArgs& a, hipStream_t s) {
  const int64_t grid = (a.n * a.Hv + 7) / 8 * 8 * ((a.V + 15) / 16);
  for (int64_t first = 0; first < grid; first += kGdrBlocks) {
    const dim3 g((unsigned)(grid - first < kGdrBlocks ? grid - first : kGdrBlocks)), b(512);
    if (a.V % 16 == 0 || a.V % 16 >= 4) hipLaunchKernelGGL((gdr_chain_kernel<T, KP, true>), g, b, 0, s, a, first);
    else hipLaunchKernelGGL((gdr_chain_kernel<T, KP, false>), g, b, 0, s, a, first);
    if (int rc = check_launch("gdr_chain_kernel")) return rc;
  }
  return ATK_OK;
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

// A token at a time takes 1.1 us for each where few heads run, two launches on a chunk 12 to 18 us
// whatever it holds (128 x 128, bf16, the one against the other.  1 sequence, 16 heads: 8 tokens 11.9 us
// and 13.6, 10 tokens 14.2 and 13.6, 12 tokens 16.6 and 13.7; 4 sequences: 10 tokens 14.8 and 16.9, 12
// tokens 16.9 and 17.0; 16 sequences, 32 heads: 10 tokens 44.8 and 59.4, 16 tokens 67.8 and 58.5).  Such
// calls keep the state in registers and need no workspace.  A packed row counts by its own length: those of
// its sequences are on the device.
static bool gdr_by_token(int64_t tokens) { return tokens <= 10; }

// Checks a call and lays out its workspace: the bytes it takes, or 0 with *rc set.
size_t gdr_plan(const atk_gated_delta_args* p, bool backward, GdrArgs* a, int* rc) {
  *rc = ATK_OK;
  if (!p) return *rc = fail(ATK_EINVAL, "gated delta: null arguments"), 0;
  if (!dtype_ok(p->dtype) || !dtype_ok(p->g_dtype) || !dtype_ok(p->beta_dtype))
    return *rc = fail(ATK_EINVAL, "gated delta: unknown dtype code"), 0;
  if (!gdr_gate_ok(p->g_dtype, p->dtype) || !gdr_gate_ok(p->beta_dtype, p->dtype))
    return *rc = fail(ATK_EINVAL, "gated delta: g and beta must be of the inputs' type or fp32"), 0;
  if (p->N < 0 || p->T < 0 || p->Hk <= 0 || p->Hv <= 0 || p->K <= 0 || p->V <= 0)
    return *rc = fail(ATK_EINVAL, "gated delta: bad sizes"), 0;
  if (p->Hv % p->Hk) return *rc = fail(ATK_EINVAL, "gated delta: value heads must be a multiple of key heads"), 0;
  // chunks; in doubles, since N and T may be anything yet
  const double slots = p->cu_seqlens ? (double)(p->T / kGdrC) + (double)p->N : (double)((p->T + kGdrC - 1) / kGdrC) * (double)p->N;
  if (p->K > kGdrMaxK || p->Hv > 65535 || p->N > 65535 || p->T >= ((int64_t)1 << 31) - 64 ||
      p->V > (1 << 24) || slots > 2147483647.0)
    return *rc = fail(ATK_UNSUPPORTED, "gated delta: more than %d key columns, 65535 heads or sequences, or 2^31 tokens", kGdrMaxK), 0;
  // a chunk's states are indexed in 32 bits by the backward, columns padded to its tiles
  if (backward && ((int64_t)p->V + 31) / 32 * 32 * gdr_padded_k(p->K) > 0x7fffffff)
    return *rc = fail(ATK_UNSUPPORTED, "gated delta backward: states of more than 2^31 elements"), 0;
  *a = GdrArgs{};
  a->q = p->q; a->k = p->k; a->v = p->v; a->g = p->g; a->beta = p->beta; a->o = p->out;
  a->s0 = static_cast<const float*>(p->initial_state); a->s1 = static_cast<float*>(p->final_state); a->cu = p->cu_seqlens;
  for (int i = 0; i < 3; ++i) {
    a->q_s[i] = p->q_stride[i]; a->k_s[i] = p->k_stride[i]; a->v_s[i] = p->v_stride[i];
    a->g_s[i] = p->g_stride[i]; a->b_s[i] = p->beta_stride[i];
  }
  a->n = p->N; a->T = p->T; a->slots = (int64_t)slots;
  a->Hk = p->Hk; a->Hv = p->Hv; a->group = p->Hv / p->Hk; a->K = p->K; a->V = p->V;
  a->VP = (a->V + 31) / 32 * 32;
  a->g_dtype = p->g_dtype; a->b_dtype = p->beta_dtype; a->scale = p->scale;
  if (!backward && gdr_by_token(p->T)) return 0;
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
  if (gdr_by_token(p->T)) return gdr_tokens(a, p->dtype, s);
  if (int r = gdr_prepare(a, p->dtype, false, s)) return r;
  const int dtype = p->dtype;
  return ATK_GDR_TYPED(launch_chain, a, s);
}

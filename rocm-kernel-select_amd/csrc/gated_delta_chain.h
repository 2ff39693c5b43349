// The chain that passes the state of the gated delta rule from chunk to chunk: the forward's, and the
// backward's second run of it, which shares a launch with the chain of the state's gradient.
#pragma once
#include "gated_delta.h"

namespace atk {

// Workgroup -> (value tile, head, sequence).  Workgroups are dealt to the 8 XCDs in turn; all value
// tiles of a head and sequence get the same one, since they read the same fragments through its L2.
__device__ __forceinline__ bool gdr_chain_place(const GdrArgs& a, int64_t block, int tiles, int* tile, int* h, int64_t* n) {
  const int64_t j = block / 8, unit = j / tiles * 8 + block % 8;
  *tile = (int)(j % tiles);
  *h = (int)(unit % a.Hv);
  *n = unit / a.Hv;
  return *n < a.n;
}

// Waves of a SIMD that a chain is compiled for: with four (128 registers) two workgroups share a CU,
// where more of them run than there are CUs (7 packed sequences, 16 heads of 64 x 64 fp16: 64 us against
// 70).  Wider operands would spill.
template <typename T, int KP> inline constexpr int kChainWaves = KP * kParts<T> <= 128 ? 4 : 2;

template <typename T, int KP, bool KEEP>
struct GdrChainLds {
  static constexpr int KS = KP / 32;
  f32x4 kp[4][4][64];                      // partial sums [state wave][token tile][lane]
  uint2 xl[2][3][64][2], el[2][3][64][2];  // X and E U in parts, as B is read
  f32x4 vl[4][64];                         // V
  float rl[192];                           // the chunk's decays and betas
  uint4 sl[KEEP ? 1 : KS][3][64];          // the state in parts, for the outputs
  f32x4 ul[KEEP ? 1 : 4][64];              // U, fp32
  T ol[KEEP ? 1 : 4][16][20];              // an output tile on its way to rows
};

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
// longer than they have.  bf16, 8192 tokens, 32 heads of 128 x 128: 128 steps in 236 to 253 us, 1.9 us
// each, the matrix units 22 % busy; a CU issues about 105 vector loads and stores a step, which is what
// the step waits for beside the three products.  (All four waves on both the state and the outputs,
// loads after each barrier: 943 us.)
// FULL: no tile of value columns ends in one of fewer than 4, so a lane has 4 columns of a token in one
// load or store (the last of a tile that V ends in overlap).
template <typename T, int KP, bool KEEP, bool FULL>
__device__ __forceinline__ void gdr_chain(const GdrArgs& a, char* lds, int64_t block) {
  constexpr int NP = kParts<T>, KS = KP / 32, MT = KP / 64, KW = MT > 1 ? MT / 2 : 1, OP = kOutParts<T>;
  constexpr int KF = KS * 4 * NP * 64;
  using Lds = GdrChainLds<T, KP, KEEP>;
  Lds& L = *reinterpret_cast<Lds*>(lds);
  auto& kp = L.kp;
  auto& xl = L.xl;
  auto& el = L.el;
  auto& vl = L.vl;
  auto& rl = L.rl;
  auto& sl = L.sl;
  auto& ul = L.ul;
  auto& ol = L.ol;
  const int tid = threadIdx.x, lane = tid & 63, c = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int tile, h;
  int64_t n;
  const int tiles = KEEP ? a.VP / 16 : (a.V + 15) / 16;
  if (!gdr_chain_place(a, block, tiles, &tile, &h, &n)) return;
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
      f32x4 rest, beta, spoilt;  // NaN where X is not finite, else 0
      float all;
      {
        const f32x4 v = vl[wave][lane], y0 = kp[0][wave][lane], y1 = kp[1][wave][lane], y2 = kp[2][wave][lane], y3 = kp[3][wave][lane];
        const f32x4 grown = *reinterpret_cast<const f32x4*>(&rl[16 * wave + 4 * g]);
        const f32x4 z = (y0 + y1) + (y2 + y3);
        float x[4];
        bf16x4 parts[3];
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = v[r] - grown[r] * z[r];
        __builtin_amdgcn_sched_barrier(0);  // (what follows would not fit the registers beside the partial sums)
        rest = *reinterpret_cast<const f32x4*>(&rl[64 + 16 * wave + 4 * g]);
        beta = *reinterpret_cast<const f32x4*>(&rl[128 + 16 * wave + 4 * g]);
        all = rl[63];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          spoilt[r] = x[r] * 0.f;
          x[r] = gdr_finite(x[r]);
        }
        split_parts<3, 4>(x, parts);
#pragma unroll
        for (int p = 0; p < 3; ++p) xl[wave >> 1][p][lane][wave & 1] = __builtin_bit_cast(uint2, parts[p]);
        // U is not finite where X is not, so neither is the state after the chunk
        if constexpr (!KEEP) {
          beta += spoilt;
          asm volatile("" : "+v"(beta));
        }
      }
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
        if constexpr (KEEP) e += spoilt;
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
        const f32x4 before = y;
        auto half = [&](const uint4 (&p)[OP], int s, f32x4 w, bool clean) {
          bf16x8 parts[OP];
          uint4 b[OP];
          const f32x4 lo = ul[2 * s][lane], hi = ul[2 * s + 1][lane];
          float x[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
          if (clean)
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = gdr_finite(x[i]);
          split_parts<OP, 8>(x, parts);
#pragma unroll
          for (int i = 0; i < OP; ++i) b[i] = __builtin_bit_cast(uint4, parts[i]);
          return mma_parts<OP, OP>(p, b, w);
        };
        y = half(pa[0], 0, y, false);
        if (two) z = half(pa[1], 1, z, false);
        y += z;
        // loads before the store: what waits for them would wait for a store in front of them too
        const uint4* __restrict__ now = pf;
        pf += more ? pstep : 0;
        load_p();
        __builtin_amdgcn_sched_barrier(0);
        if (__any(gdr_spoilt<4>(y))) {  // again, without what is not finite
          y = before;
          const int l = gdr_lane();
#pragma nounroll
          for (int s = 0; s <= (two ? 1 : 0); ++s) {
            uint4 p[OP];
#pragma unroll
            for (int i = 0; i < OP; ++i) p[i] = now[(s * OP + i) * 64 + l];
            y = half(p, s, y, true);
          }
          int first = kGdrC;  // of this column's tokens whose U is not finite
#pragma nounroll
          for (int i = 16 * m + 15; i >= 0; --i)
            first = gdr_spoilt<1>(&reinterpret_cast<const float*>(&ul[i >> 4][16 * ((i >> 2) & 3) + (l & 15)])[i & 3]) ? i : first;
#pragma unroll
          for (int r = 0; r < 4; ++r) y[r] = 16 * m + 4 * (l >> 4) + r < first ? y[r] : gdr_nan();
        }
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

}  // namespace atk

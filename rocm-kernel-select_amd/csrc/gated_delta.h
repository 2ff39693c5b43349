// What the kernels of the gated delta rule share: argument structs, limits, and the fragments that
// their matrix products are fed with.
//
// The products run on bf16 MFMA with fp32 accumulators, and the state, the decays and everything
// that is chained over the sequence are fp32.  So an fp32 operand enters a product as three bf16
// parts that sum to it (8 bits each, 24 in all), and a product takes the parts' products down to
// 2^-16 of the largest: 3 MFMAs where the other operand is a bf16 input (exact in one part), 6 where
// it is fp32 too.  An fp16 input is exact in two parts, an fp32 one in three.
#pragma once
#include "atk_common.h"

namespace atk {

constexpr int kGdrMaxK = 256;   // key columns: a state's rows
constexpr int kGdrC = 64;       // tokens of a chunk
// workgroups of 512 that one launch of a chain has at most: with fewer than 2^32 threads in a launch, a
// call of more heads, sequences and value tiles takes several (a multiple of the 8 XCDs each)
constexpr int64_t kGdrBlocks = (int64_t)1 << 21;

struct GdrStepArgs {
  const void* q; const void* k; const void* v; const void* g; const void* beta;
  float* state; void* o; const int* slots;
  int64_t n, n_slots, state_stride;
  int64_t q_sb, q_sh, k_sb, k_sh, v_sb, v_sh, g_sb, g_sh, b_sb, b_sh;  // strides in elements: sequence, head
  int Hv, group, K, V, g_dtype, b_dtype;
  float scale;
};

// A whole call on sequences.  Strides in elements: batch, token, head.
struct GdrArgs {
  const void* q; const void* k; const void* v; const void* g; const void* beta;
  void* o; const float* s0; float* s1; const int* cu;
  int64_t q_s[3], k_s[3], v_s[3], g_s[3], b_s[3];
  int64_t n, T;          // sequences; tokens of each (of the packed row with cu)
  int64_t slots;         // chunks, unused ones of packed sequences among them
  int Hk, Hv, group, K, V, g_dtype, b_dtype;
  float scale;
  // workspace: fragments by (key head, slot) and (value head, slot), and each chunk's decays; the chunks
  // of a sequence follow each other, so a chain's next loads are near its last
  uint4* kf; uint4* qf; uint4* ktf; uint4* tf; uint4* pf;
  void* dump;            // 256 elements that nobody reads
  float* row;            // [Hv][slot][3][64]: exp(G_i), exp(G_63 - G_i), beta_i
  // the backward's: fragments of Q^T, (1 + diag(beta) W)^-T and lower(Q K^T * D)^T; each chunk's G / ln 2
  // as two floats; the state and the errors that the forward chain had at each chunk, and the gradients of
  // the state after it and of U: [Hv][slot] matrices
  // of KP or 64 rows and VP columns in gdr_kept's order, fp32, VP = V padded to 32
  uint4* qtf; uint4* ttf; uint4* ptf;
  float2* gsum;
  float* sc; float* ec; float* dsc; float* drc;
  const void* dout; const float* ds1; float* ds0;
  void* dq; void* dk; void* dv; void* dg; void* dbeta;
  int VP;
};

// Host side, shared by the forward and the backward: fragments of all chunks.
int gdr_prepare(const GdrArgs& a, int dtype, bool backward, hipStream_t s);
int gdr_tokens(const GdrArgs& a, int dtype, hipStream_t s);  // forward, a token at a time
size_t gdr_plan(const atk_gated_delta_args* p, bool backward, GdrArgs* a, int* rc);
inline bool gdr_gate_ok(int gate, int dtype) { return gate == dtype || gate == ATK_F32; }  // what gdr_gate reads
inline int gdr_padded_k(int K) { return K <= 64 ? 64 : K <= 128 ? 128 : 256; }

// Where sequence n's tokens and chunks lie.  A packed sequence has the chunk slots from
// begin / 64 + n on: the next one's begin at or after its end, whatever the lengths, so no prefix
// sum over the lengths is needed.  Offsets are clamped to the row, so bad ones stay in bounds.
struct GdrSeq {
  int64_t batch, begin, len, slot;
};
__device__ __forceinline__ GdrSeq gdr_seq(const int* __restrict__ cu, int64_t T, int64_t n) {
  if (!cu) return {n, 0, T, n * ((T + kGdrC - 1) / kGdrC)};
  int64_t b = cu[n], e = cu[n + 1];
  b = b < 0 ? 0 : b > T ? T : b;
  e = e < b ? b : e > T ? T : e;
  return {0, b, e - b, b / kGdrC + n};
}
// The sequence that chunk slot `slot` belongs to; a slot that no chunk has gets one past its end.
__device__ __forceinline__ int64_t gdr_seq_of_slot(const int* __restrict__ cu, int64_t T, int64_t n, int64_t slot) {
  if (!cu) return (uint32_t)slot / (uint32_t)((T + kGdrC - 1) / kGdrC);  // (both below 2^31)
  int64_t lo = 0, hi = n - 1;  // the last sequence whose first slot is not after `slot`
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) / 2;
    if (gdr_seq(cu, T, mid).slot <= slot) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// A gate or strength, of T or fp32, as two halves of 16 bits (an fp32 one's low and high): no branch on
// the type around the load, which would make the loads before and after it wait for each other.
struct GdrGate {
  unsigned short lo, hi;
};
__device__ __forceinline__ GdrGate gdr_gate_load(const void* p, int dtype, int64_t i) {
  const int wide = dtype == ATK_F32;
  const unsigned short* at = static_cast<const unsigned short*>(p) + (i << wide);
  return {at[0], at[wide]};
}
template <typename T>
__device__ __forceinline__ float gdr_gate(GdrGate v, int dtype) {
  if constexpr (sizeof(T) == 2)
    if (dtype != ATK_F32) return to_f32(__builtin_bit_cast(T, v.lo));
  return __uint_as_float((unsigned)v.hi << 16 | v.lo);
}

// bf16 parts that hold an input exactly
template <typename T> inline constexpr int kParts = sizeof(T) == 4 ? 3 : 2;
template <> inline constexpr int kParts<__bf16> = 1;

// D[4 g + r][lane & 15] += sum over k < 32 of A[lane & 15][k] B[k][lane & 15], g = lane / 16; a lane
// holds elements 8 g .. 8 g + 7 of its row of A and of its column of B.
__device__ __forceinline__ f32x4 mma(const uint4& a, const uint4& b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
// The same of operands in NA and NB parts, the small products first.
template <int NA, int NB>
__device__ __forceinline__ f32x4 mma_parts(const uint4 (&a)[NA], const uint4 (&b)[NB], f32x4 c) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int p = 0; p < NA; ++p)
#pragma unroll
      for (int q = 0; q < NB; ++q)
        if (p + q == s) c = mma(a[p], b[q], c);
  return c;
}

// A product's result D has rows 4 g + r in a lane; as the next product's B it needs 8 of 32.  So the 32
// are taken in the order that gives a lane its own: element i of lane group g is row gdr_at(g, i) of two
// row tiles, and every A that meets such a B has its columns in that order too.
__device__ __forceinline__ constexpr int gdr_at(int g, int i) { return i < 4 ? 4 * g + i : 12 + 4 * g + i; }

// Where a kept matrix has element r of the accumulators of row tile 0 and value tile `tile`, from its
// start; row tile t is 512 t further.  Read, 32 columns of a row tile are one operand in whole lanes: 8
// columns of a row each.
__device__ __forceinline__ int gdr_kept(int tile, int row_tiles, int c, int g) {
  return (tile >> 1) * row_tiles * 512 + (16 * ((tile & 1) * 2 + (c >> 3)) + 4 * g) * 8 + (c & 7);
}

// v[0..N) as NP parts of N bf16 each
template <int NP, int N, typename P>
__device__ __forceinline__ void split_parts(const float* v, P (&out)[NP]) {
  typedef float f2 __attribute__((ext_vector_type(2)));
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    f2 r = {v[i], v[i + 1]};
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      const b2 h = __builtin_convertvector(r, b2);
      out[p][i] = h[0];
      out[p][i + 1] = h[1];
      if (p + 1 < NP) r -= __builtin_convertvector(h, f2);
    }
  }
}

// The same for N row tiles that meet one B: the tiles take turns, so that no product waits for the one
// before it.
template <int N, int NA, int NB>
__device__ __forceinline__ void mma_tiles(const uint4 (&a)[N][NA], const uint4 (&b)[NB], f32x4 (&c)[N]) {
#pragma unroll
  for (int s = 2; s >= 0; --s)
#pragma unroll
    for (int p = 0; p < NA; ++p)
#pragma unroll
      for (int q = 0; q < NB; ++q)
        if (p + q == s) {
#pragma unroll
          for (int n = 0; n < N; ++n) c[n] = mma(a[n][p], b[q], c[n]);
          __builtin_amdgcn_sched_barrier(0);  // (the compiler would run each tile's products in a row)
        }
}

// parts that an fp32 matrix is multiplied in where the product is only rounded to T: two of bf16 (16
// bits) are beyond what a 16-bit result shows
template <typename T> inline constexpr int kOutParts = sizeof(T) == 4 ? 3 : 2;

// A zero of a triangular factor times a NaN or an infinity is NaN, and would carry it to the tokens before
// its own.  So what such a factor is multiplied with is clamped to numbers that bf16 has (a NaN too), and
// the rows that the recurrence spoils, those from the first such one on, are made NaN afterwards.
__device__ __forceinline__ float gdr_finite(float v) {
  float most = 0x1.fep127f;
  asm("" : "+s"(most));  // (a scalar register's, both signs)
  return __builtin_amdgcn_fmed3f(v, -most, most);
}
// Whether any of N values is a NaN or an infinity.
template <int N, typename V>
__device__ __forceinline__ bool gdr_spoilt(const V& v) {
  float z[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; ++i) z[i & 1] = fmaf(v[i], 0.f, z[i & 1]);
  return z[0] + z[1] != 0.f;
}
// The lane, computed here, and not kept in a register from before a loop for a branch that is hardly
// ever taken.
__device__ __forceinline__ int gdr_lane() {
  int zero = 0;
  asm volatile("" : "+v"(zero));
  return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
}
__device__ __forceinline__ float gdr_nan() {
  int nan = 0x7fc00000;
  asm volatile("" : "+v"(nan));
  return __int_as_float(nan);
}

// exp(G_i - G_j) from G / ln 2 in two floats each: the difference of near sums is exact
__device__ __forceinline__ float gdr_decay(float2 i, float2 j) {
  return __builtin_amdgcn_exp2f((i.x - j.x) + (i.y - j.y));
}

// fragments of the lower triangle of a 64 x 64 matrix in 16 x 32 tiles (row tile m, column half s)
constexpr int kTri = 6;
__device__ __forceinline__ int tri_lower(int m, int s) { return m < 2 ? m : 2 * m - 2 + s; }
__device__ __forceinline__ int tri_upper(int m, int s) { return m < 2 ? 2 * m + s : m + 2; }

}  // namespace atk

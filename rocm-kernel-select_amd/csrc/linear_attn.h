// What the kernels of linear attention with a decay for each head share: argument structs, limits, and where
// sequences, segments and chunks lie.  Fragments and parts of products are those of the gated delta rule.
#pragma once
#include "gated_delta.h"

namespace atk {

constexpr int kLaMaxK = 256;                      // key columns: a state's rows
constexpr int64_t kLaBlocks = (int64_t)1 << 23;   // workgroups of 256 in a launch of fewer than 2^32 threads

// One chunked product over the sequences:
//   out_i = sum over j of D_ij (a_i . b_j) c_j + f_i S^T a_i
// with j up to i (or, in reverse, from i on), D_ij the decay between the two, f_i the one between i and the
// chunk's first end that S stands at, and S the sum of decayed b c^T so far.  The forward has a, b, c = q, k, v;
// the gradients: dq from dO, v, k; dk from v, dO, q in reverse; dv from k, q, dO in reverse.
struct LaRole {
  const void* a; const void* b; const void* c; const void* e;
  int64_t a_s[3], b_s[3], c_s[3], e_s[3];  // strides in elements: batch, token, head
  int a_key, b_key, c_key;                 // whether the head is the key head (e's is c's other side: the key head)
  int AD, CD;                              // columns of a and b, and of c, in all
  int a_tiles;                             // tiles of a's columns, each a sum of its own
  int reverse;
  int transposed;                          // whether S as stored has its rows over c's columns
  int guard;                               // whether rows before the first non-finite c stay clean
  const float* s_first;                    // state that the first segment starts from, or null (zeros)
  const float* s_between;                  // [slot][Hv] states at the ends (in reverse: the starts) of segments, or null
  float* s_last;                           // where the last segment's state goes, or null
  void* out;                               // T (B, T, heads of out, CD), or
  float* parts;                            // fp32 sums [head of the group * a_tiles + a tile][B T][Hk][CD]
  float* dots;                             // [tile][Hv][B T]: e_i . out_i over the tile's columns
  const float* x_last; const float* x_between; float* x_out;  // [tile][slot][Hv]: sum of S and the other direction's state
};

struct LaArgs {
  LaRole role[3];
  const void* g; int64_t g_s[3];
  const int* cu;
  int64_t n, T, B;          // sequences; tokens of each (of the packed row with cu); first axis of the tensors
  int64_t slots, seg;       // segments (unused ones of packed sequences among them), tokens of one
  int Hk, Hv, group, K, V, g_dtype, fixed;
  float scale;
};

// Where sequence n's tokens and segments lie.  A packed sequence has the segment slots from begin / seg + n
// on: the next one's begin at or after its end, so no prefix sum over the lengths is needed.  Offsets are
// clamped to the row.
struct LaSeq {
  int64_t batch, begin, len, slot;
};
__device__ __forceinline__ LaSeq la_seq(const LaArgs& a, int64_t n) {
  if (!a.cu) return {n, 0, a.T, n * (a.T > a.seg ? (a.T + a.seg - 1) / a.seg : 1)};
  int64_t b = a.cu[n], e = a.cu[n + 1];
  b = b < 0 ? 0 : b > a.T ? a.T : b;
  e = e < b ? b : e > a.T ? a.T : e;
  return {0, b, e - b, b / a.seg + n};
}
__device__ __forceinline__ int64_t la_seq_of_slot(const LaArgs& a, int64_t slot) {
  if (!a.cu) return slot / (a.T > a.seg ? (a.T + a.seg - 1) / a.seg : 1);
  int64_t lo = 0, hi = a.n - 1;  // the last sequence whose first slot is not after `slot`
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) / 2;
    if (la_seq(a, mid).slot <= slot) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}
__device__ __forceinline__ int64_t la_segments(const LaSeq& s, int64_t seg) { return s.len > seg ? (s.len + seg - 1) / seg : 1; }

// Workgroup -> (tile, value head, slot).  Workgroups are dealt to the 8 XCDs in turn; the tiles and value
// heads of a key head get the same one, since they read the same rows through its L2.
__device__ __forceinline__ bool la_place(const LaArgs& a, int64_t block, int tiles, int* tile, int* h, int64_t* slot) {
  const int per = tiles * a.group;
  const int64_t j = block / 8, unit = j / per * 8 + block % 8;
  const int in = (int)(j % per);
  *tile = in % tiles;
  *h = (int)(unit % a.Hk) * a.group + in / tiles;
  *slot = unit / a.Hk;
  return *slot < a.slots;
}
inline int64_t la_grid(const LaArgs& a, int tiles) { return (a.slots * a.Hk + 7) / 8 * 8 * tiles * a.group; }

// Launchers, each for one type: outputs of roles first .. first + roles - 1, which share AD's padding and dots;
// states of segments alone (roles 0 .. roles - 1, forward and reverse).
template <typename T> int la_launch_out(const LaArgs& a, int first, int roles, bool dots, hipStream_t s);
template <typename T> int la_launch_states(const LaArgs& a, int roles, float* const* to, float* decays, hipStream_t s);

inline int la_padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
// columns of c that a workgroup has: 128 (32 a wave) where the state's rows leave the registers for it
inline int la_wide(int rows, int cols) { return rows <= 128 && cols > 64 ? 2 : 1; }

}  // namespace atk

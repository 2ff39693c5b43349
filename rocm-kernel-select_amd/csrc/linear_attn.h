// What the kernels of linear attention with a decay for each head share: argument structs, limits, and where
// sequences, segments and chunks lie.  Fragments and parts of products are those of the gated delta rule.
#pragma once
#include "gated_delta.h"

namespace atk {

constexpr int kLaMaxK = 256;                      // key columns: a state's rows
constexpr int kLaBlocks = 1 << 21;                // workgroups of 256 in a launch: fewer than 2^32 threads, with three roles too

// One chunked product over the sequences, of which the forward and the gradients are four:
//   out_i = scale sum over j of D_ij (a_i . b_j) c_j + f_i S^T a_i
// with j up to i (or, in reverse, from i on), D_ij the decay between the two, S the sum of decayed b c^T of the
// chunks before (in reverse: after), f_i the decay between i and where S stands.
//   a, b, c        forward: q, k, v;  dv: k, q, dO in reverse;  dq: dO, v, k;  dk: v, dO, q in reverse
// In reverse b c^T is scaled where it enters S, else where S is read.
enum LaMode { kLaFwd = 0, kLaDv = 1, kLaDq = 2, kLaDk = 3 };
constexpr bool la_reverse(int mode) { return mode == kLaDv || mode == kLaDk; }
// whether a and b are of the value heads, c and out of the key heads, and S as stored has its rows over c's columns
constexpr bool la_swapped(int mode) { return mode >= kLaDq; }

struct LaRole {
  const void* a; const void* b; const void* c;
  const void* e;                           // dots: the rows that out is multiplied with (of the key heads)
  int64_t a_s[3], b_s[3], c_s[3], e_s[3];  // strides in elements: batch, token, head
  int AD, CD;                              // columns of a and b, and of c, in all
  int a_tiles;                             // tiles of a's columns, each a sum of its own
  const float* s_first;                    // state that the first segment starts from, or null (zeros)
  const float* s_between;                  // [end][Hv] states where segments of a sequence meet, or null
  float* s_last;                           // where the last segment's state goes, or null
  void* out;                               // T (B, T, heads of out, CD), or
  float* parts;                            // fp32 sums [head of the group * a_tiles + a tile][B T][Hk][CD]
  float* dots;                             // [tile][Hv][B T]: e_i . out_i over the tile's columns, but for j = i
  // [tile][slot][Hv]: inner product of S, without the last token's term, and the other direction's state
  const float* x_last; const float* x_between; float* x_out;
};

struct LaArgs {
  LaRole role[3];
  const void* g; int64_t g_s[3];
  const int* cu;
  int64_t T, B;             // tokens of a sequence (of the packed row with cu); first axis of the tensors
  int n, slots, seg;        // sequences; segments (unused ones of packed sequences among them), tokens of one
  int ends;                 // places for states where two segments meet
  int Hk, Hv, group, K, V, g_dtype, fixed;
  FastDiv by_hk, by_hv, by_seg, by_segs;  // segments of a sequence where all have as many
  float scale;
};

// Where sequence n's tokens and segments lie.  A packed sequence has the segment slots from begin / seg + n
// on: the next one's begin at or after its end, so no prefix sum over the lengths is needed.  The state where its
// segments z and z + 1 meet has the place `end` + z: that of the one token i seg (la_segment_at) in segment z.
// Offsets are clamped to the row.
struct LaSeq {
  int batch, begin, len, slot, segs, end;
};
__device__ __forceinline__ int la_segments(const LaArgs& a, int len) {
  return len > a.seg ? (int)fdiv((uint32_t)(len - 1), a.by_seg) + 1 : 1;
}
__device__ __forceinline__ LaSeq la_seq(const LaArgs& a, int n) {
  const int T = (int)a.T;
  if (!a.cu) return {n, 0, T, n * (int)a.by_segs.d, (int)a.by_segs.d, n * (int)a.by_segs.d};
  int b = a.cu[n], e = a.cu[n + 1];
  b = b < 0 ? 0 : b > T ? T : b;
  e = e < b ? b : e > T ? T : e;
  const int i = (int)fdiv((uint32_t)b, a.by_seg);
  return {0, b, e - b, i + n, la_segments(a, e - b), i + (i * a.seg < b)};
}
// The last of n sequences that `before` holds for, or the first (it holds up to one, if offsets are in order): by a
// wave, 64 at a time.
template <typename F>
__device__ __forceinline__ int la_last(int n, F before) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int step = (hi - lo + 63) / 64, at = lo + (int)(threadIdx.x & 63) * step;
    const uint64_t in = __ballot(at < hi && before(at));
    lo += (in ? 63 - __builtin_clzll(in) : 0) * step;
    hi = lo + step < hi ? lo + step : hi;
  }
  return lo;
}
__device__ __forceinline__ int la_seq_of_slot(const LaArgs& a, int slot) {
  if (!a.cu) return (int)fdiv((uint32_t)slot, a.by_segs);
  return la_last(a.n, [&](int n) { return la_seq(a, n).slot <= slot; });
}
// Where all that is asked for is sequences of more than one segment, those are found by the tokens i seg, of which each
// segment of `seg` tokens has one: fewer than slots where sequences are many and short.  The segment with that
// token, or false.
__device__ __forceinline__ bool la_segment_at(const LaArgs& a, int i, int* n, LaSeq* seq, int* z) {
  const int token = i * a.seg;
  *n = la_last(a.n, [&](int m) { return la_seq(a, m).begin <= token; });
  *seq = la_seq(a, *n);
  *z = (int)fdiv((uint32_t)(token - seq->begin), a.by_seg);
  return token >= seq->begin && token < seq->begin + seq->len;
}

// Tokens of a packed row that no sequence has, before the first and after the last, have results of zero: f(from,
// to) for those among the slot's share of the row, whichever sequence has the slot, if any.
template <typename F>
__device__ __forceinline__ void la_outside(const LaArgs& a, int slot, F f) {
  if (!a.cu) return;
  const LaSeq last = la_seq(a, a.n - 1);
  const int64_t lo = la_seq(a, 0).begin, hi = last.begin + last.len;
  const int64_t b = (int64_t)slot * a.seg, e = b + a.seg < a.T ? b + a.seg : a.T;
  if (b < lo) f(b, e < lo ? e : lo);
  if (e > hi) f(b > hi ? b : hi, e);
}

// Workgroup -> (tile, value head, slot).  Workgroups are dealt to the 8 XCDs in turn; the tiles and value
// heads of a key head get the same one, since they read the same rows through its L2.  A launch begins with
// the first workgroup of unit `unit0`, a multiple of 8.
struct LaGrid {
  FastDiv per, tiles;  // workgroups of a unit (tiles of the value heads of a key head); tiles of a head
  int unit0, slots;
};
__device__ __forceinline__ bool la_place(const LaArgs& a, const LaGrid& gr, int* tile, int* h, int* slot) {
  const uint32_t j = blockIdx.x / 8, u = fdiv(j, gr.per), unit = gr.unit0 + u * 8 + blockIdx.x % 8;
  const uint32_t in = j - u * gr.per.d, head = fdiv(in, gr.tiles), s = fdiv(unit, a.by_hk);
  *tile = (int)(in - head * gr.tiles.d);
  *h = (int)((unit - s * a.by_hk.d) * a.group + head);
  *slot = (int)s;
  return s < (uint32_t)gr.slots;
}

// Launchers, each for one type: the outputs of role 0, or all gradients (dq, dk, dv are roles 0, 1 and 2); what
// segments add to the states, forward and, with roles 2, in reverse.
template <typename T> int la_launch_out(const LaArgs& a, hipStream_t s);
template <typename T> int la_launch_grads(const LaArgs& a, bool dots, hipStream_t s);
template <typename T> int la_launch_states(const LaArgs& a, int roles, float* const* to, float* decays, hipStream_t s);

inline int la_padded(int d) { return d <= 64 ? 64 : d <= 128 ? 128 : 256; }
// 16 columns of c that each wave of a workgroup has, times: two where the state's rows leave the registers for it,
// unless that leaves more than half of the CUs without a workgroup (C entry, call after call, bf16, 128 x 128: 4 sequences of
// 37 tokens, 16 heads, 8.7 us and 7.7 with one; 8192 tokens of 32 heads 131 and 156).  A launch of three roles has three
// times as many (gradients, 512 tokens of 16 heads: 39 us with two and 44 with one).
inline int la_wide(const LaArgs& a, int rows, int cols, int roles) {
  const int64_t cus = device_cu_count() > 0 ? device_cu_count() : 256;
  return rows <= 128 && cols > 64 && (int64_t)a.slots * a.Hv * ((cols + 127) / 128) * 2 * roles > cus ? 2 : 1;
}

}  // namespace atk

// What the attention kernels share: the operands' description, the rows and keys
// of a sequence, and the hand-over between the kernels on half-precision planes
// (attention_split.hip) and those on tiles in registers (attention.hip).
#pragma once

#include <algorithm>

#include "tokens.h"

namespace nt {

// One head-grouped operand: row R is at outer (R / G) + inner (R % G); keys
// have G = 1.
template <class T> struct Rows {
  T *p;
  int64_t sB, sOuter, sInner, sHead; // batch, token, head of a group, key head
};

struct AttnShape {
  int B, Tq, Tk, Hk, G, D;
  int W;         // elements of the operands' rows, D to whole 16 bytes
  int rows;      // Tq G
  FastDivU32 by_group;
  int causal;    // 0 no, 1 the queries end with the sequence, 2 they begin at `start`
  int64_t start;
  Tokens starts, lengths; // p null: none
  int *err;
};

// Which of the two kinds of kernels computes a (sequence, key head): the packing
// kernel leaves a word for each of its tiles, not 0 where half precision cannot
// hold the tile's values.  words null: no packing took place.
struct AttnGate {
  const uint32_t *words;
  int per;    // looked at of each (sequence, key head)
  int stride; // from one to the next
};

// Whether any word is set; the same for all work-items of the workgroup.
__device__ __forceinline__ bool gate_set(const AttnGate &g, uint32_t bh) {
  uint32_t any = 0;
  for (int i = threadIdx.x; i < g.per; i += blockDim.x)
    any |= g.words[int64_t(bh) * g.stride + i];
  return __syncthreads_or(int(any)) != 0;
}

template <class T> struct AttnFwd {
  AttnShape s;
  Rows<const T> q, k, v;
  T *y;            // [B, Tq, H, D]
  T *lse;          // [B, Hk, rows], base 2; null: not wanted
  T scale2;        // scale log2 e
  int splits;      // of the keys
  T *part_acc;     // [tile, split, 16, D]
  T *part_stat;    // [tile, split, 2, 16]
  int vec;         // rows of all operands are whole, aligned 16-byte pieces
  AttnGate gate;
};

template <class T> struct AttnBwd {
  AttnShape s;
  Rows<const T> q, k, v, g, y;
  const T *lse;         // [B, Hk, rows]
  T *dq;                // [B, Tq, H, D]
  T *dk, *dv;           // [B, Tk, Hk, D]; either may be null
  T scale, scale2;
  AttnGate gate;
};

// Workgroup id -> (sequence, key head) of `heads`, item of `items` each; items
// rise in the order of dispatch, the longest first under a causal mask.
// Workgroups are dealt to the 8 XCDs round-robin.  Some heads at a time are walked
// together, a multiple of 8: every XCD then has heads of its own, whose keys its L2
// holds, and the same mixture of long items and short ones; enough of them that
// an XCD's 32 CUs have two rounds of items, so that short ones fill the gaps that
// long ones leave.  (Consecutive ids on one XCD left a third of the CUs without
// work: 8192 tokens, 4 key heads, forward 1.01 ms for 0.77; 8 heads at a time of 64
// with 8 items each nearly half.)  The last heads % 8 share the XCDs.
__device__ __forceinline__ void head_item(uint32_t id, uint32_t heads, uint32_t items,
                                          uint32_t &head, uint32_t &item) {
  const uint32_t together = items >= 64 ? 8 : (64 + items - 1) / items * 8;
  const uint32_t turn = id / (together * items), r = id - turn * together * items;
  const uint32_t left = heads - turn * together, n = left < together ? left : together;
  item = r / n;
  head = turn * together + (r - item * n);
}

// Keys of sequence b, and the position of its first query among them.
__device__ __forceinline__ void sequence(const AttnShape &s, int b, bool report, int &n,
                                         int &first) {
  n = s.Tk;
  if (s.lengths.p) {
    const int64_t v = s.lengths[b];
    if (report && (v < 0 || v > s.Tk))
      *s.err = NT_ERR_INDEX;
    n = int(v < 0 ? 0 : v > s.Tk ? s.Tk : v);
  }
  if (s.causal == 1)
    first = n - s.Tq;
  else {
    const int64_t v = s.starts.p ? s.starts[b] : s.start;
    // beyond these nothing changes
    first = int(v < -int64_t(s.Tq) ? -int64_t(s.Tq) : v > s.Tk ? s.Tk : v);
  }
}

// How many keys query i of a sequence sees.
__device__ __forceinline__ int seen(const AttnShape &s, int n, int first, int i) {
  if (!s.causal)
    return n;
  const int e = first + i + 1;
  return e < 0 ? 0 : e < n ? e : n;
}

// 16 bytes at element d of a row of W elements, a multiple of 16 bytes; zeros past
// its end.  No branches (one for each load kept the loads apart and filled the scalar
// registers with lane masks): in place of a row that is not there, callers read one
// that is, and leave out what comes of it.
template <class T>
__device__ __forceinline__ typename RowVec<T>::V piece(const T *row, int d, int W) {
  using R = RowVec<T>;
  typename R::V v = R::load(row + std::min(d, W - R::N));
#pragma unroll
  for (int j = 0; j < R::N; ++j)
    v[j] = d < W ? v[j] : T(0);
  return v;
}

// W, which the compiler does not know to be the same for every `by`: comparisons with
// it are made again for each.  (Kept through a loop, a lane mask for each piece of a row
// outgrew the scalar registers.)
template <class B> __device__ __forceinline__ int afresh(int W, B by) {
  asm("" : "+v"(W) : "v"(by));
  return W;
}

// attention_split.hip: whether its kernels take a product of this shape, and
// their launches.  The forward launch leaves a.gate for the kernels that follow
// it; `words` is its memory, which must outlive them.
bool split_takes(const AttnShape &s, bool backward);
size_t split_gate_words(const AttnShape &s, bool backward);
void run_split(AttnFwd<float> &a, uint32_t *words);
void run_split_bwd(AttnBwd<float> &a, uint32_t *words);

} // namespace nt

// Attention and its gradients in float32 on the half-precision matrix cores, for
// products large enough that arithmetic bounds them (attention.hip has the
// mathematics, and the kernels for all others).
//
// A float32 x, scaled by a power of two to below 2^15, is hi + 2^-12 lo with hi the
// nearest half and lo the nearest half of 2^12 times the rest.  Products of halves
// are exact in float32, so a . b is hi hi' + 2^-12 (lo hi' + hi lo') on
// v_mfma_f32_32x32x16_f16, which does sixteen times the work of the float32
// instructions: 5.3 times their rate with three products for one.
//
// What that loses.  A half is normal from 2^-14 on: a scaled x of at least that is off
// by 2^-22 of itself at most, 2^-24 in the root mean square (a float32 is off by 2^-24
// at most), and what is left out of a product, lo lo', is 2^-22 of it at most.  Below
// 2^-14 both grow as 1 / x, and at 2^-17 they are 2^-20 and, with a factor from 2^-14
// on, 2^-19.  (Without the 2^12, x of 2^-3 and less would lose bits.)  So a value may lie
// 2^28 below the largest that shares its power of two; groups with one that is not
// zero and lies below 2^-17, which for normally distributed numbers is one element in
// 2^30, are not computed here (see the gate below).  Probabilities and ds, which the
// kernels form, are scaled for each row (or key) and step of 32 or 64 items by the
// largest among these; of smaller ones the same holds, and those 2^31 and more below it
// keep an error of 2^-50 of the largest.
//
// The matrix cores do not round their running sums to nearest, so no long sum
// stays in them: the products of 32 or 64 rows are summed there, the small ones
// apart from the large ones, and the vector unit adds that to the running result.
//
// A packing kernel writes the operands as planes of halves in the order in which
// the other kernels' LDS and registers hold them, 32 rows to a unit:
//   row form  pieces of 32 rows by 16 d: lane l has row l % 32, 8 d's from
//             8 (l / 32), 16 bytes; an operand of sums over d
//   col form  pieces of 32 d by 16 rows: lane l has column l % 32 and rows
//             4 h .. 4 h + 3, 8 + 4 h .. 8 + 4 h + 3, h = l / 32, which are the
//             rows that a lane of a 32 by 32 result holds: probabilities go from
//             one matrix instruction into the next without leaving their lane
// A unit is a plane of hi pieces and one of lo pieces.  Keys, values and queries
// have one power of two to a tile of 64 rows (the forward pass's queries, which are not
// packed, one to a row), gradients one to a row.
//
// The gate: a tile with a value that is not finite, that is not zero and lies below
// 2^-17 once scaled, or that is 2^18 or more (products of three such and sums of them
// could pass float32's range before they are scaled back) is reported in a word, and
// the whole (sequence, key head) is then left to attention.hip's kernels, queued behind.
// So a masked key's value coarsens no other, nor does a large column.
//
// Every kernel's own rows (queries forward and for dq, keys for dk and dv) are the
// lanes of a result, l % 32, and the other operand's units stream through two
// stages of LDS, loaded there directly.  The matrix cores are what bounds them, or the
// power that they draw: 8192 tokens, 16 heads over 4 of 128, causal, take 781 us
// forward, 1330 for dq, 1342 and 862 for dk and dv, 41 and 82 for packing, 79 for
// adding parts; 3 products for one make that 1.06, 0.93, 0.92 and 0.96 PFLOP/s of the
// 1.07 that a large float16 product of the library's reaches here, at 1.8 to 2.2 GHz.
// With heads of 64 the exponentials and conversions weigh as much as the products: 4 x
// 2048 tokens, 16 heads, 126, 193 and 281 us, 0.73 to 0.82 PFLOP/s.  (lo without its
// 2^12, in one sum with hi, was 4 to 5% faster.)  Row statistics, rescaling and masks are
// then a lane's own, and sums over own rows' columns need no exchange.
#include <algorithm>
#include <cmath>

#include "attention.h"

namespace nt {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx16 __attribute__((ext_vector_type(16)));

constexpr int SA_UNIT = 32, SA_TILE = 64; // rows of a unit, of a packed tile
constexpr float SA_INF = std::numeric_limits<float>::infinity();
// Row statistics of a unit for the gradients: [lse, delta / scale, scale, limit][32].
constexpr int SA_STATS = 4 * SA_UNIT;

// Bytes of a unit's form, DB = padded width / 32.
template <int DB> constexpr int SA_CHUNK = DB * 4096;

__device__ __forceinline__ float pow2(int k) { // -126 <= k <= 127
  return __uint_as_float(uint32_t(127 + k) << 23);
}

// The power of two that takes a largest magnitude into [2^14, 2^15), as an
// exponent; 0 for 0.
__device__ __forceinline__ int up_exponent(float most) {
  if (most == 0.f)
    return 0;
  const int e = int(__float_as_uint(most) >> 23) - 127; // subnormals: -127
  return min(14 - e, 126);
}

constexpr float SA_LO = 4096.f;          // lo is so many times the rest
constexpr float SA_LEAST = 0x1p-17f;     // of a scaled value that is not zero
constexpr float SA_MOST = 0x1p18f;       // of a value
// Gradients' powers of two reach dv's and dk's sums times this, so that a probability
// times that of a small row is no subnormal number.
constexpr int SA_LIFT = 40;

// hi, two values to an instruction; lo, rounded once, as a sum of mixed types:
// 2^12 x - 2^12 hi is exact.
__device__ __forceinline__ void split8(const float (&x)[8], half8 &hi, half8 &lo) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  typedef _Float16 half2v __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const half2v h = __builtin_convertvector(float2v{x[j], x[j + 1]}, half2v);
    hi[j] = h.x, hi[j + 1] = h.y;
    lo[j] = _Float16(fmaf(float(h.x), -SA_LO, x[j] * SA_LO));
    lo[j + 1] = _Float16(fmaf(float(h.y), -SA_LO, x[j + 1] * SA_LO));
  }
}

// Magnitudes as integers in their order, zero the largest.
__device__ __forceinline__ uint32_t nonzero_bits(float x) {
  return (__float_as_uint(x) & 0x7fffffffu) - 1;
}

__device__ __forceinline__ floatx16 mma(half8 a, half8 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Row of a 32 by 32 result's element r in lane half h.
__device__ __forceinline__ int row32(int h, int r) { return 8 * (r >> 2) + 4 * h + (r & 3); }

// ---------------------------------------------------------------- packing

struct PackTensor {
  Rows<const float> x;
  char *row, *col;   // units of all (sequence, key head)s; null: not wanted
  float *scale;      // [bh, tiles]; null: one to a row, in `stats`
  int rows, tiles;
  int keys;          // rows from the sequence's length on are zeros
  uint32_t blocks;   // first workgroup of the next tensor
  int word;          // where its words begin among a (sequence, key head)'s
};

struct PackArgs {
  AttnShape s;
  PackTensor t[4];
  uint32_t *words;
  int stride;        // words of a (sequence, key head)
  int zero;          // the one among them that later kernels set; -1: none
  // the gradient's: y, the forward statistics, and what becomes of them
  Rows<const float> y;
  const float *lse;
  float *stats;
};

// A workgroup packs a tile of 64 rows, by way of LDS.  HBM bound: 4 bytes read,
// 4 written for each form.
template <int DB> __global__ __launch_bounds__(256) void attn_pack_kernel(const PackArgs a) {
  constexpr int DP = 32 * DB, PITCH = DP + 4, CH = SA_CHUNK<DB>;
  __shared__ float x[SA_TILE * PITCH];
  __shared__ float factor[SA_TILE];
  __shared__ uint32_t wave_most[4], wave_least[4];
  int which = 0;
  while (blockIdx.x >= a.t[which].blocks)
    ++which;
  const PackTensor &t = a.t[which];
  const AttnShape &s = a.s;
  const uint32_t id = blockIdx.x - (which ? a.t[which - 1].blocks : 0);
  const int bh = int(id / uint32_t(t.tiles)), tile = int(id - uint32_t(bh) * uint32_t(t.tiles));
  const int b = bh / s.Hk, hk = bh % s.Hk;
  int n, first;
  sequence(s, b, false, n, first);
  const int rows = t.keys ? min(n, t.rows) : t.rows;
  const float *base = t.x.p + b * t.x.sB + hk * t.x.sHead;
  auto address = [&](int row) {
    if (t.keys)
      return base + int64_t(row) * t.x.sOuter;
    const uint32_t i = s.by_group.div(uint32_t(row));
    return base + int64_t(i) * t.x.sOuter + int64_t(uint32_t(row) - i * uint32_t(s.G)) * t.x.sInner;
  };
  for (int i = threadIdx.x; i < SA_TILE * (DP / 4); i += 256) {
    const int r = i / (DP / 4), d = i % (DP / 4) * 4, row = tile * SA_TILE + r;
    const bool live = row < rows;
    const auto v = piece(live ? address(row) : base, d, s.W);
#pragma unroll
    for (int j = 0; j < 4; ++j)
      x[r * PITCH + d + j] = live ? v[j] : 0.f;
  }
  __syncthreads();
  // four work-items to a row: its largest magnitude (NaN above infinity) and its
  // smallest but zero
  const int r = threadIdx.x / 4, part = threadIdx.x % 4;
  uint32_t most = 0, least = ~0u;
  for (int d = part; d < DP; d += 4) {
    most = max(most, __float_as_uint(x[r * PITCH + d]) & 0x7fffffffu);
    least = min(least, nonzero_bits(x[r * PITCH + d]));
  }
  // of the row where that has a power of two of its own, and of the tile
  auto group = [&](int from, int to) {
#pragma unroll
    for (int o = from; o < to; o <<= 1) {
      most = max(most, uint32_t(__shfl_xor(int(most), o)));
      least = min(least, uint32_t(__shfl_xor(int(least), o)));
    }
  };
  group(1, 4);
  if (t.scale) {
    group(4, 64);
    if ((threadIdx.x & 63) == 0) {
      wave_most[threadIdx.x >> 6] = most;
      wave_least[threadIdx.x >> 6] = least;
    }
    __syncthreads();
    most = max(max(wave_most[0], wave_most[1]), max(wave_most[2], wave_most[3]));
    least = min(min(wave_least[0], wave_least[1]), min(wave_least[2], wave_least[3]));
  }
  // a gradient's row of zeros counts least among the rows that it is summed with
  const int up = !t.scale && most == 0 ? 126 : up_exponent(__uint_as_float(most));
  const bool bad = most >= __float_as_uint(SA_MOST) ||
                   (most != 0 && __uint_as_float(least + 1) * pow2(up) < SA_LEAST);
  if (t.scale) {
    if (threadIdx.x == 0)
      t.scale[int64_t(bh) * t.tiles + tile] = pow2(-up);
  } else { // the gradient: its rows' statistics
    const int row = tile * SA_TILE + r;
    float dot = 0.f;
    uint32_t i = 0;
    if (row < rows) {
      i = s.by_group.div(uint32_t(row));
      const float *y = a.y.p + b * a.y.sB + hk * a.y.sHead + int64_t(i) * a.y.sOuter +
                       int64_t(uint32_t(row) - i * uint32_t(s.G)) * a.y.sInner;
      for (int d = part * 4; d < s.W; d += 16) {
        const auto v = RowVec<float>::load(y + d);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          dot = fmaf(x[r * PITCH + d + j], v[j], dot);
      }
    }
    dot += __shfl_xor(dot, 1);
    dot += __shfl_xor(dot, 2);
    if (part == 0) {
      const int limit = row < rows ? seen(s, n, first, int(i)) : 0;
      float *st = a.stats + (int64_t(bh) * t.tiles * 2 + tile * 2 + r / SA_UNIT) * SA_STATS +
                  r % SA_UNIT;
      // a row that sees nothing: exp2(z - inf) = 0
      st[0] = limit > 0 ? a.lse[int64_t(bh) * t.rows + row] : SA_INF;
      st[SA_UNIT] = dot * pow2(up);
      st[2 * SA_UNIT] = pow2(min(SA_LIFT - up, 127));
      reinterpret_cast<int *>(st)[3 * SA_UNIT] = limit;
    }
  }
  if (part == 0)
    factor[r] = pow2(up);
  const int any = __syncthreads_or(int(bad)); // (also: the factors are there)
  if (threadIdx.x == 0) {
    a.words[int64_t(bh) * a.stride + t.word + tile] = uint32_t(any != 0);
    if (a.zero >= 0 && which == 0 && tile == 0)
      a.words[int64_t(bh) * a.stride + a.zero] = 0;
  }
  const int64_t unit0 = (int64_t(bh) * t.tiles + tile) * 2;
  // pieces of both units, a wave for each
  const int lane = threadIdx.x & 63, l = lane & 31, h = lane >> 5;
  for (int p = threadIdx.x >> 6; p < 4 * DB; p += 4) {
    const int unit = p / (2 * DB), f = p % (2 * DB);
    float v[8];
    half8 vh, vl;
    if (t.row) {
      const int rr = unit * SA_UNIT + l;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = x[rr * PITCH + f * 16 + 8 * h + j] * factor[rr];
      split8(v, vh, vl);
      char *to = t.row + (unit0 + unit) * CH + f * 1024 + lane * 16;
      *reinterpret_cast<half8 *>(to) = vh;
      *reinterpret_cast<half8 *>(to + CH / 2) = vl;
    }
    if (t.col) {
      const int db = f / 2, ks = f % 2;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int rr = unit * SA_UNIT + ks * 16 + (j < 4 ? 4 * h + j : 4 + 4 * h + j);
        v[j] = x[rr * PITCH + db * 32 + l] * factor[rr];
      }
      split8(v, vh, vl);
      char *to = t.col + (unit0 + unit) * CH + f * 1024 + lane * 16;
      *reinterpret_cast<half8 *>(to) = vh;
      *reinterpret_cast<half8 *>(to + CH / 2) = vl;
    }
  }
}

// ----------------------------------------------------------------- shared

__device__ __forceinline__ void load_lds(const char *from, char *to, int lane) {
  __builtin_amdgcn_global_load_lds(
      (const __attribute__((address_space(1))) void *)(from + lane * 16),
      (__attribute__((address_space(3))) void *)to, 16, 0, 0);
}

// This wave's direct loads have landed, and every wave is past the stage before.
__device__ __forceinline__ void stage_ready() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}

__device__ __forceinline__ half8 frag(const char *p, int lane) {
  return *reinterpret_cast<const half8 *>(p + lane * 16);
}

// A hi piece and the lo piece that belongs to it.
struct Pair {
  half8 h, l;
};

// Pieces are read two pairs ahead of the matrix instructions that take them, across
// the ends of sums too: the reads stay where they are written, and only other
// work moves past them.  (The compiler put each right before its use; the wait on
// LDS was a third of the waves' time.)
__device__ __forceinline__ void keep_order() {
  __builtin_amdgcn_sched_barrier(0x2 | 0x4 | 0x10); // vector, scalar, global memory
}

// How the small products are kept from the large ones'.  APART: in a sum of their own.
// In turn, where registers are short (two waves to a SIMD, heads of 65 to 128): first
// the small ones, whose sum the large ones are added to; the hi pieces wait for their
// turn in registers where those are two or four, else they are read again.
template <int DB> constexpr bool SA_APART = DB <= 2 || DB > 4;

// sum over NF pieces of (pieces . operand), pieces at at(0) ..; pre holds the first
// two pairs and gets those at next(0) and next(1).
template <int NF, bool APART, int HALF, class At, class Next>
__device__ __forceinline__ floatx16 stream_sum(At at, Next next, const half8 *hi, const half8 *lo,
                                               Pair (&pre)[2], int lane) {
  auto pair = [&](const char *p) { return Pair{frag(p, lane), frag(p + HALF, lane)}; };
  floatx16 small{};
  if constexpr (APART) {
    floatx16 large{};
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const Pair x = pre[f & 1];
      pre[f & 1] = pair(f + 2 < NF ? at(f + 2) : next(f + 2 - NF));
      keep_order();
      small = mma(x.l, hi[f], small);
      large = mma(x.h, hi[f], large);
      small = mma(x.h, lo[f], small);
      keep_order();
    }
#pragma unroll
    for (int r = 0; r < 16; ++r)
      large[r] = fmaf(small[r], 1.f / SA_LO, large[r]);
    return large;
  } else {
    constexpr bool KEEP = NF <= 4;
    half8 xh[KEEP ? NF : 2];
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const Pair x = pre[f & 1];
      if constexpr (KEEP) {
        xh[f] = x.h;
        pre[f & 1] = pair(f + 2 < NF ? at(f + 2) : next(f + 2 - NF));
      } else if (f + 2 < NF) {
        pre[f & 1] = pair(at(f + 2));
      } else {
        xh[f & 1] = frag(at(f & 1), lane);
      }
      keep_order();
      small = mma(x.l, hi[f], small);
      small = mma(x.h, lo[f], small);
      keep_order();
    }
    small *= 1.f / SA_LO;
#pragma unroll
    for (int f = 0; f < NF; ++f) {
      const half8 x = xh[KEEP ? f : f & 1];
      if constexpr (!KEEP) {
        if (f + 2 < NF)
          xh[f & 1] = frag(at(f + 2), lane);
        else
          pre[f & 1] = pair(next(f & 1));
        keep_order();
      }
      small = mma(x, hi[f], small);
    }
    keep_order();
    return small;
  }
}

// items' row form (a unit) . own rows: result[item, own]; pre and next as above.
template <int DB, class Next>
__device__ __forceinline__ floatx16 dots32(const char *unit, const half8 (&hi)[2 * DB],
                                           const half8 (&lo)[2 * DB], Pair (&pre)[2], Next next,
                                           int lane) {
  return stream_sum<2 * DB, SA_APART<DB>, SA_CHUNK<DB> / 2>(
      [&](int f) { return unit + f * 1024; }, next, hi, lo, pre, lane);
}

// The first two pairs of a form.
template <int DB> __device__ __forceinline__ void first_pairs(Pair (&pre)[2], const char *p,
                                                              int lane) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
    pre[i] = {frag(p + i * 1024, lane), frag(p + SA_CHUNK<DB> / 2 + i * 1024, lane)};
}

// The lane's 16 results of a unit as operand: two groups of 16 items.
__device__ __forceinline__ void split16(const floatx16 &x, half8 *hi, half8 *lo) {
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j)
      v[j] = x[8 * k + j];
    split8(v, hi[k], lo[k]);
  }
}

// A power of two that takes the 32 items' largest magnitude in this lane's column
// (both halves') below 2^15, and its inverse.
__device__ __forceinline__ float column_factor(const floatx16 &x, float &inverse) {
  float most = 0.f;
#pragma unroll
  for (int r = 0; r < 16; ++r)
    most = fmaxf(most, fabsf(x[r]));
  most = fmaxf(most, __shfl_xor(most, 32));
  const int e = int(__float_as_uint(most) >> 23);
  const int up = min(268 - e, 253);
  inverse = __uint_as_float(uint32_t(254 - up) << 23);
  return __uint_as_float(uint32_t(up) << 23);
}

// acc = acc + k (items' col form (a unit) . x); pre holds its first pairs and gets
// those at `after`.
template <int DB>
__device__ __forceinline__ void sums32(floatx16 (&acc)[DB], const char *unit, const half8 (&hi)[2],
                                       const half8 (&lo)[2], float k, Pair (&pre)[2],
                                       const char *after, int lane) {
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    const floatx16 t = stream_sum<2, SA_APART<DB>, SA_CHUNK<DB> / 2>(
        [&](int f) { return unit + (2 * db + f) * 1024; },
        [&](int f) { return (db + 1 < DB ? unit + (2 * db + 2) * 1024 : after) + f * 1024; }, hi,
        lo, pre, lane);
#pragma unroll
    for (int r = 0; r < 16; ++r)
      acc[db][r] = fmaf(t[r], k, acc[db][r]);
  }
}

// Stores a lane's own row of 32 DB columns, times k.
template <int DB>
__device__ __forceinline__ void store_row(float *p, const floatx16 (&acc)[DB], float k, int D,
                                          int h) {
#pragma unroll
  for (int db = 0; db < DB; ++db)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * db + 8 * q + 4 * h;
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = acc[db][4 * q + j] * k;
      if (d + 4 <= D)
        RowVec<float>::store(p + d, RowVec<float>::V{v[0], v[1], v[2], v[3]});
      else
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (d + j < D)
            p[d + j] = v[j];
    }
}

// ---------------------------------------------------------------- forward

// Eight waves, two to a SIMD, and 64 keys a step; of heads over 128 wide four waves,
// which need the registers of two, and 32 keys, as many as LDS holds twice.
template <int DB> constexpr int SF_WAVES = DB <= 4 ? 8 : 4;
template <int DB> constexpr int SF_ROWS = SF_WAVES<DB> * SA_UNIT;
template <int DB> constexpr int SF_UNITS = DB <= 4 ? 2 : 1;

struct SplitFwd {
  AttnShape s;
  Rows<const float> q;
  const char *k, *v;             // row form, col form
  const float *k_scale, *v_scale;
  int tiles;                     // of 64 keys
  float *y, *lse;
  float scale2;
  AttnGate gate;
  uint32_t *q_word;              // of each (sequence, key head), gate.stride apart
  int parts;                     // of the keys; over one: sums [part][bh, row][D] and
  float *sums, *tops;            // maxima, sums of p [part][2][bh, row]
};

template <int DB>
__global__ __launch_bounds__(64 * SF_WAVES<DB>, (DB <= 4 ? 2 : 1)) void attn_split_fwd_kernel(const SplitFwd a) {
  constexpr int CH = SA_CHUNK<DB>, UNITS = SF_UNITS<DB>, STEP = UNITS * SA_UNIT;
  __shared__ __attribute__((aligned(1024))) char lds[2][2 * UNITS * CH];
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tiles = uint32_t(s.rows + SF_ROWS<DB> - 1) / SF_ROWS<DB>;
  const uint32_t parts = uint32_t(a.parts);
  uint32_t bh, item;
  head_item(blockIdx.x, uint32_t(s.B) * uint32_t(s.Hk), tiles * parts, bh, item);
  const int tile = int(tiles - 1 - item / parts); // the most keys first
  const int part = int(item % parts);
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, threadIdx.x == 0, keys, first);
  if (gate_set(a.gate, bh))
    return;
  auto limit_of = [&](int row) {
    return seen(s, keys, first, int(s.by_group.div(uint32_t(row))));
  };
  const int row0 = tile * SF_ROWS<DB> + wave * SA_UNIT, row = row0 + n;
  const bool live = row < s.rows;
  const int limit = live ? limit_of(row) : 0;
  const int end = row0 < s.rows ? limit_of(min(row0 + SA_UNIT, s.rows) - 1) : 0; // of any row
  const int all = row0 < s.rows ? limit_of(row0) : 0;                           // of every row
  const int group_end = limit_of(min((tile + 1) * SF_ROWS<DB>, s.rows) - 1);
  const char *kp = a.k + int64_t(bh) * a.tiles * 2 * CH, *vp = a.v + int64_t(bh) * a.tiles * 2 * CH;
  auto issue = [&](char *stage, int it) {
#pragma unroll
    for (int j = 0; j < 2 * DB; ++j) {
      const int p = j % DB * SF_WAVES<DB> + wave;
      load_lds((j < DB ? kp : vp) + int64_t(it) * UNITS * CH + p * 1024,
               stage + (j < DB ? 0 : UNITS * CH) + p * 1024, lane);
    }
  };
  const int all_steps = (group_end + STEP - 1) / STEP;
  const int per = (all_steps + a.parts - 1) / a.parts;
  const int begin = min(part * per, all_steps), steps = min(begin + per, all_steps);
  if (begin < steps)
    issue(lds[begin & 1], begin);
  // own row: one power of two, and the sign of the scale
  half8 qh[2 * DB], ql[2 * DB];
  float q_scale;
  {
    const uint32_t i = s.by_group.div(uint32_t(row));
    const float *qp = a.q.p + b * a.q.sB + hk * a.q.sHead;
    if (live)
      qp += int64_t(i) * a.q.sOuter + int64_t(uint32_t(row) - i * uint32_t(s.G)) * a.q.sInner;
    float v[2 * DB][8];
    float most = 0.f;
    uint32_t least = ~0u;
#pragma unroll
    for (int f = 0; f < 2 * DB; ++f)
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const auto x = piece(qp, 16 * f + 8 * h + 4 * u, s.W);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[f][4 * u + j] = x[j];
          most = fmaxf(most, fabsf(x[j]));
          least = min(least, nonzero_bits(x[j]));
        }
      }
    most = fmaxf(most, __shfl_xor(most, 32));
    const int up = up_exponent(most < SA_INF ? most : 0.f);
    const float k = a.scale2 > 0.f ? pow2(up) : a.scale2 < 0.f ? -pow2(up) : 0.f;
    q_scale = pow2(-up);
    // (a row that is no number, or infinite, gives what it gives here too)
    if (most > 0.f && most < SA_INF &&
        (most >= SA_MOST || __uint_as_float(least + 1) * pow2(up) < SA_LEAST))
      a.q_word[int64_t(bh) * a.gate.stride] = 1;
#pragma unroll
    for (int f = 0; f < 2 * DB; ++f) {
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[f][j] *= k;
      split8(v[f], qh[f], ql[f]);
    }
  }
  const float c = fabsf(a.scale2);
  floatx16 acc[DB]{};
  float m = -SA_INF, l = 0.f;
  for (int it = begin; it < steps; ++it) {
    stage_ready();
    if (it + 1 < steps)
      issue(lds[(it + 1) & 1], it + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (it * STEP >= end)
      continue;
    const char *st = lds[it & 1];
    // positive and finite, so that it takes -inf to -inf
    const float cz = fminf(fmaxf(c * q_scale * a.k_scale[int64_t(bh) * a.tiles + it * UNITS / 2], 1.2e-38f),
                           3.4e38f);
    float v_scale = a.v_scale[int64_t(bh) * a.tiles + it * UNITS / 2];
    floatx16 z[UNITS];
    Pair pre[2];
    first_pairs<DB>(pre, st, lane);
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      z[u] = dots32<DB>(st + u * CH, qh, ql, pre,
                        [&](int f) { return st + (u + 1) * CH + f * 1024; }, lane);
    if (it * STEP + STEP > all)
#pragma unroll
      for (int u = 0; u < UNITS; ++u)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          z[u][r] = it * STEP + u * SA_UNIT + row32(h, r) < limit ? z[u][r] : -SA_INF;
    float top = -SA_INF;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        top = fmaxf(top, z[u][r]);
    top = fmaxf(top, __shfl_xor(top, 32));
    // Probabilities relative to this step's largest, so that none is too small for its
    // halves beside a larger one of another step, whose values may be far smaller.
    const float here = top * cz, base = here == -SA_INF ? 0.f : here;
    const float next = fmaxf(m, here), whole = next == -SA_INF ? 0.f : next;
    const float shrink = __builtin_amdgcn_exp2f(m - whole);
    const float weight = __builtin_amdgcn_exp2f(here - whole);
    m = next;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        // times 2^14, which the quotient by l takes out again
        z[u][r] = __builtin_amdgcn_exp2f(fmaf(z[u][r], cz, 14.f - base));
        sum += z[u][r];
      }
    l = fmaf(l, shrink, sum * weight);
    half8 ph[2 * UNITS], pl[2 * UNITS];
#pragma unroll
    for (int u = 0; u < UNITS; ++u)
      split16(z[u], ph + 2 * u, pl + 2 * u);
    v_scale *= weight;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      const floatx16 o = stream_sum<2 * UNITS, SA_APART<DB>, CH / 2>(
          [&](int f) { return st + (UNITS + f / 2) * CH + (2 * db + f % 2) * 1024; },
          [&](int f) { return st + UNITS * CH + (2 * (db + 1 < DB ? db + 1 : 0) + f) * 1024; }, ph, pl,
          pre, lane);
#pragma unroll
      for (int r = 0; r < 16; ++r)
        acc[db][r] = fmaf(o[r], v_scale, acc[db][r] * shrink);
    }
  }
  if (!live)
    return;
  l += __shfl_xor(l, 32);
  if (a.parts > 1) {
    const int64_t rows = int64_t(s.B) * s.Hk * s.rows, at = int64_t(bh) * s.rows + row;
    store_row<DB>(a.sums + (part * rows + at) * s.D, acc, 1.f, s.D, h);
    if (h == 0) {
      a.tops[2 * part * rows + at] = m;
      a.tops[(2 * part + 1) * rows + at] = l;
    }
    return;
  }
  const uint32_t i = s.by_group.div(uint32_t(row));
  const int64_t head = int64_t(hk) * s.G + (uint32_t(row) - i * uint32_t(s.G));
  store_row<DB>(a.y + ((int64_t(b) * s.Tq + i) * s.Hk * s.G + head) * s.D, acc,
                limit > 0 ? 1.f / l : 0.f, s.D, h);
  if (a.lse && h == 0)
    a.lse[int64_t(bh) * s.rows + row] = m == -SA_INF ? 0.f : m + (log2f(l) - 14.f);
}

// Rows whose keys were split into at most 64 parts: a wave for each row.
__global__ __launch_bounds__(256) void attn_split_join_kernel(const SplitFwd a) {
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63;
  // a workgroup's rows belong to one (sequence, key head)
  const uint32_t groups = uint32_t(s.rows + 3) / 4, bh = blockIdx.x / groups;
  if (gate_set(a.gate, bh))
    return;
  const int row = int(blockIdx.x - bh * groups) * 4 + int(threadIdx.x >> 6);
  if (row >= s.rows)
    return;
  const int64_t rows = int64_t(s.B) * s.Hk * s.rows, at = int64_t(bh) * s.rows + row;
  float m = -SA_INF, l = 0.f;
  if (lane < a.parts) {
    m = a.tops[2 * lane * rows + at];
    l = a.tops[(2 * lane + 1) * rows + at];
  }
  float top = m;
#pragma unroll
  for (int o = 32; o; o >>= 1)
    top = fmaxf(top, __shfl_xor(top, o));
  const float weight = __builtin_amdgcn_exp2f(m - (top == -SA_INF ? 0.f : top));
  float total = l * weight;
#pragma unroll
  for (int o = 32; o; o >>= 1)
    total += __shfl_xor(total, o);
  int keys, first;
  sequence(s, int(bh) / s.Hk, false, keys, first);
  const uint32_t i = s.by_group.div(uint32_t(row));
  const float k = seen(s, keys, first, int(i)) > 0 ? 1.f / total : 0.f;
  const int64_t head = int64_t(bh % uint32_t(s.Hk)) * s.G + (uint32_t(row) - i * uint32_t(s.G));
  float *y = a.y + ((int64_t(bh / uint32_t(s.Hk)) * s.Tq + i) * s.Hk * s.G + head) * s.D;
  // a row of up to 256 at once
  float v[4] = {};
#pragma unroll 8
  for (int p = 0; p < a.parts; ++p) {
    const float w = __shfl(weight, p);
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (64 * c < s.D)
        v[c] = fmaf(a.sums[(p * rows + at) * s.D + min(64 * c + lane, s.D - 1)], w, v[c]);
  }
#pragma unroll
  for (int c = 0; c < 4; ++c)
    if (64 * c + lane < s.D)
      y[64 * c + lane] = v[c] * k;
  if (a.lse && lane == 0)
    a.lse[at] = top == -SA_INF ? 0.f : top + (log2f(total) - 14.f);
}

// --------------------------------------------------------------- backward

// Two waves to a SIMD: two workgroups of four on a CU, or where the stages fill more
// than half of its LDS one of eight; of heads over 128 wide one wave to a SIMD.
template <int DB> constexpr int SB_WAVES = DB <= 2 || DB > 4 ? 4 : 8;
template <int DB> constexpr int SB_ROWS = SB_WAVES<DB> * SA_UNIT;
// Stages of so many bytes: two, or as LDS (160 KB) has it one, loaded when all waves
// are done with it.
constexpr int SB_STAGES(int bytes) { return 2 * bytes <= 150 * 1024 ? 2 : 1; }

struct SplitBwd {
  AttnShape s;
  const char *q_row, *q_col, *g_row, *g_col, *k_row, *k_col, *v_row;
  const float *q_scale, *k_scale, *v_scale; // [bh, tiles]
  const float *stats;                       // [bh, units][SA_STATS]
  int q_tiles, k_tiles;                     // of 64 rows
  float *dq, *dk, *dv;                      // [parts] of the result's size each
  int q_parts, parts;                       // of dq's keys, of dk's and dv's rows
  float scale, scale2;
  AttnGate gate;
};

template <int DB>
__device__ __forceinline__ void load_own(const char *unit, half8 (&hi)[2 * DB],
                                         half8 (&lo)[2 * DB], int lane) {
#pragma unroll
  for (int f = 0; f < 2 * DB; ++f) {
    hi[f] = frag(unit + f * 1024, lane);
    lo[f] = frag(unit + SA_CHUNK<DB> / 2 + f * 1024, lane);
  }
}

template <int DB>
__global__ __launch_bounds__(64 * SB_WAVES<DB>, (DB <= 4 ? 2 : 1)) void attn_split_dq_kernel(
    const SplitBwd a) {
  constexpr int CH = SA_CHUNK<DB>, WAVES = SB_WAVES<DB>;
  constexpr int STAGES = SB_STAGES(3 * CH);
  __shared__ __attribute__((aligned(1024))) char lds[STAGES][3 * CH];
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tiles = uint32_t(s.rows + SB_ROWS<DB> - 1) / SB_ROWS<DB>;
  const uint32_t parts = uint32_t(a.q_parts);
  uint32_t bh, item;
  head_item(blockIdx.x, uint32_t(s.B) * uint32_t(s.Hk), tiles * parts, bh, item);
  const int tile = int(tiles - 1 - item / parts), part = int(item % parts);
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, false, keys, first);
  if (gate_set(a.gate, bh))
    return;
  auto limit_of = [&](int row) {
    return seen(s, keys, first, int(s.by_group.div(uint32_t(row))));
  };
  const int row0 = tile * SB_ROWS<DB> + wave * SA_UNIT, row = row0 + n;
  const bool on = row0 < s.rows; // of the wave
  const int end = on ? limit_of(min(row0 + SA_UNIT, s.rows) - 1) : 0;
  const int all = on ? limit_of(row0) : 0;
  const int group_end = limit_of(min((tile + 1) * SB_ROWS<DB>, s.rows) - 1);
  const int64_t kv = int64_t(bh) * a.k_tiles * 2 * CH;
  auto issue = [&](char *stage, int it) {
#pragma unroll
    for (int j = 0; j < 12 * DB; j += WAVES) {
      const int p = j + wave, form = (4 * DB % WAVES ? p : j) / (4 * DB);
      if (p < 12 * DB)
        load_lds((form == 0 ? a.k_row : form == 1 ? a.v_row : a.k_col) + kv + int64_t(it) * CH +
                     (p - form * 4 * DB) * 1024,
                 stage + p * 1024, lane);
    }
  };
  const int all_steps = (group_end + SA_UNIT - 1) / SA_UNIT;
  const int per = (all_steps + a.q_parts - 1) / a.q_parts;
  const int begin = min(part * per, all_steps), steps = min(begin + per, all_steps);
  if (STAGES == 2 && begin < steps)
    issue(lds[begin & (STAGES - 1)], begin);
  half8 qh[2 * DB], ql[2 * DB], gh[2 * DB], gl[2 * DB];
  const int64_t unit = int64_t(bh) * a.q_tiles * 2 + (on ? row0 / SA_UNIT : 0);
  load_own<DB>(a.q_row + unit * CH, qh, ql, lane);
  load_own<DB>(a.g_row + unit * CH, gh, gl, lane);
  const float *st = a.stats + unit * SA_STATS + n;
  const float lse = st[0], delta = st[SA_UNIT], g_scale = st[2 * SA_UNIT];
  const int limit = reinterpret_cast<const int *>(st)[3 * SA_UNIT];
  const float c = a.scale2 * a.q_scale[unit / 2];
  floatx16 acc[DB]{};
  for (int it = begin; it < steps; ++it) {
    if constexpr (STAGES == 1) {
      __syncthreads();
      issue(lds[0], it);
    }
    stage_ready();
    if (STAGES == 2 && it + 1 < steps)
      issue(lds[(it + 1) & (STAGES - 1)], it + 1);
    __builtin_amdgcn_sched_barrier(0);
    if (it * SA_UNIT >= end)
      continue;
    const char *stage = lds[it & (STAGES - 1)];
    const float k_scale = a.k_scale[int64_t(bh) * a.k_tiles + it / 2];
    const float v_scale = a.v_scale[int64_t(bh) * a.k_tiles + it / 2];
    Pair pre[2];
    first_pairs<DB>(pre, stage, lane);
    const floatx16 z = dots32<DB>(stage, qh, ql, pre,
                                  [&](int f) { return stage + CH + f * 1024; }, lane);
    floatx16 ds = dots32<DB>(stage + CH, gh, gl, pre,
                             [&](int f) { return stage + 2 * CH + f * 1024; }, lane);
    const float cz = c * k_scale;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const float p = __builtin_amdgcn_exp2f(fmaf(z[r], cz, -lse));
      ds[r] = p * fmaf(ds[r], v_scale, -delta);
    }
    if (it * SA_UNIT + SA_UNIT > all)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        ds[r] = it * SA_UNIT + row32(h, r) < limit ? ds[r] : 0.f;
    float inverse;
    const float k = column_factor(ds, inverse);
    ds *= k;
    half8 hi[2], lo[2];
    split16(ds, hi, lo);
    sums32<DB>(acc, stage + 2 * CH, hi, lo, inverse * k_scale, pre, stage, lane);
  }
  if (row >= s.rows)
    return;
  const uint32_t i = s.by_group.div(uint32_t(row));
  const int64_t head = int64_t(hk) * s.G + (uint32_t(row) - i * uint32_t(s.G));
  const int64_t size = int64_t(s.B) * s.Hk * s.rows * s.D;
  store_row<DB>(a.dq + part * size + ((int64_t(b) * s.Tq + i) * s.Hk * s.G + head) * s.D, acc,
                a.scale * (g_scale * pow2(-SA_LIFT)), s.D, h);
}

// DK, DV: which of the two.  Both in one kernel share the probabilities; of heads
// over 64 wide both sums and both own operands do not fit the registers of two
// waves to a SIMD, and one wave leaves the matrix cores idle while it forms
// probabilities: 8192 tokens, 16 heads over 4 of 128, 2.53 ms in one kernel where two,
// which form them twice, took 2.07 (2.20 with lo times 2^12).
template <int DB, bool DK, bool DV>
__global__ __launch_bounds__(64 * SB_WAVES<DB>, (DB <= 4 ? 2 : 1)) void attn_split_dkv_kernel(
    const SplitBwd a) {
  constexpr int CH = SA_CHUNK<DB>, STAT = SA_STATS * 4, WAVES = SB_WAVES<DB>;
  // a stage: q's rows; g's (DK); g's columns (DV); q's columns (DK)
  constexpr int FORMS = 1 + 2 * DK + DV, G_ROW = CH, G_COL = DK ? 2 * CH : CH,
                Q_COL = (2 + DV) * CH;
  constexpr int STAGES = SB_STAGES(FORMS * CH + STAT);
  __shared__ __attribute__((aligned(1024))) char lds[STAGES][FORMS * CH + STAT];
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, n = lane & 31, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t tiles = uint32_t(s.Tk + SB_ROWS<DB> - 1) / SB_ROWS<DB>;
  uint32_t bh, u;
  head_item(blockIdx.x, uint32_t(s.B) * uint32_t(s.Hk), tiles * uint32_t(a.parts), bh, u);
  const int tile = int(u / uint32_t(a.parts)), part = int(u % uint32_t(a.parts));
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, false, keys, first);
  if (gate_set(a.gate, bh))
    return;
  auto limit_of = [&](int row) {
    return seen(s, keys, first, int(s.by_group.div(uint32_t(row))));
  };
  const int key0 = tile * SB_ROWS<DB>, own0 = key0 + wave * SA_UNIT, key = own0 + n;
  // units from the first query that sees any of these keys on, this part of them
  const int units = (s.rows + SA_UNIT - 1) / SA_UNIT;
  int from = 0;
  if (key0 >= keys)
    from = units;
  else if (s.causal && key0 > first)
    from = int(min(int64_t(key0 - first) * s.G / SA_UNIT, int64_t(units)));
  const int per = (units - from + a.parts - 1) / a.parts;
  const int u0 = min(from + part * per, units), u1 = min(u0 + per, units);
  const int64_t base = int64_t(bh) * a.q_tiles * 2;
  auto issue = [&](char *stage, int it) {
    const int64_t at = (base + it) * CH;
#pragma unroll
    for (int j = 0; j < FORMS * 4 * DB; j += WAVES) {
      const int p = j + wave, to = (4 * DB % WAVES ? p : j) / (4 * DB) * CH;
      const char *x = to == 0             ? a.q_row
                      : DK && to == G_ROW ? a.g_row
                      : DV && to == G_COL ? a.g_col
                                          : a.q_col;
      if (p < FORMS * 4 * DB)
        load_lds(x + at + p * 1024 - to, stage + p * 1024, lane);
    }
    if (wave < 2) // the rows' statistics, 4 bytes a lane
      __builtin_amdgcn_global_load_lds(
          (const __attribute__((address_space(1))) void *)(a.stats + (base + it) * SA_STATS +
                                                           wave * 64 + lane),
          (__attribute__((address_space(3))) void *)(stage + FORMS * CH + wave * 256), 4, 0, 0);
  };
  if (STAGES == 2 && u0 < u1)
    issue(lds[0], u0);
  half8 kh[2 * DB], kl[2 * DB], vh[2 * DB], vl[2 * DB];
  const bool on = own0 < keys;
  const int64_t unit = int64_t(bh) * a.k_tiles * 2 + (on ? own0 / SA_UNIT : 0);
  load_own<DB>(a.k_row + unit * CH, kh, kl, lane);
  if constexpr (DK)
    load_own<DB>(a.v_row + unit * CH, vh, vl, lane);
  const float v_scale = a.v_scale[unit / 2], c = a.scale2 * a.k_scale[unit / 2];
  floatx16 dk[DB]{}, dv[DB]{};
  for (int it = u0; it < u1; ++it) {
    const int buf = (it - u0) & (STAGES - 1);
    if constexpr (STAGES == 1) {
      __syncthreads();
      issue(lds[0], it);
    }
    stage_ready();
    if (STAGES == 2 && it + 1 < u1)
      issue(lds[buf ^ (STAGES - 1)], it + 1);
    __builtin_amdgcn_sched_barrier(0);
    const int r0 = it * SA_UNIT;
    if (!on || limit_of(min(r0 + SA_UNIT, s.rows) - 1) <= own0)
      continue;
    const char *stage = lds[buf];
    const float *st = reinterpret_cast<const float *>(stage + FORMS * CH);
    const float q_scale = a.q_scale[int64_t(bh) * a.q_tiles + it / 2], cz = c * q_scale;
    Pair pre[2];
    first_pairs<DB>(pre, stage, lane);
    floatx16 w = dots32<DB>(stage, kh, kl, pre,
                            [&](int f) { return stage + CH + f * 1024; }, lane);
    floatx16 ds{};
    if constexpr (DK)
      ds = dots32<DB>(stage + G_ROW, vh, vl, pre,
                      [&](int f) { return stage + 2 * CH + f * 1024; }, lane);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const float4 lse = *reinterpret_cast<const float4 *>(st + 8 * q + 4 * h);
      const float4 delta = *reinterpret_cast<const float4 *>(st + SA_UNIT + 8 * q + 4 * h);
      const float4 g = *reinterpret_cast<const float4 *>(st + 2 * SA_UNIT + 8 * q + 4 * h);
      const float ls[4] = {lse.x, lse.y, lse.z, lse.w};
      const float de[4] = {delta.x, delta.y, delta.z, delta.w};
      const float gs[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * q + j;
        // p times the row's scale (and 2^SA_LIFT): what multiplies its packed gradient
        w[r] = __builtin_amdgcn_exp2f(fmaf(w[r], cz, -ls[j])) * gs[j];
        if constexpr (DK)
          ds[r] = w[r] * fmaf(ds[r], v_scale, -de[j]);
      }
    }
    if (limit_of(r0) < own0 + SA_UNIT)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int4 limit =
            *reinterpret_cast<const int4 *>(st + 3 * SA_UNIT + 8 * q + 4 * h);
        const int li[4] = {limit.x, limit.y, limit.z, limit.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          w[4 * q + j] = key < li[j] ? w[4 * q + j] : 0.f;
          if constexpr (DK)
            ds[4 * q + j] = key < li[j] ? ds[4 * q + j] : 0.f;
        }
      }
    half8 hi[2], lo[2];
    float inverse;
    if constexpr (DV) {
      const float k = column_factor(w, inverse);
      w *= k;
      split16(w, hi, lo);
      sums32<DB>(dv, stage + G_COL, hi, lo, inverse, pre, DK ? stage + Q_COL : stage, lane);
    }
    if constexpr (DK) {
      const float k = column_factor(ds, inverse);
      ds *= k;
      split16(ds, hi, lo);
      sums32<DB>(dk, stage + Q_COL, hi, lo, inverse * q_scale, pre, stage, lane);
    }
  }
  if (key >= s.Tk)
    return;
  const int64_t size = int64_t(s.B) * s.Tk * s.Hk * s.D;
  const int64_t at = part * size + ((int64_t(b) * s.Tk + key) * s.Hk + hk) * s.D;
  if (DK && a.dk)
    store_row<DB>(a.dk + at, dk, a.scale * pow2(-SA_LIFT), s.D, h);
  if (DV && a.dv)
    store_row<DB>(a.dv + at, dv, pow2(-SA_LIFT), s.D, h);
}

// The parts of a gradient [B, T, Hk G, D] added up in order; what the gate left to
// other kernels is not written.
__global__ __launch_bounds__(256) void attn_split_parts_kernel(const float *parts, float *out,
                                                               int count, int B, int T, int Hk,
                                                               int GD, AttnGate gate) {
  const uint32_t groups = uint32_t((int64_t(T) * GD + 255) / 256), bh = blockIdx.x / groups;
  if (gate_set(gate, bh))
    return;
  const int64_t i = int64_t(blockIdx.x - bh * groups) * 256 + threadIdx.x;
  const int64_t t = i / GD;
  if (t >= T)
    return;
  const int64_t b = bh / uint32_t(Hk), hk = bh % uint32_t(Hk);
  const int64_t at = ((b * T + t) * Hk + hk) * GD + (i - t * GD);
  const int64_t size = int64_t(B) * T * Hk * GD;
  float x = 0.f;
#pragma unroll 8
  for (int p = 0; p < count; ++p)
    x += parts[p * size + at];
  out[at] = x;
}

// ------------------------------------------------------------------- host

namespace {

int tiles_of(int rows) { return (rows + SA_TILE - 1) / SA_TILE; }

// Into how many parts `groups` workgroups' `steps` steps are split: one where there
// are two for each CU, else as many as make that, of at least four steps.
int parts_of(int64_t groups, int64_t steps) {
  const int64_t want = 2 * int64_t(device_cu_count()) / groups;
  return int(std::max<int64_t>(1, std::min<int64_t>({want, steps / 4, 32})));
}

void add_parts(const float *parts, float *out, int count, const AttnShape &s, int T, int G,
               const AttnGate &gate) {
  const int64_t groups = (int64_t(T) * G * s.D + 255) / 256;
  attn_split_parts_kernel<<<dim3(uint32_t(groups * s.B * s.Hk)), 256, 0, stream()>>>(
      parts, out, count, s.B, T, s.Hk, G * s.D, gate);
  NT_LAUNCH_CHECK();
}

template <class F> void dispatch_blocks(int D, F &&f) {
  switch ((D + 31) / 32) {
  case 1:
    return f.template operator()<1>();
  case 2:
    return f.template operator()<2>();
  case 3:
    return f.template operator()<3>();
  case 4:
    return f.template operator()<4>();
  case 5:
    return f.template operator()<5>();
  case 6:
    return f.template operator()<6>();
  default:
    return f.template operator()<8>();
  }
}

} // namespace

// From the size on at which packing, another launch or two and half-empty
// tiles cost less than the matrix cores save.  Both sides in us, B, Tq, Tk, H, Hk, D,
// this kind second.  Forward: 8 256 256 8 8 64 24 and 29, 1 1024 1024 4 4 64 30 and
// 31, 4 2048 2048 16 16 64 about 470 and 165; of few rows 4 16 4096 32 8 128 85 and
// 110.  Backward: 1 256 256 16 16 64 33 and 48, 16 128 128 8 8 64 48 and 46, 1 512 512
// 8 8 64 52 and 52, 1 1024 1024 4 4 64 89 and 53, 8 1 8192 64 2 128 870 and 237; of
// long axes with little beside them 1 64 2000 8 8 64 88 and 38.
bool split_takes(const AttnShape &s, bool backward) {
  const double work = double(s.B) * s.Hk * s.rows * s.Tk * s.D;
  if (backward && std::max(s.rows, s.Tk) >= 640 && work >= double(1 << 25))
    return true;
  return backward ? work >= double(1 << 27) : s.rows >= 128 && work >= 3.0 * double(1 << 27);
}

size_t split_gate_words(const AttnShape &s, bool backward) {
  const size_t k = size_t(tiles_of(s.Tk)), q = size_t(tiles_of(s.rows));
  return size_t(s.B) * size_t(s.Hk) * (2 * k + (backward ? 2 * q : 1));
}

void run_split(AttnFwd<float> &a, uint32_t *words) {
  const AttnShape &s = a.s;
  const uint32_t bhs = uint32_t(s.B) * uint32_t(s.Hk);
  const int tiles = tiles_of(s.Tk);
  a.gate = {words, 2 * tiles + 1, 2 * tiles + 1}; // the keys', the values', the queries'
  dispatch_blocks(s.D, [&]<int DB>() {
    const size_t form = size_t(bhs) * size_t(tiles) * 2 * SA_CHUNK<DB>;
    DeviceScratch planes(2 * form + 2 * size_t(bhs) * size_t(tiles) * sizeof(float));
    char *k = planes.get<char>(), *v = k + form;
    float *k_scale = reinterpret_cast<float *>(v + form), *v_scale = k_scale + bhs * size_t(tiles);
    PackArgs p{};
    p.s = s;
    p.words = words;
    p.stride = a.gate.stride;
    p.zero = 2 * tiles;
    p.t[0] = {a.k, k, nullptr, k_scale, s.Tk, tiles, 1, bhs * uint32_t(tiles), 0};
    p.t[1] = {a.v, nullptr, v, v_scale, s.Tk, tiles, 1, 2 * bhs * uint32_t(tiles), tiles};
    attn_pack_kernel<DB><<<dim3(p.t[1].blocks), 256, 0, stream()>>>(p);
    NT_LAUNCH_CHECK();
    SplitFwd f{};
    f.s = s;
    f.q = a.q;
    f.k = k, f.v = v;
    f.k_scale = k_scale, f.v_scale = v_scale;
    f.tiles = tiles;
    f.y = a.y, f.lse = a.lse;
    f.scale2 = a.scale2;
    f.gate = {words, 2 * tiles, a.gate.stride}; // the queries' are set meanwhile
    f.q_word = words + 2 * tiles;
    const uint32_t groups = bhs * uint32_t((s.rows + SF_ROWS<DB> - 1) / SF_ROWS<DB>);
    f.parts = parts_of(groups, tiles * 2 / SF_UNITS<DB>);
    const size_t rows = size_t(bhs) * size_t(s.rows), kept = f.parts > 1 ? size_t(f.parts) : 0;
    DeviceScratch sums(kept * rows * size_t(s.D + 2) * sizeof(float));
    f.sums = sums.get<float>();
    f.tops = f.sums + kept * rows * size_t(s.D);
    attn_split_fwd_kernel<DB>
        <<<dim3(groups * uint32_t(f.parts)), 64 * SF_WAVES<DB>, 0, stream()>>>(f);
    NT_LAUNCH_CHECK();
    if (f.parts > 1) {
      attn_split_join_kernel<<<dim3(bhs * uint32_t((s.rows + 3) / 4)), 256, 0, stream()>>>(f);
      NT_LAUNCH_CHECK();
    }
  });
}

void run_split_bwd(AttnBwd<float> &a, uint32_t *words) {
  const AttnShape &s = a.s;
  const uint32_t bhs = uint32_t(s.B) * uint32_t(s.Hk);
  const int kt = tiles_of(s.Tk), qt = tiles_of(s.rows);
  a.gate = {words, 2 * kt + 2 * qt, 2 * kt + 2 * qt};
  dispatch_blocks(s.D, [&]<int DB>() {
    const size_t kform = size_t(bhs) * size_t(kt) * 2 * SA_CHUNK<DB>;
    const size_t qform = size_t(bhs) * size_t(qt) * 2 * SA_CHUNK<DB>;
    const size_t rows = size_t(bhs) * size_t(qt) * 2 * SA_STATS;
    DeviceScratch planes(3 * kform + 4 * qform);
    DeviceScratch scales((size_t(bhs) * size_t(2 * kt + qt) + rows) * sizeof(float));
    SplitBwd f{};
    f.s = s;
    char *at = planes.get<char>();
    auto take = [&](size_t n) { return (at += n) - n; };
    char *q_row = take(qform), *q_col = take(qform), *g_row = take(qform), *g_col = take(qform);
    char *k_row = take(kform), *k_col = take(kform), *v_row = take(kform);
    float *stats = scales.get<float>(), *k_scale = stats + rows;
    float *v_scale = k_scale + size_t(bhs) * size_t(kt), *q_scale = v_scale + size_t(bhs) * size_t(kt);
    PackArgs p{};
    p.s = s;
    p.words = words;
    p.stride = a.gate.stride;
    p.zero = -1;
    p.y = a.y;
    p.lse = a.lse;
    p.stats = stats;
    const uint32_t kb = bhs * uint32_t(kt), qb = bhs * uint32_t(qt);
    p.t[0] = {a.k, k_row, k_col, k_scale, s.Tk, kt, 1, kb, 0};
    p.t[1] = {a.v, v_row, nullptr, v_scale, s.Tk, kt, 1, 2 * kb, kt};
    p.t[2] = {a.q, q_row, q_col, q_scale, s.rows, qt, 0, 2 * kb + qb, 2 * kt};
    p.t[3] = {a.g, g_row, g_col, nullptr, s.rows, qt, 0, 2 * kb + 2 * qb, 2 * kt + qt};
    attn_pack_kernel<DB><<<dim3(p.t[3].blocks), 256, 0, stream()>>>(p);
    NT_LAUNCH_CHECK();
    f.q_row = q_row, f.q_col = q_col, f.g_row = g_row, f.g_col = g_col;
    f.k_row = k_row, f.k_col = k_col, f.v_row = v_row;
    f.q_scale = q_scale, f.k_scale = k_scale, f.v_scale = v_scale;
    f.stats = stats;
    f.q_tiles = qt, f.k_tiles = kt;
    f.scale = a.scale, f.scale2 = a.scale2;
    f.gate = a.gate;
    if (a.dq) {
      const uint32_t groups = bhs * uint32_t((s.rows + SB_ROWS<DB> - 1) / SB_ROWS<DB>);
      f.q_parts = parts_of(groups, 2 * kt);
      const size_t size = size_t(bhs) * size_t(s.rows) * size_t(s.D);
      DeviceScratch sums(f.q_parts > 1 ? size * size_t(f.q_parts) * sizeof(float) : 0);
      f.dq = f.q_parts > 1 ? sums.get<float>() : a.dq;
      attn_split_dq_kernel<DB>
          <<<dim3(groups * uint32_t(f.q_parts)), 64 * SB_WAVES<DB>, 0, stream()>>>(f);
      NT_LAUNCH_CHECK();
      if (f.q_parts > 1)
        add_parts(f.dq, a.dq, f.q_parts, s, s.Tq, s.G, a.gate);
    }
    if (a.dk || a.dv) {
      // Few tiles of keys under a causal mask, each of another length, even out
      // with shorter parts.
      const uint32_t groups = bhs * uint32_t((s.Tk + SB_ROWS<DB> - 1) / SB_ROWS<DB>);
      f.parts = parts_of(s.causal ? (groups + 1) / 2 : groups, 2 * qt);
      const size_t size = size_t(s.B) * size_t(s.Tk) * size_t(s.Hk) * size_t(s.D);
      DeviceScratch sums(f.parts > 1 ? 2 * size * size_t(f.parts) * sizeof(float) : 0);
      f.dk = a.dk && f.parts > 1 ? sums.get<float>() : a.dk;
      f.dv = a.dv && f.parts > 1 ? sums.get<float>() + size * size_t(f.parts) : a.dv;
      const dim3 grid(groups * uint32_t(f.parts));
      if constexpr (DB <= 2) {
        attn_split_dkv_kernel<DB, true, true><<<grid, 64 * SB_WAVES<DB>, 0, stream()>>>(f);
        NT_LAUNCH_CHECK();
      } else {
        if (a.dv) {
          attn_split_dkv_kernel<DB, false, true><<<grid, 64 * SB_WAVES<DB>, 0, stream()>>>(f);
          NT_LAUNCH_CHECK();
        }
        if (a.dk) {
          attn_split_dkv_kernel<DB, true, false><<<grid, 64 * SB_WAVES<DB>, 0, stream()>>>(f);
          NT_LAUNCH_CHECK();
        }
      }
      if (f.parts > 1) {
        if (a.dk)
          add_parts(f.dk, a.dk, f.parts, s, s.Tk, 1, a.gate);
        if (a.dv)
          add_parts(f.dv, a.dv, f.parts, s, s.Tk, 1, a.gate);
      }
    }
  });
}

} // namespace nt

// Attention, its gradients, and attention over a cache of keys and values.
//
//   z = scale q . k over the keys that a query sees,  p = softmax z,  y = sum p v
//   dv = sum p g,   ds = p (g . v - delta),  delta = g . y
//   dq = scale sum ds k,   dk = scale sum ds q
//
// q, y and g are [B, Tq, H, D], k and v [B, Tk, Hk, D]; head h reads key head
// h / (H / Hk).  The H / Hk query heads of a key head are rows beside one
// another here: row R of a (sequence, key head) is query R / G of its head
// R % G, G = H / Hk, so that one read of a key serves all of them.  The
// forward pass keeps z's running maximum and sum (base 2) and never stores p;
// the backward pass forms p again from the rows' maximum plus log sum.
//
// The kernels of this file work on tiles of 16 rows by 16 keys, in registers,
// on the 16x16x4 matrix instructions of float32 and float64.  A lane l has
// n = l % 16 and h = l / 16.  With
//
//   dots   S[item, own] = sum over d of X[item, d] own[own, d]
//   sums   acc[own, d] += sum over items of a[own, item] X[item, d]
//
// the same registers serve as dots' result and as sums' operand: dots leaves a
// lane the own row n and four items, which is what sums' instruction r (its
// k index runs over h) takes of it.  So probabilities never leave their lane.
// Forward: own = queries, items = keys; dots with k, sums with v.  dq: dots
// with k and with v, sums with k.  dk and dv: own = keys, items = queries,
// dots with q and g, sums with q and g.  The order of d within dots and of the
// columns within sums is permuted so that every lane loads 16 bytes.
//
// A workgroup's four waves have the same own rows and every fourth block of
// items; they are joined in LDS in a fixed order, and so are the parts of rows
// whose keys are split over workgroups (few rows over a long cache).
//
// What lies from lengths[b] on has no influence.  Within the length, a key that
// only some rows of a tile see may hold anything: where such a block has a value
// that is not finite, the sums go over visible pairs one by one (0 times an
// infinity would be NaN).
//
// What bounds them: few rows over a long cache, HBM (8 tokens of 32 heads over caches
// of up to 8192 x 8 x 128: 77 us for 403 MB and 7 for joining the 16 parts, 5.2 TB/s;
// of rows that four heads share, 12 of each instruction's 16 are empty, which costs
// nothing here); small texts, latency (4 x 128 tokens, 4 heads of 64: 8 us forward,
// 11 backward, of which an empty launch is 3); float64, loads that little hides (one
// or two waves to a SIMD): 2 x 1024 x 8 heads of 64 both passes 17 TFLOP/s of the 71 that
// a large product reaches, 2000 x 4 heads of 128 18.
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>

#include "attention.h"

namespace nt {

constexpr int AT_WAVES = 4;
constexpr int AT_MAX_D = 256;

template <class T> struct Mma;
template <> struct Mma<float> {
  typedef float V4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ V4 mma(float a, float b, V4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
  }
  // Row of a result's element r in lane group h.
  static __device__ __forceinline__ int row(int h, int r) { return 4 * h + r; }
  static __device__ __forceinline__ float exp2(float x) { return __builtin_amdgcn_exp2f(x); }
  static __device__ __forceinline__ float log2(float x) { return ::log2f(x); }
};
template <> struct Mma<double> {
  typedef double V4 __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ V4 mma(double a, double b, V4 c) {
    return __builtin_amdgcn_mfma_f64_16x16x4f64(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ int row(int h, int r) { return h + 4 * r; }
  static __device__ __forceinline__ double exp2(double x) { return ::exp2(x); }
  static __device__ __forceinline__ double log2(double x) { return ::log2(x); }
};

template <class T> constexpr T NEG_INF = -std::numeric_limits<T>::infinity();

// A row's share of a lane as operand of dots: pieces at 4 N c + N h.
template <class T, int DP> struct Frag {
  static constexpr int N = RowVec<T>::N, C = DP / (4 * N);
  typename RowVec<T>::V v[C];
  // From element d0 of a row of W on.
  __device__ __forceinline__ void load(const T *row, int d0, int W, int h) {
    W = afresh(W, row);
#pragma unroll
    for (int c = 0; c < C; ++c)
      v[c] = piece(row, d0 + 4 * N * c + N * h, W);
  }
  // A row of DP elements, aligned: no branch, so that many loads go out together.
  __device__ __forceinline__ void load_whole(const T *row, int h) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      v[c] = *reinterpret_cast<const typename RowVec<T>::V *>(row + 4 * N * c + N * h);
  }
};

template <class T, int DP>
__device__ __forceinline__ typename Mma<T>::V4 dots(const Frag<T, DP> &items,
                                                    const Frag<T, DP> &own) {
  typename Mma<T>::V4 s{};
#pragma unroll
  for (int c = 0; c < Frag<T, DP>::C; ++c)
#pragma unroll
    for (int e = 0; e < Frag<T, DP>::N; ++e)
      s = Mma<T>::mma(items.v[c][e], own.v[c][e], s);
  return s;
}

// The sum of a lane's elements' products.
template <class T, int DP>
__device__ __forceinline__ T times(const Frag<T, DP> &a, const Frag<T, DP> &b) {
  T sum = 0;
#pragma unroll
  for (int c = 0; c < Frag<T, DP>::C; ++c)
#pragma unroll
    for (int e = 0; e < Frag<T, DP>::N; ++e)
      sum = fma(a.v[c][e], b.v[c][e], sum);
  return sum;
}

// Columns of dk and dv that a workgroup keeps, at most 512 bytes of each; of float32
// rows over 128 wide, two workgroups form the same probabilities (float64 rows over 64
// wide have kernels of their own below).
template <class T, int DP> constexpr int KEY_COLUMNS = std::min(DP, 512 / int(sizeof(T)));

// Items' rows as operand of sums: of the four items row(h, r), pieces at
// 16 N c + N n of a workgroup's columns.  Where a result's columns are: see
// Sums::column.
template <class T, int DP> struct Items {
  static constexpr int N = RowVec<T>::N, C = DP / (16 * N);
  typename RowVec<T>::V v[4][C];
  // The columns from d0 on of a row of W.
  __device__ __forceinline__ void load(int r, const T *row, int d0, int W, int n) {
    W = afresh(W, row);
#pragma unroll
    for (int c = 0; c < C; ++c)
      v[r][c] = piece(row, d0 + N * (16 * c + n), W);
  }
  __device__ __forceinline__ void load_whole(int r, const T *p, int n) {
#pragma unroll
    for (int c = 0; c < C; ++c)
      v[r][c] = *reinterpret_cast<const typename RowVec<T>::V *>(p + N * (16 * c + n));
  }
};

template <class T, int DP> struct Sums {
  using V4 = typename Mma<T>::V4;
  static constexpr int N = RowVec<T>::N, C = DP / (16 * N);
  V4 acc[C][N]; // acc[c][e][r]: column(c, e, r) of the own row n
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e)
        acc[c][e] = V4{};
  }
  static __device__ __forceinline__ int column(int c, int e, int h, int r) {
    return 16 * N * c + N * Mma<T>::row(h, r) + e;
  }
  __device__ __forceinline__ void scale(T f) {
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
      for (int e = 0; e < N; ++e)
        acc[c][e] *= f;
  }
  __device__ __forceinline__ void add(const T (&a)[4], const Items<T, DP> &x) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int e = 0; e < N; ++e)
          acc[c][e] = Mma<T>::mma(x.v[r][c][e], a[r], acc[c][e]);
  }
  // The same over visible pairs only, from memory: `row(item)` is the item's row from
  // the sums' first column on, null past the end, with W elements from there (none, or
  // fewer than none, where the columns begin past its end).  In place of what lies past
  // its end its last piece is read, for sums that no one stores: no branches of a lane.
  template <class F>
  __device__ __forceinline__ void add_visible(const T (&a)[4], const bool (&vis)[4], int W,
                                              int lane, F row) {
    const int n = lane & 15, h = lane >> 4;
#pragma unroll 1
    for (int item = 0; item < 16; ++item) {
      const T *p = row(item);
      T w = 0;
      int on = 0;
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          if (Mma<T>::row(g, r) == item) {
            w = __shfl(a[r], n + 16 * g);
            on = __shfl(int(vis[r]), n + 16 * g);
          }
      if (p == nullptr)
        continue;
      const int last = afresh(W, item) - N;
#pragma unroll
      for (int c = 0; c < C; ++c)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const auto x = RowVec<T>::load(p + std::min(column(c, 0, h, r), last));
#pragma unroll
          for (int e = 0; e < N; ++e)
            acc[c][e][r] = on ? fma(w, x[e], acc[c][e][r]) : acc[c][e][r];
        }
    }
  }
};

// Joins the four waves' sums, each first multiplied by its lane's factor
// (of row n), and hands 16 by 16 N of them at a time to `out(row, column, value)`.
template <class T, int DP, class F>
__device__ __forceinline__ void join_waves(Sums<T, DP> &s, T factor, T *lds, F out) {
  constexpr int N = RowVec<T>::N, W = 16 * N; // columns of a turn
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
#pragma unroll
  for (int c = 0; c < Sums<T, DP>::C; ++c) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < N; ++e)
#pragma unroll
      for (int r = 0; r < 4; ++r)
        lds[(wave * 16 + n) * W + N * Mma<T>::row(h, r) + e] = s.acc[c][e][r] * factor;
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * W; i += 64 * AT_WAVES) {
      T v = lds[i];
#pragma unroll
      for (int w = 1; w < AT_WAVES; ++w)
        v += lds[w * 16 * W + i];
      out(i / W, c * W + i % W, v);
    }
  }
}

template <class T> constexpr int JOIN_ELEMENTS = AT_WAVES * 16 * 16 * RowVec<T>::N;

template <class T> __device__ __forceinline__ bool finite(typename RowVec<T>::V v) {
  bool f = true;
#pragma unroll
  for (int j = 0; j < RowVec<T>::N; ++j)
    f = f && __builtin_isfinite(v[j]);
  return f;
}

template <class T, int DP> __device__ __forceinline__ bool all_finite(const Items<T, DP> &x) {
  bool f = true;
#pragma unroll
  for (int r = 0; r < 4; ++r)
#pragma unroll
    for (int c = 0; c < Items<T, DP>::C; ++c)
      f = f && finite<T>(x.v[r][c]);
  return __all(f);
}

// ---------------------------------------------------------------- forward

// Tiles of 16 keys that a wave takes at a time, two blocks of which fit its registers
// beside two waves to a SIMD.
template <class T, int DP> constexpr int FWD_TILES = DP * sizeof(T) <= 256 ? 2 : 1;
// Rows of 1 KB, and of 512 bytes in float64, need the registers of one wave to a SIMD.
template <class T, int DP>
constexpr int FWD_WAVES =
    DP * sizeof(T) == 1024 || (sizeof(T) == 8 && DP * sizeof(T) == 512) ? 1 : 2;

// Tile `item` of a (sequence, key head).  WHOLE: rows of DP elements, aligned.
// MAY_AHEAD: the next keys may be loaded under a block.
template <class T, int DP, bool WHOLE, bool MAY_AHEAD>
__device__ __forceinline__ void attn_fwd_tile(const AttnFwd<T> &a, uint32_t bh, uint32_t item,
                                              uint32_t split) {
  using M = Mma<T>;
  constexpr int TILES = FWD_TILES<T, DP>;
  __shared__ T lds[JOIN_ELEMENTS<T>];
  __shared__ T stat[2][AT_WAVES][16];
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
  const uint32_t tiles = uint32_t(s.rows + 15) / 16;
  // long rows first: under a causal mask the last tiles see the most keys
  const int tile = int(tiles - 1 - item);
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, threadIdx.x == 0, keys, first);
  const int row = tile * 16 + n;
  const bool live = row < s.rows;
  const uint32_t at = uint32_t(std::min(row, s.rows - 1));
  const uint32_t qi = s.by_group.div(at), qg = at - qi * uint32_t(s.G);
  const int limit = live ? seen(s, keys, first, int(qi)) : 0;
  const int last = std::min(tile * 16 + 15, s.rows - 1);
  const int end = seen(s, keys, first, int(s.by_group.div(uint32_t(last)))); // of any row
  const int all = seen(s, keys, first, int(s.by_group.div(uint32_t(tile * 16)))); // of every row
  const T *qp = a.q.p + b * a.q.sB + hk * a.q.sHead + int64_t(qi) * a.q.sOuter +
                int64_t(qg) * a.q.sInner;
  const T *kp = a.k.p + b * a.k.sB + hk * a.k.sHead;
  const T *vp = a.v.p + b * a.v.sB + hk * a.v.sHead;
  Frag<T, DP> q;
  q.load(qp, 0, s.W, h);
  Sums<T, DP> sums;
  sums.clear();
  T m = NEG_INF<T>, l = 0;
  // this workgroup's blocks of keys, dealt to its waves
  const int blocks = (end + 16 * TILES - 1) / (16 * TILES);
  const int per = (blocks + a.splits - 1) / a.splits;
  const int stop = std::min(blocks, int(split + 1) * per);
  struct Keys {
    Frag<T, DP> k[TILES];
  };
  constexpr int STEP = 16 * TILES;
  // past the end the last key again, which no row sees there
  auto load_keys = [&](Keys &x, int j0) {
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int j = j0 + 16 * i + n;
      const T *p = kp + int64_t(std::min(j, end - 1)) * a.k.sOuter;
      if constexpr (WHOLE)
        x.k[i].load_whole(p, h);
      else
        x.k[i].load(p, 0, s.W, h);
    }
  };
  Items<T, DP> v[TILES];
  auto load_values = [&](int j0) {
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int j = j0 + 16 * i + M::row(h, r);
        const T *p = vp + int64_t(std::min(j, end - 1)) * a.v.sOuter;
        if constexpr (WHOLE)
          v[i].load_whole(r, p, n);
        else
          v[i].load(r, p, 0, s.W, n);
      }
  };
  auto take = [&](const Keys &x, int j0) {
    T z[TILES][4];
    bool vis[TILES][4];
    T top = NEG_INF<T>;
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const auto d = dots<T, DP>(x.k[i], q);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        vis[i][r] = j0 + 16 * i + M::row(h, r) < limit;
        z[i][r] = vis[i][r] ? d[r] * a.scale2 : NEG_INF<T>;
        top = fmax(top, z[i][r]);
      }
    }
    top = fmax(top, __shfl_xor(top, 16));
    top = fmax(top, __shfl_xor(top, 32));
    const T next = fmax(m, top);
    // a row that has seen nothing but -inf: exp2(-inf - 0) = 0, not NaN
    const T base = next == NEG_INF<T> ? T(0) : next;
    const T shrink = M::exp2(m - base);
    m = next;
    l *= shrink;
    sums.scale(shrink);
    T sum = 0;
#pragma unroll
    for (int i = 0; i < TILES; ++i)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // fmax drops a NaN; here it comes back
        z[i][r] = vis[i][r] ? M::exp2(z[i][r] - base) : T(0);
        sum += z[i][r];
      }
    l += sum;
#pragma unroll
    for (int i = 0; i < TILES; ++i) {
      const int j = j0 + 16 * i;
      if (j + 16 > all && !all_finite<T, DP>(v[i]))
        sums.add_visible(z[i], vis[i], s.W, lane, [&](int item) {
          return j + item < end ? vp + int64_t(j + item) * a.v.sOuter : nullptr;
        });
      else
        sums.add(z[i], v[i]);
    }
  };
  // A block's values and the next block's keys are on their way while its scores
  // are formed: few rows over many keys wait for memory.
  int blk = int(split) * per + wave;
  // (not of rows that leave no registers for two blocks of keys)
  constexpr bool AHEAD =
      MAY_AHEAD && (WHOLE || DP * sizeof(T) < 512 || (sizeof(T) == 4 && DP == 256));
  if constexpr (AHEAD) {
    if (blk < stop) {
      Keys x, y;
      load_keys(x, blk * STEP);
      auto turn = [&](const Keys &now, Keys &next) {
        const bool more = blk + AT_WAVES < stop;
        load_values(blk * STEP);
        if (more)
          load_keys(next, (blk + AT_WAVES) * STEP);
        take(now, blk * STEP);
        blk += AT_WAVES;
        return more;
      };
      while (turn(x, y) && turn(y, x))
        ;
    }
  } else {
    for (; blk < stop; blk += AT_WAVES) {
      Keys x;
      load_keys(x, blk * STEP);
      load_values(blk * STEP);
      take(x, blk * STEP);
    }
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (h == 0) {
    stat[0][wave][n] = m;
    stat[1][wave][n] = l;
  }
  __syncthreads();
  T top = stat[0][0][n];
#pragma unroll
  for (int w = 1; w < AT_WAVES; ++w)
    top = fmax(top, stat[0][w][n]);
  const T base = top == NEG_INF<T> ? T(0) : top;
  T total = 0;
#pragma unroll
  for (int w = 0; w < AT_WAVES; ++w)
    total += stat[1][w][n] * M::exp2(stat[0][w][n] - base);
  const T mine = M::exp2(m - base);
  if (a.splits > 1) {
    const int64_t slot = (int64_t(bh) * tiles + item) * a.splits + split;
    if (wave == 0 && h == 0) {
      a.part_stat[slot * 32 + n] = top;
      a.part_stat[slot * 32 + 16 + n] = total;
    }
    join_waves<T, DP>(sums, mine, lds, [&](int r, int d, T v) {
      if (d < s.D && tile * 16 + r < s.rows)
        a.part_acc[(slot * 16 + r) * s.D + d] = v;
    });
    return;
  }
  if (a.lse && wave == 0 && h == 0 && live)
    a.lse[int64_t(bh) * s.rows + row] = top == NEG_INF<T> ? T(0) : top + M::log2(total);
  const T factor = limit > 0 ? mine / total : T(0);
  join_waves<T, DP>(sums, factor, lds, [&](int r, int d, T v) {
    const int w = tile * 16 + r;
    if (d >= s.D || w >= s.rows)
      return;
    const uint32_t i = s.by_group.div(uint32_t(w));
    const int64_t head = int64_t(hk) * s.G + (uint32_t(w) - i * uint32_t(s.G));
    a.y[((int64_t(b) * s.Tq + i) * s.Hk * s.G + head) * s.D + d] = v;
  });
}

template <class T, int DP, bool WHOLE>
__global__ __launch_bounds__(64 * AT_WAVES, (FWD_WAVES<T, DP>)) void attn_fwd_kernel(
    const AttnFwd<T> a) {
  const uint32_t splits = uint32_t(a.splits);
  uint32_t bh, item;
  head_item(blockIdx.x, uint32_t(a.s.B) * uint32_t(a.s.Hk),
            uint32_t(a.s.rows + 15) / 16 * splits, bh, item);
  attn_fwd_tile<T, DP, WHOLE, true>(a, bh, item / splits, item % splits);
}

// What the kernels on half-precision planes left: the tiles of each (sequence,
// key head) dealt to `groups` workgroups.
template <int DP>
__global__ __launch_bounds__(64 * AT_WAVES) void attn_fwd_left_kernel(
    const AttnFwd<float> a, uint32_t groups) {
  const uint32_t bh = blockIdx.x / groups;
  if (!gate_set(a.gate, bh))
    return;
  const uint32_t tiles = uint32_t(a.s.rows + 15) / 16;
  for (uint32_t t = blockIdx.x % groups; t < tiles; t += groups) {
    __syncthreads();
    attn_fwd_tile<float, DP, false, false>(a, bh, t, 0);
  }
}

// Rows whose keys were split into at most 64 parts: a workgroup for each row, its
// waves every fourth part, joined in order.
template <class T>
__global__ __launch_bounds__(256) void attn_join_kernel(const AttnFwd<T> a) {
  const AttnShape &s = a.s;
  __shared__ T lds[3][AT_MAX_D];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int bh = int(blockIdx.x / uint32_t(s.rows)), row = int(blockIdx.x % uint32_t(s.rows));
  const int tiles = (s.rows + 15) / 16, n = row & 15;
  // the slots are numbered with the tiles backwards, as their workgroups were
  const int64_t slot = (int64_t(bh) * tiles + (tiles - 1 - row / 16)) * a.splits;
  T m = NEG_INF<T>, l = 0;
  if (lane < a.splits) {
    m = a.part_stat[(slot + lane) * 32 + n];
    l = a.part_stat[(slot + lane) * 32 + 16 + n];
  }
  T top = m;
#pragma unroll
  for (int o = 32; o; o >>= 1)
    top = fmax(top, __shfl_xor(top, o));
  const T weight = Mma<T>::exp2(m - (top == NEG_INF<T> ? T(0) : top));
  T total = l * weight;
#pragma unroll
  for (int o = 32; o; o >>= 1)
    total += __shfl_xor(total, o);
  T v[AT_MAX_D / 64];
#pragma unroll
  for (int c = 0; c < AT_MAX_D / 64; ++c) {
    v[c] = 0;
    const int d = c * 64 + lane;
#pragma unroll 4
    for (int k = wave; k < a.splits; k += 4) {
      const T w = __shfl(weight, k);
      if (d < s.D)
        v[c] = fma(a.part_acc[((slot + k) * 16 + n) * s.D + d], w, v[c]);
    }
    if (wave && d < s.D)
      lds[wave - 1][d] = v[c];
  }
  __syncthreads();
  if (wave)
    return;
  int keys, first;
  sequence(s, bh / s.Hk, false, keys, first);
  const uint32_t i = s.by_group.div(uint32_t(row));
  const bool any = seen(s, keys, first, int(i)) > 0;
  if (a.lse && lane == 0)
    a.lse[int64_t(bh) * s.rows + row] = top == NEG_INF<T> ? T(0) : top + Mma<T>::log2(total);
  const int64_t head = int64_t(bh % s.Hk) * s.G + (uint32_t(row) - i * uint32_t(s.G));
  T *y = a.y + ((int64_t(bh / s.Hk) * s.Tq + i) * s.Hk * s.G + head) * s.D;
#pragma unroll
  for (int c = 0; c < AT_MAX_D / 64; ++c) {
    const int d = c * 64 + lane;
    if (d < s.D) {
      for (int w = 0; w < 3; ++w)
        v[c] += lds[w][d];
      y[d] = any ? v[c] / total : T(0);
    }
  }
}

// --------------------------------------------------------------- backward

// A row's delta = g . y is formed where it is needed: a launch less, for one more
// row read with each of g.

template <class T, int DP>
__device__ __forceinline__ void attn_dq_tile(const AttnBwd<T> &a, uint32_t bh, uint32_t item) {
  using M = Mma<T>;
  __shared__ T lds[JOIN_ELEMENTS<T>];
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
  const uint32_t tiles = uint32_t(s.rows + 15) / 16;
  const int tile = int(tiles - 1 - item);
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, false, keys, first);
  const int row = tile * 16 + n;
  const bool live = row < s.rows;
  const uint32_t at = uint32_t(std::min(row, s.rows - 1));
  const uint32_t qi = s.by_group.div(at), qg = at - qi * uint32_t(s.G);
  const int limit = live ? seen(s, keys, first, int(qi)) : 0;
  const int last = std::min(tile * 16 + 15, s.rows - 1);
  const int end = seen(s, keys, first, int(s.by_group.div(uint32_t(last))));
  const int all = seen(s, keys, first, int(s.by_group.div(uint32_t(tile * 16))));
  const T *kp = a.k.p + b * a.k.sB + hk * a.k.sHead;
  const T *vp = a.v.p + b * a.v.sB + hk * a.v.sHead;
  const T *gp = a.g.p + b * a.g.sB + hk * a.g.sHead + int64_t(qi) * a.g.sOuter +
                int64_t(qg) * a.g.sInner;
  Frag<T, DP> q, g;
  q.load(a.q.p + b * a.q.sB + hk * a.q.sHead + int64_t(qi) * a.q.sOuter +
             int64_t(qg) * a.q.sInner,
         0, s.W, h);
  g.load(gp, 0, s.W, h);
  const T lse = a.lse[int64_t(bh) * s.rows + at];
  const T *yp = a.y.p + b * a.y.sB + hk * a.y.sHead + int64_t(qi) * a.y.sOuter +
                int64_t(qg) * a.y.sInner;
  T delta = 0;
#pragma unroll 1
  for (int d = 0; d < s.W; d += 4 * RowVec<T>::N * 4) {
    Frag<T, 16 * RowVec<T>::N> x, y;
    x.load(gp, d, s.W, h);
    y.load(yp, d, s.W, h);
    delta += times<T, 16 * RowVec<T>::N>(x, y);
  }
  delta += __shfl_xor(delta, 16);
  delta += __shfl_xor(delta, 32);
  Sums<T, DP> sums;
  sums.clear();
  for (int j0 = wave * 16; j0 < end; j0 += 16 * AT_WAVES) {
    Items<T, DP> x;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int j = j0 + M::row(h, r);
      x.load(r, kp + int64_t(std::min(j, end - 1)) * a.k.sOuter, 0, s.W, n);
    }
    const int64_t j = std::min(j0 + n, end - 1);
    Frag<T, DP> f;
    f.load(kp + j * a.k.sOuter, 0, s.W, h);
    const auto z = dots<T, DP>(f, q);
    f.load(vp + j * a.v.sOuter, 0, s.W, h);
    const auto dp = dots<T, DP>(f, g);
    T ds[4];
    bool vis[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vis[r] = j0 + M::row(h, r) < limit;
      ds[r] = vis[r] ? M::exp2(z[r] * a.scale2 - lse) * (dp[r] - delta) : T(0);
    }
    if (j0 + 16 > all && !all_finite<T, DP>(x))
      sums.add_visible(ds, vis, s.W, lane, [&](int item) {
        return j0 + item < end ? kp + int64_t(j0 + item) * a.k.sOuter : nullptr;
      });
    else
      sums.add(ds, x);
  }
  join_waves<T, DP>(sums, a.scale, lds, [&](int r, int d, T v) {
    const int w = tile * 16 + r;
    if (d >= s.D || w >= s.rows)
      return;
    const uint32_t i = s.by_group.div(uint32_t(w));
    const int64_t head = int64_t(hk) * s.G + (uint32_t(w) - i * uint32_t(s.G));
    a.dq[((int64_t(b) * s.Tq + i) * s.Hk * s.G + head) * s.D + d] = v;
  });
}

template <class T, int DP>
__device__ __forceinline__ void attn_dkv_tile(const AttnBwd<T> &a, uint32_t bh, uint32_t item,
                                              int col0) {
  using M = Mma<T>;
  constexpr int SC = KEY_COLUMNS<T, DP>;
  __shared__ T lds[JOIN_ELEMENTS<T>];
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
  const int key0 = int(item) * 16, key = key0 + n;
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, false, keys, first);
  const T *qp = a.q.p + b * a.q.sB + hk * a.q.sHead;
  const T *gp = a.g.p + b * a.g.sB + hk * a.g.sHead;
  const T *yp = a.y.p + b * a.y.sB + hk * a.y.sHead;
  auto at = [&](const T *p, const Rows<const T> &x, int row) {
    const uint32_t i = s.by_group.div(uint32_t(row));
    return p + int64_t(i) * x.sOuter + int64_t(uint32_t(row) - i * uint32_t(s.G)) * x.sInner;
  };
  Frag<T, DP> k, v;
  const int64_t own_key = std::min(key, s.Tk - 1);
  k.load(a.k.p + b * a.k.sB + hk * a.k.sHead + own_key * a.k.sOuter, 0, s.W, h);
  v.load(a.v.p + b * a.v.sB + hk * a.v.sHead + own_key * a.v.sOuter, 0, s.W, h);
  Sums<T, SC> dk, dv;
  dk.clear();
  dv.clear();
  // rows before the first query that sees any of these keys take no part
  int row0 = 0;
  if (key0 >= keys)
    row0 = s.rows;
  else if (s.causal && key0 > first)
    row0 = int(std::min<int64_t>(int64_t(key0 - first) * s.G, s.rows)) & ~15;
  const int clear = key0 + 16; // a row that sees so many sees all of this tile
  for (int r0 = row0 + wave * 16; r0 < s.rows; r0 += 16 * AT_WAVES) {
    Items<T, SC> xq, xg;
    auto load = [&](Items<T, SC> &x, const T *base, const Rows<const T> &of) {
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = r0 + M::row(h, r);
        x.load(r, at(base, of, row < s.rows ? row : 0), col0, s.W, n);
      }
    };
    load(xq, qp, a.q);
    load(xg, gp, a.g);
    T lse[4], delta[4];
    int limit[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = r0 + M::row(h, r);
      const bool on = row < s.rows;
      lse[r] = a.lse[int64_t(bh) * s.rows + (on ? row : 0)];
      limit[r] = on ? seen(s, keys, first, int(s.by_group.div(uint32_t(row)))) : 0;
    }
    const bool live = r0 + n < s.rows;
    const int own = live ? r0 + n : 0;
    Frag<T, DP> x, y;
    x.load(at(qp, a.q, own), 0, s.W, h);
    const auto z = dots<T, DP>(x, k);
    if constexpr (DP * sizeof(T) == 1024) // (the registers are full)
      __builtin_amdgcn_sched_barrier(0);
    x.load(at(gp, a.g, own), 0, s.W, h);
    y.load(at(yp, a.y, own), 0, s.W, h);
    const auto dp = dots<T, DP>(x, v);
    T product = times<T, DP>(x, y);
    product += __shfl_xor(product, 16);
    product += __shfl_xor(product, 32);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      delta[r] = __shfl(product, M::row(h, r));
    T p[4], ds[4];
    bool vis[4], some = false;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vis[r] = key < limit[r];
      some = some || limit[r] < clear;
      p[r] = vis[r] ? M::exp2(z[r] * a.scale2 - lse[r]) : T(0);
      ds[r] = vis[r] ? p[r] * (dp[r] - delta[r]) : T(0);
    }
    auto row_of = [&](const T *base, const Rows<const T> &x) {
      return [&, base](int item) {
        return r0 + item < s.rows ? at(base, x, r0 + item) + col0 : nullptr;
      };
    };
    if (__any(some) && !all_finite<T, SC>(xg))
      dv.add_visible(p, vis, s.W - col0, lane, row_of(gp, a.g));
    else
      dv.add(p, xg);
    if (__any(some) && !all_finite<T, SC>(xq))
      dk.add_visible(ds, vis, s.W - col0, lane, row_of(qp, a.q));
    else
      dk.add(ds, xq);
  }
  auto store = [&](T *out) {
    return [&, out](int r, int d, T x) {
      d += col0;
      if (d < s.D && key0 + r < s.Tk)
        out[((int64_t(b) * s.Tk + key0 + r) * s.Hk + hk) * s.D + d] = x;
    };
  };
  if (a.dv)
    join_waves<T, SC>(dv, T(1), lds, store(a.dv));
  if (a.dk)
    join_waves<T, SC>(dk, a.scale, lds, store(a.dk));
}

// Both gradients in one launch: tiles of keys, then tiles of rows.
template <class T, int DP>
__global__ __launch_bounds__(64 * AT_WAVES) void attn_bwd_kernel(const AttnBwd<T> a,
                                                                 uint32_t key_blocks) {
  constexpr uint32_t KEY_GROUPS = DP / KEY_COLUMNS<T, DP>;
  const AttnShape &s = a.s;
  const uint32_t heads = uint32_t(s.B) * uint32_t(s.Hk);
  uint32_t bh, item;
  if (blockIdx.x < key_blocks) {
    head_item(blockIdx.x, heads, uint32_t(s.Tk + 15) / 16 * KEY_GROUPS, bh, item);
    const int col0 = int(item % KEY_GROUPS) * KEY_COLUMNS<T, DP>;
    if (col0 < s.D)
      attn_dkv_tile<T, DP>(a, bh, item / KEY_GROUPS, col0);
  } else {
    head_item(blockIdx.x - key_blocks, heads, uint32_t(s.rows + 15) / 16, bh, item);
    attn_dq_tile<T, DP>(a, bh, item);
  }
}

// As attn_fwd_left_kernel.
template <int DP, bool DQ, bool DKV>
__global__ __launch_bounds__(64 * AT_WAVES) void attn_bwd_left_kernel(const AttnBwd<float> a,
                                                                     uint32_t groups) {
  const uint32_t bh = blockIdx.x / groups;
  if (!gate_set(a.gate, bh))
    return;
  const uint32_t rows = uint32_t(a.s.rows + 15) / 16, keys = uint32_t(a.s.Tk + 15) / 16;
  if (DQ && a.dq)
    for (uint32_t t = blockIdx.x % groups; t < rows; t += groups) {
      __syncthreads();
      attn_dq_tile<float, DP>(a, bh, t);
    }
  if (DKV && (a.dk || a.dv))
    for (uint32_t t = blockIdx.x % groups; t < keys; t += groups) {
      for (int col0 = 0; col0 < a.s.D; col0 += KEY_COLUMNS<float, DP>) {
        __syncthreads();
        attn_dkv_tile<float, DP>(a, bh, t, col0);
      }
    }
}

// ------------------------------------------------------- wide float64 rows

// float64 rows over 64 wide: a workgroup's four waves take the same items, each a
// quarter of the elements of every row, so that a quarter of the own rows, of the items
// and of the sums' columns lies in a wave's registers and no score is formed twice.  A
// score is the sum of the waves' four parts, which they exchange through two buffers
// of LDS, one barrier to a tile.  (Workgroups that formed all scores again for each 64
// columns, one wave to a SIMD, took 1100 us for 776 of 2000 x 4 heads of 128 and 2040
// for 950 of 900 x 6 over 3 of 256, both passes.)
template <class T, int DP> constexpr bool SHARED_ITEMS = sizeof(T) == 8 && DP >= 128;

// The waves' parts of a tile's result, summed in order; `turn` alternates.
template <class T> struct Exchange {
  using V4 = typename Mma<T>::V4;
  T part[2][AT_WAVES][4][64];
  __device__ __forceinline__ void put(int turn, int wave, int lane, V4 v) {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      part[turn][wave][r][lane] = v[r];
  }
  __device__ __forceinline__ V4 get(int turn, int lane) const {
    V4 v;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      v[r] = part[turn][0][r][lane];
#pragma unroll
      for (int w = 1; w < AT_WAVES; ++w)
        v[r] += part[turn][w][r][lane];
    }
    return v;
  }
};

// Calls out(column, value) for the own row n's sums, times a factor.
template <class T, int DP, class F>
__device__ __forceinline__ void each_sum(const Sums<T, DP> &s, T factor, int h, F out) {
#pragma unroll
  for (int c = 0; c < Sums<T, DP>::C; ++c)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int e = 0; e < Sums<T, DP>::N; ++e)
        out(Sums<T, DP>::column(c, e, h, r), s.acc[c][e][r] * factor);
}

template <class T, int DP>
__global__ __launch_bounds__(64 * AT_WAVES, DP <= 128 ? 2 : 1) void attn_wide_fwd_kernel(const AttnFwd<T> a) {
  using M = Mma<T>;
  constexpr int PART = DP / AT_WAVES;
  __shared__ Exchange<T> scores;
  const AttnShape &s = a.s;
  const uint32_t splits = uint32_t(a.splits), tiles = uint32_t(s.rows + 15) / 16;
  uint32_t bh, item;
  head_item(blockIdx.x, uint32_t(s.B) * uint32_t(s.Hk), tiles * splits, bh, item);
  const uint32_t split = item % splits;
  item /= splits;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
  const int col0 = wave * PART, tile = int(tiles - 1 - item);
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, threadIdx.x == 0, keys, first);
  const int row = tile * 16 + n;
  const bool live = row < s.rows;
  const uint32_t at = uint32_t(std::min(row, s.rows - 1));
  const uint32_t qi = s.by_group.div(at), qg = at - qi * uint32_t(s.G);
  const int limit = live ? seen(s, keys, first, int(qi)) : 0;
  const int last = std::min(tile * 16 + 15, s.rows - 1);
  const int end = seen(s, keys, first, int(s.by_group.div(uint32_t(last)))); // of any row
  const int all = seen(s, keys, first, int(s.by_group.div(uint32_t(tile * 16)))); // of every row
  const T *kp = a.k.p + b * a.k.sB + hk * a.k.sHead;
  const T *vp = a.v.p + b * a.v.sB + hk * a.v.sHead;
  Frag<T, PART> q;
  q.load(a.q.p + b * a.q.sB + hk * a.q.sHead + int64_t(qi) * a.q.sOuter +
             int64_t(qg) * a.q.sInner,
         col0, s.W, h);
  Sums<T, PART> sums;
  sums.clear();
  T m = NEG_INF<T>, l = 0;
  const int blocks = (end + 15) / 16, per = (blocks + int(splits) - 1) / int(splits);
  const int stop = std::min(blocks, int(split + 1) * per);
  Frag<T, PART> k;
  auto load_keys = [&](int blk) { // past the end the last key again, which no row sees
    k.load(kp + int64_t(std::min(blk * 16 + n, end - 1)) * a.k.sOuter, col0, s.W, h);
  };
  int turn = 0, blk = int(split) * per;
  if (blk < stop)
    load_keys(blk);
  for (; blk < stop; ++blk, turn ^= 1) {
    const int j0 = blk * 16;
    Items<T, PART> v;
#pragma unroll
    for (int r = 0; r < 4; ++r)
      v.load(r, vp + int64_t(std::min(j0 + M::row(h, r), end - 1)) * a.v.sOuter, col0, s.W, n);
    scores.put(turn, wave, lane, dots<T, PART>(k, q));
    load_keys(std::min(blk + 1, stop - 1)); // on their way over the barrier
    __syncthreads();
    const auto d = scores.get(turn, lane);
    T z[4], top = NEG_INF<T>;
    bool vis[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vis[r] = j0 + M::row(h, r) < limit;
      z[r] = vis[r] ? d[r] * a.scale2 : NEG_INF<T>;
      top = fmax(top, z[r]);
    }
    top = fmax(top, __shfl_xor(top, 16));
    top = fmax(top, __shfl_xor(top, 32));
    const T next = fmax(m, top);
    const T base = next == NEG_INF<T> ? T(0) : next;
    const T shrink = M::exp2(m - base);
    m = next;
    l *= shrink;
    sums.scale(shrink);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      z[r] = vis[r] ? M::exp2(z[r] - base) : T(0);
      l += z[r];
    }
    if (j0 + 16 > all && !all_finite<T, PART>(v))
      sums.add_visible(z, vis, s.W - col0, lane, [&](int i) {
        return j0 + i < end ? vp + int64_t(j0 + i) * a.v.sOuter + col0 : nullptr;
      });
    else
      sums.add(z, v);
  }
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  if (splits > 1) {
    const int64_t slot = (int64_t(bh) * tiles + item) * splits + split;
    if (wave == 0 && h == 0) {
      a.part_stat[slot * 32 + n] = m;
      a.part_stat[slot * 32 + 16 + n] = l;
    }
    each_sum(sums, T(1), h, [&](int d, T x) {
      if (col0 + d < s.D && live)
        a.part_acc[(slot * 16 + n) * s.D + col0 + d] = x;
    });
    return;
  }
  if (!live)
    return;
  if (a.lse && wave == 0 && h == 0)
    a.lse[int64_t(bh) * s.rows + row] = m == NEG_INF<T> ? T(0) : m + M::log2(l);
  T *y = a.y + ((int64_t(b) * s.Tq + qi) * s.Hk * s.G + int64_t(hk) * s.G + qg) * s.D + col0;
  each_sum(sums, limit > 0 ? T(1) / l : T(0), h, [&](int d, T x) {
    if (col0 + d < s.D)
      y[d] = x;
  });
}

template <class T, int DP>
__device__ __forceinline__ void attn_wide_dq_tile(const AttnBwd<T> &a, uint32_t bh, uint32_t item,
                                                  Exchange<T> &scores, Exchange<T> &others) {
  using M = Mma<T>;
  constexpr int PART = DP / AT_WAVES;
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
  const int col0 = wave * PART, tile = int(uint32_t(s.rows + 15) / 16 - 1 - item);
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, false, keys, first);
  const int row = tile * 16 + n;
  const bool live = row < s.rows;
  const uint32_t at = uint32_t(std::min(row, s.rows - 1));
  const uint32_t qi = s.by_group.div(at), qg = at - qi * uint32_t(s.G);
  const int limit = live ? seen(s, keys, first, int(qi)) : 0;
  const int last = std::min(tile * 16 + 15, s.rows - 1);
  const int end = seen(s, keys, first, int(s.by_group.div(uint32_t(last))));
  const int all = seen(s, keys, first, int(s.by_group.div(uint32_t(tile * 16))));
  const T *kp = a.k.p + b * a.k.sB + hk * a.k.sHead;
  const T *vp = a.v.p + b * a.v.sB + hk * a.v.sHead;
  const T *gp = a.g.p + b * a.g.sB + hk * a.g.sHead + int64_t(qi) * a.g.sOuter +
                int64_t(qg) * a.g.sInner;
  const T *yp = a.y.p + b * a.y.sB + hk * a.y.sHead + int64_t(qi) * a.y.sOuter +
                int64_t(qg) * a.y.sInner;
  Frag<T, PART> q, g;
  q.load(a.q.p + b * a.q.sB + hk * a.q.sHead + int64_t(qi) * a.q.sOuter +
             int64_t(qg) * a.q.sInner,
         col0, s.W, h);
  g.load(gp, col0, s.W, h);
  const T lse = a.lse[int64_t(bh) * s.rows + at];
  T delta = 0;
#pragma unroll 1
  for (int d = 0; d < s.W; d += 16 * RowVec<T>::N) {
    Frag<T, 16 * RowVec<T>::N> x, y;
    x.load(gp, d, s.W, h);
    y.load(yp, d, s.W, h);
    delta += times<T, 16 * RowVec<T>::N>(x, y);
  }
  delta += __shfl_xor(delta, 16);
  delta += __shfl_xor(delta, 32);
  Sums<T, PART> sums;
  sums.clear();
  int turn = 0;
  for (int j0 = 0; j0 < end; j0 += 16, turn ^= 1) {
    Frag<T, PART> k, v;
    Items<T, PART> x;
    const int64_t j = std::min(j0 + n, end - 1);
    k.load(kp + j * a.k.sOuter, col0, s.W, h);
    v.load(vp + j * a.v.sOuter, col0, s.W, h);
#pragma unroll
    for (int r = 0; r < 4; ++r)
      x.load(r, kp + int64_t(std::min(j0 + M::row(h, r), end - 1)) * a.k.sOuter, col0, s.W, n);
    scores.put(turn, wave, lane, dots<T, PART>(k, q));
    others.put(turn, wave, lane, dots<T, PART>(v, g));
    __syncthreads();
    const auto z = scores.get(turn, lane), dp = others.get(turn, lane);
    T ds[4];
    bool vis[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      vis[r] = j0 + M::row(h, r) < limit;
      ds[r] = vis[r] ? M::exp2(z[r] * a.scale2 - lse) * (dp[r] - delta) : T(0);
    }
    if (j0 + 16 > all && !all_finite<T, PART>(x))
      sums.add_visible(ds, vis, s.W - col0, lane, [&](int i) {
        return j0 + i < end ? kp + int64_t(j0 + i) * a.k.sOuter + col0 : nullptr;
      });
    else
      sums.add(ds, x);
  }
  if (!live)
    return;
  T *out = a.dq + ((int64_t(b) * s.Tq + qi) * s.Hk * s.G + int64_t(hk) * s.G + qg) * s.D + col0;
  each_sum(sums, a.scale, h, [&](int d, T x) {
    if (col0 + d < s.D)
      out[d] = x;
  });
}

template <class T, int DP>
__device__ __forceinline__ void attn_wide_dkv_tile(const AttnBwd<T> &a, uint32_t bh, uint32_t item,
                                                   Exchange<T> &scores, Exchange<T> &others,
                                                   T (&deltas)[2][AT_WAVES][16]) {
  using M = Mma<T>;
  constexpr int PART = DP / AT_WAVES;
  const AttnShape &s = a.s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, n = lane & 15, h = lane >> 4;
  const int col0 = wave * PART, key0 = int(item) * 16, key = key0 + n;
  const int b = int(bh) / s.Hk, hk = int(bh) % s.Hk;
  int keys, first;
  sequence(s, b, false, keys, first);
  const T *qp = a.q.p + b * a.q.sB + hk * a.q.sHead;
  const T *gp = a.g.p + b * a.g.sB + hk * a.g.sHead;
  const T *yp = a.y.p + b * a.y.sB + hk * a.y.sHead;
  auto at = [&](const T *p, const Rows<const T> &x, int row) {
    const uint32_t i = s.by_group.div(uint32_t(row));
    return p + int64_t(i) * x.sOuter + int64_t(uint32_t(row) - i * uint32_t(s.G)) * x.sInner;
  };
  Frag<T, PART> k, v;
  const int64_t own_key = std::min(key, s.Tk - 1);
  k.load(a.k.p + b * a.k.sB + hk * a.k.sHead + own_key * a.k.sOuter, col0, s.W, h);
  v.load(a.v.p + b * a.v.sB + hk * a.v.sHead + own_key * a.v.sOuter, col0, s.W, h);
  Sums<T, PART> dk, dv;
  dk.clear();
  dv.clear();
  // rows before the first query that sees any of these keys take no part
  int row0 = 0;
  if (key0 >= keys)
    row0 = s.rows;
  else if (s.causal && key0 > first)
    row0 = int(std::min<int64_t>(int64_t(key0 - first) * s.G, s.rows)) & ~15;
  const int clear = key0 + 16; // a row that sees so many sees all of this tile
  int turn = 0;
  for (int r0 = row0; r0 < s.rows; r0 += 16, turn ^= 1) {
    const int own = r0 + n < s.rows ? r0 + n : 0;
    Frag<T, PART> x, g, y;
    x.load(at(qp, a.q, own), col0, s.W, h);
    g.load(at(gp, a.g, own), col0, s.W, h);
    y.load(at(yp, a.y, own), col0, s.W, h);
    Items<T, PART> xq, xg;
    T lse[4];
    int limit[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int row = r0 + M::row(h, r);
      const bool on = row < s.rows;
      xg.load(r, at(gp, a.g, on ? row : 0), col0, s.W, n);
      xq.load(r, at(qp, a.q, on ? row : 0), col0, s.W, n);
      lse[r] = a.lse[int64_t(bh) * s.rows + (on ? row : 0)];
      limit[r] = on ? seen(s, keys, first, int(s.by_group.div(uint32_t(row)))) : 0;
    }
    scores.put(turn, wave, lane, dots<T, PART>(x, k));
    others.put(turn, wave, lane, dots<T, PART>(g, v));
    T product = times<T, PART>(g, y);
    product += __shfl_xor(product, 16);
    product += __shfl_xor(product, 32);
    if (h == 0)
      deltas[turn][wave][n] = product;
    __syncthreads();
    const auto z = scores.get(turn, lane), dp = others.get(turn, lane);
    T p[4], ds[4];
    bool vis[4], some = false;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      T delta = 0;
#pragma unroll
      for (int w = 0; w < AT_WAVES; ++w)
        delta += deltas[turn][w][M::row(h, r)];
      vis[r] = key < limit[r];
      some = some || limit[r] < clear;
      p[r] = vis[r] ? M::exp2(z[r] * a.scale2 - lse[r]) : T(0);
      ds[r] = vis[r] ? p[r] * (dp[r] - delta) : T(0);
    }
    auto row_of = [&](const T *base, const Rows<const T> &of) {
      return [&, base](int i) {
        return r0 + i < s.rows ? at(base, of, r0 + i) + col0 : nullptr;
      };
    };
    if (__any(some) && !all_finite<T, PART>(xg))
      dv.add_visible(p, vis, s.W - col0, lane, row_of(gp, a.g));
    else
      dv.add(p, xg);
    if (__any(some) && !all_finite<T, PART>(xq))
      dk.add_visible(ds, vis, s.W - col0, lane, row_of(qp, a.q));
    else
      dk.add(ds, xq);
  }
  if (key >= s.Tk)
    return;
  const int64_t out = ((int64_t(b) * s.Tk + key) * s.Hk + hk) * s.D + col0;
  if (a.dv)
    each_sum(dv, T(1), h, [&](int d, T x) {
      if (col0 + d < s.D)
        a.dv[out + d] = x;
    });
  if (a.dk)
    each_sum(dk, a.scale, h, [&](int d, T x) {
      if (col0 + d < s.D)
        a.dk[out + d] = x;
    });
}

// As attn_bwd_kernel.
template <class T, int DP>
__global__ __launch_bounds__(64 * AT_WAVES, DP <= 128 ? 2 : 1) void attn_wide_bwd_kernel(
    const AttnBwd<T> a, uint32_t key_blocks) {
  __shared__ Exchange<T> scores, others;
  __shared__ T deltas[2][AT_WAVES][16];
  const AttnShape &s = a.s;
  const uint32_t heads = uint32_t(s.B) * uint32_t(s.Hk);
  uint32_t bh, item;
  if (blockIdx.x < key_blocks) {
    head_item(blockIdx.x, heads, uint32_t(s.Tk + 15) / 16, bh, item);
    attn_wide_dkv_tile<T, DP>(a, bh, item, scores, others, deltas);
  } else {
    head_item(blockIdx.x - key_blocks, heads, uint32_t(s.rows + 15) / 16, bh, item);
    attn_wide_dq_tile<T, DP>(a, bh, item, scores, others);
  }
}

// x [B, tokens, heads, D] -> contiguous rows of W elements, zeros past D.
template <class T>
__global__ __launch_bounds__(256) void attn_pad_kernel(const Rows<const T> x, T *to, int64_t rows,
                                                       int tokens, int heads, int D, int W) {
  using R = RowVec<T>;
  const int per = W / R::N;
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x, row = i / per;
  if (row >= rows)
    return;
  const int d = int(i - row * per) * R::N;
  const int64_t t = row / heads;
  const T *p = x.p + t / tokens * x.sB + t % tokens * x.sOuter + row % heads * x.sInner;
  typename R::V v{};
#pragma unroll
  for (int j = 0; j < R::N; ++j)
    if (d + j < D)
      v[j] = p[d + j];
  R::store(to + row * W + d, v);
}

// ------------------------------------------------------------------- host

namespace {

void check_heads(const nt_view *v, const nt_view *like, const char *what) {
  check_view(v, what);
  if (v->dtype != like->dtype)
    fail(NT_ERR_VALUE, std::string("attention: ") + what + " has another dtype than q");
  if (v->ndim != 4)
    fail(NT_ERR_RUNTIME, std::string("attention: ") + what + " must be [B, T, heads, D]");
  if (v->shape[0] != like->shape[0] || v->shape[3] != like->shape[3])
    fail(NT_ERR_RUNTIME, std::string("attention: ") + what + " has another batch or width");
  if (v->shape[3] > 1 && v->strides[3] != 1)
    fail(NT_ERR_RUNTIME, std::string("attention: ") + what + " needs adjacent elements in a head");
}

Tokens per_sequence(const nt_view *v, int64_t B, const char *what) {
  Tokens t{};
  if (v == nullptr)
    return t;
  t = token_view(v, "attention");
  if (v->shape[0] != B)
    fail(NT_ERR_RUNTIME, std::string("attention: one of ") + what + " for each sequence");
  return t;
}

// Tiles of 16 rows of one launch: its work-items are counted in 32 bits, with three
// workgroups of 256 at most for a tile of rows and one of keys.
constexpr int64_t MOST_TILES = int64_t(1) << 21;

// Some of the sequences of a view [B, ...], or of a contiguous array of B parts.
nt_view sequences(const nt_view *v, int64_t b, int64_t n) {
  nt_view p = *v;
  p.offset += b * p.strides[0];
  p.shape[0] = n;
  return p;
}
nt_view parts(const nt_view *v, int64_t B, int64_t b, int64_t n) {
  nt_view p = *v;
  const int64_t each = numel(v) / B;
  p.offset += b * each;
  p.ndim = 1;
  p.shape[0] = n * each;
  p.strides[0] = 1;
  return p;
}

// Into how many launches' worth of sequences a call goes: one but for very many
// rows.  0: the views are not what they should be, which attn_shape reports.
int64_t sequences_at_once(const nt_view *q, const nt_view *k) {
  if (q == nullptr || k == nullptr || q->ndim != 4 || k->ndim != 4 || q->shape[0] < 2 ||
      k->shape[2] < 1)
    return 0;
  for (const nt_view *v : {q, k})
    for (int i = 0; i < 4; ++i)
      if (v->shape[i] < 0 || v->shape[i] >= (int64_t(1) << 30))
        return 0;
  const int64_t Hk = k->shape[2];
  const int64_t rows = std::max(q->shape[1] * (q->shape[2] / Hk), k->shape[1]);
  if (rows >= (int64_t(1) << 30))
    return 0;
  return std::max<int64_t>(1, (MOST_TILES - 1) / std::max<int64_t>(1, Hk * ((rows + 15) / 16)));
}

AttnShape attn_shape(const nt_view *q, const nt_view *k, const nt_view *v,
                     const nt_view *lengths, const nt_view *starts, int64_t start,
                     int32_t causal, double scale) {
  check_heads(q, q, "q");
  if (!(std::abs(scale) < (q->dtype == NT_FLOAT32 ? 0x1p127 : 0x1p1023)))
    fail(NT_ERR_VALUE, "attention: the scale must be finite in the operands' type");
  check_heads(k, q, "k");
  check_heads(v, q, "v");
  require_same_shape(k, v, "attention");
  const int64_t B = q->shape[0], Tq = q->shape[1], H = q->shape[2], D = q->shape[3];
  const int64_t Tk = k->shape[1], Hk = k->shape[2];
  if (causal < 0 || causal > 2)
    fail(NT_ERR_VALUE, "attention: causal is 0, 1 or 2");
  if (D < 1 || D > AT_MAX_D)
    fail(NT_ERR_VALUE, "attention: heads of 1 to 256 elements");
  if (Hk < 1 || H < 1 || H % Hk)
    fail(NT_ERR_VALUE, "attention: the query heads must be a multiple of the key heads");
  constexpr int64_t MOST = int64_t(1) << 30;
  const int64_t G = H / Hk;
  if (B >= MOST || Tk >= MOST || Tq >= MOST || H >= MOST || Tq * G >= MOST || B * Hk >= MOST ||
      (B * Hk) * ((std::max(Tq * G, Tk) + 15) / 16) >= MOST_TILES)
    fail(NT_ERR_VALUE, "attention: too many rows");
  AttnShape s{};
  s.B = int(B), s.Tq = int(Tq), s.Tk = int(Tk), s.Hk = int(Hk), s.G = int(G), s.D = int(D);
  s.W = int((D * int64_t(dtype_size(q->dtype)) + 15) / 16 * 16 / int64_t(dtype_size(q->dtype)));
  s.rows = int(Tq * G);
  s.by_group = FastDivU32(uint32_t(G));
  s.causal = causal;
  s.start = start;
  s.lengths = per_sequence(lengths, B, "lengths");
  s.starts = per_sequence(starts, B, "starts");
  s.err = deferred_error_word();
  return s;
}

// q, g (G heads to a group) or k, v (G = 1).
template <class T> Rows<T> rows_of(const nt_view *v, int64_t G) {
  Rows<T> r;
  r.p = typed_ptr<T>(v);
  r.sB = v->strides[0];
  r.sOuter = v->strides[1];
  r.sInner = v->strides[2];
  r.sHead = v->strides[2] * G;
  return r;
}

bool whole_pieces(const nt_view *v) {
  const int64_t n = int64_t(16 / dtype_size(v->dtype));
  bool ok = v->shape[3] % n == 0 &&
            (reinterpret_cast<uintptr_t>(v->data) + size_t(v->offset) * dtype_size(v->dtype)) %
                    16 ==
                0;
  for (int i = 0; i < 3; ++i)
    ok = ok && (v->shape[i] <= 1 || v->strides[i] % n == 0);
  return ok;
}

template <class T> T *contiguous_of(const nt_view *v, int64_t n, int dt, const char *what) {
  check_view(v, what);
  if (v->dtype != dt)
    fail(NT_ERR_VALUE, std::string("attention: ") + what + " has another dtype than q");
  if (numel(v) != n || !is_contiguous(v))
    fail(NT_ERR_RUNTIME, std::string("attention: ") + what + " must be contiguous, of " +
                             std::to_string(n) + " elements");
  return typed_ptr<T>(v);
}

// Rows whose length is no multiple of 16 bytes are copied with zeros behind them:
// the kernels read whole pieces only.
template <class T> struct Padded {
  DeviceScratch memory;
  static size_t bytes(const AttnShape &s, int64_t tokens, int64_t heads) {
    return s.W == s.D ? 0 : size_t(s.B) * size_t(tokens) * size_t(heads) * size_t(s.W) * sizeof(T);
  }
  Padded(const AttnShape &s, Rows<const T> &x, int tokens, int heads, int G)
      : memory(bytes(s, tokens, heads)) {
    if (s.W == s.D)
      return;
    const int64_t rows = int64_t(s.B) * tokens * heads;
    T *to = memory.template get<T>();
    if (rows) {
      const int64_t pieces = rows * (s.W / RowVec<T>::N);
      attn_pad_kernel<T><<<dim3(uint32_t((pieces + 255) / 256)), 256, 0, stream()>>>(
          x, to, rows, tokens, heads, s.D, s.W);
      NT_LAUNCH_CHECK();
    }
    x.p = to;
    x.sInner = s.W;
    x.sHead = int64_t(s.W) * G;
    x.sOuter = int64_t(s.W) * heads;
    x.sB = x.sOuter * tokens;
  }
};

// The padded width: the matrix instructions' columns come 16 pieces at a time.
template <class T, class F> void dispatch_width(int D, F &&f) {
  if (D <= 32 && sizeof(T) == 8)
    f.template operator()<sizeof(T) == 8 ? 32 : 64>();
  else if (D <= 64)
    f.template operator()<64>();
  else if (D <= 128)
    f.template operator()<128>();
  else
    f.template operator()<256>();
}

// Into how many parts each tile's keys are split: as many as fill the chip
// (four workgroups a CU; three and six measured no faster), with at least two blocks
// to a wave.
int key_splits(const AttnShape &s) {
  const int64_t groups = int64_t(s.B) * s.Hk * ((s.rows + 15) / 16);
  const int64_t want = int64_t(device_cu_count()) * 4 / std::max<int64_t>(groups, 1);
  const int64_t most = s.Tk / (32 * AT_WAVES * 2);
  return int(std::max<int64_t>(1, std::min({want, most, int64_t(64)})));
}

// Workgroups for each (sequence, key head) that the other kernels left, or not: those
// of one that was not leave at once, the others take its tiles in turn.  Of few, each
// has the whole chip's: with 32 at most, one of four left of 8192 x 8192 x 128 took both
// passes from 4.7 to 60 ms, with 256 to 13.7 (all four: 59 and 27; the plain form 30).
uint32_t left_groups(uint32_t bhs) { return std::clamp<uint32_t>(1024 / bhs, 1, 256); }

template <class T> void run_attention(AttnFwd<T> &a) {
  const AttnShape &s = a.s;
  if constexpr (std::is_same_v<T, float>)
    if (split_takes(s, false)) {
      DeviceScratch words(split_gate_words(s, false) * sizeof(uint32_t));
      run_split(a, words.get<uint32_t>());
      a.splits = 1;
      const uint32_t bhs = uint32_t(s.B) * uint32_t(s.Hk), groups = left_groups(bhs);
      dispatch_width<float>(s.D, [&]<int DP>() {
        attn_fwd_left_kernel<DP>
            <<<dim3(groups * bhs), 64 * AT_WAVES, 0, stream()>>>(a, groups);
      });
      NT_LAUNCH_CHECK();
      return;
    }
  const int64_t tiles = int64_t(s.B) * s.Hk * ((s.rows + 15) / 16);
  a.splits = key_splits(s);
  const size_t slots = a.splits > 1 ? size_t(tiles) * size_t(a.splits) : 0;
  DeviceScratch acc(slots * 16 * size_t(s.D) * sizeof(T)), stat(slots * 32 * sizeof(T));
  a.part_acc = acc.template get<T>();
  a.part_stat = stat.template get<T>();
  dispatch_width<T>(s.D, [&]<int DP>() {
    const dim3 grid(uint32_t(tiles * a.splits));
    if constexpr (SHARED_ITEMS<T, DP>)
      attn_wide_fwd_kernel<T, DP><<<grid, 64 * AT_WAVES, 0, stream()>>>(a);
    else if (a.vec && s.D == DP)
      attn_fwd_kernel<T, DP, true><<<grid, 64 * AT_WAVES, 0, stream()>>>(a);
    else
      attn_fwd_kernel<T, DP, false><<<grid, 64 * AT_WAVES, 0, stream()>>>(a);
  });
  NT_LAUNCH_CHECK();
  if (a.splits > 1) {
    attn_join_kernel<T>
        <<<dim3(uint32_t(int64_t(s.B) * s.Hk * s.rows)), 256, 0, stream()>>>(a);
    NT_LAUNCH_CHECK();
  }
}

template <class T> void run_attention_bwd(AttnBwd<T> &a) {
  const AttnShape &s = a.s;
  if constexpr (std::is_same_v<T, float>)
    if (split_takes(s, true)) {
      DeviceScratch words(split_gate_words(s, true) * sizeof(uint32_t));
      run_split_bwd(a, words.get<uint32_t>());
      const uint32_t bhs = uint32_t(s.B) * uint32_t(s.Hk), groups = left_groups(bhs);
      dispatch_width<float>(s.D, [&]<int DP>() {
        // (one kernel for both keeps too much of wide rows)
        attn_bwd_left_kernel<DP, true, (DP <= 128)>
            <<<dim3(groups * bhs), 64 * AT_WAVES, 0, stream()>>>(a, groups);
        if constexpr (DP > 128)
          attn_bwd_left_kernel<DP, false, true>
              <<<dim3(groups * bhs), 64 * AT_WAVES, 0, stream()>>>(a, groups);
      });
      NT_LAUNCH_CHECK();
      return;
    }
  dispatch_width<T>(s.D, [&]<int DP>() {
    const uint32_t bhs = uint32_t(s.B) * uint32_t(s.Hk);
    constexpr bool SHARED = SHARED_ITEMS<T, DP>;
    constexpr uint32_t KEY_GROUPS = SHARED ? 1 : DP / KEY_COLUMNS<T, DP>;
    const uint32_t keys = a.dk || a.dv ? bhs * uint32_t((s.Tk + 15) / 16) * KEY_GROUPS : 0;
    const uint32_t rows = a.dq ? bhs * uint32_t((s.rows + 15) / 16) : 0;
    if (keys + rows == 0)
      return;
    if constexpr (SHARED)
      attn_wide_bwd_kernel<T, DP><<<dim3(keys + rows), 64 * AT_WAVES, 0, stream()>>>(a, keys);
    else
      attn_bwd_kernel<T, DP><<<dim3(keys + rows), 64 * AT_WAVES, 0, stream()>>>(a, keys);
    NT_LAUNCH_CHECK();
  });
}

} // namespace

} // namespace nt

namespace nt {
namespace {

void attention(const nt_view *q, const nt_view *k, const nt_view *v, const nt_view *lengths,
               const nt_view *starts, int64_t start, int32_t causal, double scale,
               const nt_view *y, const nt_view *lse) {
  const AttnShape s = attn_shape(q, k, v, lengths, starts, start, causal, scale);
  dispatch_float(q->dtype, [&]<class T>() {
    AttnFwd<T> a{};
    a.s = s;
    a.q = rows_of<const T>(q, s.G);
    a.k = rows_of<const T>(k, 1);
    a.v = rows_of<const T>(v, 1);
    a.y = contiguous_of<T>(y, numel(q), q->dtype, "y");
    const int64_t rows = int64_t(s.B) * s.Hk * s.rows;
    if (lse)
      a.lse = contiguous_of<T>(lse, rows, q->dtype, "lse");
    a.scale2 = T(scale * 1.4426950408889634);
    a.vec = whole_pieces(q) && whole_pieces(k) && whole_pieces(v);
    if (rows == 0)
      return;
    const int H = s.Hk * s.G;
    Padded<T> pq(s, a.q, s.Tq, H, s.G), pk(s, a.k, s.Tk, s.Hk, 1), pv(s, a.v, s.Tk, s.Hk, 1);
    run_attention(a);
  });
}

void attention_bwd(const nt_view *q, const nt_view *k, const nt_view *v, const nt_view *lengths,
                   const nt_view *starts, int64_t start, int32_t causal, double scale,
                   const nt_view *y, const nt_view *lse, const nt_view *g, const nt_view *dq,
                   const nt_view *dk, const nt_view *dv) {
  const AttnShape s = attn_shape(q, k, v, lengths, starts, start, causal, scale);
  check_heads(g, q, "g");
  require_same_shape(g, q, "attention_bwd");
  dispatch_float(q->dtype, [&]<class T>() {
    AttnBwd<T> a{};
    a.s = s;
    a.q = rows_of<const T>(q, s.G);
    a.k = rows_of<const T>(k, 1);
    a.v = rows_of<const T>(v, 1);
    a.g = rows_of<const T>(g, s.G);
    a.y.p = contiguous_of<const T>(y, numel(q), q->dtype, "y");
    a.y.sInner = s.D;
    a.y.sHead = int64_t(s.D) * s.G;
    a.y.sOuter = a.y.sHead * s.Hk;
    a.y.sB = a.y.sOuter * s.Tq;
    a.lse = contiguous_of<const T>(lse, int64_t(s.B) * s.Hk * s.rows, q->dtype, "lse");
    if (dq)
      a.dq = contiguous_of<T>(dq, numel(q), q->dtype, "dq");
    if (dk)
      a.dk = contiguous_of<T>(dk, numel(k), q->dtype, "dk");
    if (dv)
      a.dv = contiguous_of<T>(dv, numel(v), q->dtype, "dv");
    a.scale = T(scale);
    a.scale2 = T(scale * 1.4426950408889634);
    const int H = s.Hk * s.G;
    Padded<T> pq(s, a.q, s.Tq, H, s.G), pk(s, a.k, s.Tk, s.Hk, 1), pv(s, a.v, s.Tk, s.Hk, 1);
    Padded<T> pg(s, a.g, s.Tq, H, s.G), py(s, a.y, s.Tq, H, s.G);
    run_attention_bwd(a);
  });
}

// Calls `f` with the views' sequences, as many at a time as one launch holds.
// Views of the whole call, some of them null: q, k and others with a sequence to
// each first index; from `first_array` on contiguous ones of as many equal parts.
template <size_t N, class F>
void by_sequences(const nt_view *(&views)[N], size_t first_array, F &&f) {
  const nt_view *q = views[0], *k = views[1];
  const int64_t most = sequences_at_once(q, k), B = most ? q->shape[0] : 0;
  bool whole = most == 0 || B <= most;
  for (size_t i = 0; i < N && !whole; ++i) { // not of one batch: reported by the whole call
    const nt_view *v = views[i];
    if (v && (v->ndim < 1 || v->ndim > NT_MAX_DIMS ||
              (i < first_array ? v->shape[0] != B
                               : numel(v) % B != 0 || !is_contiguous(v))))
      whole = true;
  }
  if (whole)
    return f(views);
  for (int64_t b = 0; b < B; b += most) {
    const int64_t n = std::min(most, B - b);
    nt_view some[N];
    const nt_view *at[N];
    for (size_t i = 0; i < N; ++i) {
      at[i] = nullptr;
      if (views[i]) {
        some[i] = i < first_array ? sequences(views[i], b, n) : parts(views[i], B, b, n);
        at[i] = &some[i];
      }
    }
    f(at);
  }
}

} // namespace
} // namespace nt

using namespace nt;

extern "C" {

int nt_attention(const nt_view *q, const nt_view *k, const nt_view *v, const nt_view *lengths,
                 const nt_view *starts, int64_t start, int32_t causal, double scale,
                 const nt_view *y, const nt_view *lse) {
  return guard([&] {
    const nt_view *views[] = {q, k, v, lengths, starts, y, lse};
    by_sequences(views, 5, [&](const nt_view *const *x) {
      attention(x[0], x[1], x[2], x[3], x[4], start, causal, scale, x[5], x[6]);
    });
  });
}

int nt_attention_bwd(const nt_view *q, const nt_view *k, const nt_view *v,
                     const nt_view *lengths, const nt_view *starts, int64_t start,
                     int32_t causal, double scale, const nt_view *y, const nt_view *lse,
                     const nt_view *g, const nt_view *dq, const nt_view *dk,
                     const nt_view *dv) {
  return guard([&] {
    const nt_view *views[] = {q, k, v, lengths, starts, g, y, lse, dq, dk, dv};
    by_sequences(views, 6, [&](const nt_view *const *x) {
      attention_bwd(x[0], x[1], x[2], x[3], x[4], start, causal, scale, x[6], x[7], x[5], x[8],
                    x[9], x[10]);
    });
  });
}

} // extern "C"

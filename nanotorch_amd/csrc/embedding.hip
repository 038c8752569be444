// Rows of a table looked up by token, and the table's gradient:
//
//   y[i, :]  = scale * W[t_i, :]
//   dW[v, :] = scale * sum over the i with t_i = v of g[i, :]
//
// A token equal to `padding` gives a zero row and no gradient; one outside
// the table does too, and is reported at the next synchronisation (the
// library's deferred error).  Both passes move bytes and compute almost
// nothing: the lookup reads N rows and writes N rows, the gradient reads N
// rows and writes every row of dW once, zeros included (accumulating, it
// reads and writes only the rows that a token names).
#include "tokens.h"

#include <algorithm>

namespace nt {

constexpr int EMB_THREADS = 256;

// A vector of a row's columns.  The last one of a row whose length is no
// multiple of N starts earlier, so that it is whole, and its first `skip`
// elements belong to the vector before; a row shorter than N has one vector,
// moved element by element.  EVEN: D is a multiple of N.
template <class T, bool EVEN> struct RowPart {
  using RV = RowVec<T>;
  int col, skip = 0, width = RV::N; // width < N: elements of a short row

  __device__ __forceinline__ RowPart(uint32_t c, int D) {
    col = int(c) * RV::N;
    if (!EVEN) {
      skip = max(0, min(col, col + RV::N - D));
      col -= skip;
      width = min(RV::N, D - col);
    }
  }
  template <bool STREAM = false>
  __device__ __forceinline__ typename RV::V load(const T *row) const {
    if (EVEN || width == RV::N)
      return RV::template load<STREAM>(row + col);
    typename RV::V v = {};
    for (int j = 0; j < width; ++j)
      v[j] = row[col + j];
    return v;
  }
  template <bool ACC, bool STREAM = true>
  __device__ __forceinline__ void store(T *row, typename RV::V v) const {
    T *to = row + col;
    if (EVEN || (width == RV::N && skip == 0)) {
      RV::template store<STREAM>(to, ACC ? RV::load(to) + v : v);
    } else {
#pragma unroll
      for (int j = 0; j < RV::N; ++j)
        if (j >= skip && j < width)
          to[j] = ACC ? to[j] + v[j] : v[j];
    }
  }
};

// ---------------------------------------------------------------- lookup

// Row `t` of a table, or nothing where it has no row to give.
struct Rows {
  int64_t V, padding;
  int *err;

  __device__ __forceinline__ bool has(int64_t t) const {
    if (t < 0 || t >= V) {
      *err = NT_ERR_INDEX; // the deferred-error word (host memory)
      return false;
    }
    return t != padding;
  }
};

// A workgroup writes EMB_THREADS * EMB_LOOKUP adjacent vectors of the output,
// each work-item every EMB_THREADS-th of them, so that as many loads are in
// flight.  Rows of adjacent elements.  65536 rows of 2048 float32 (0.54 GB
// written, 0.16 GB of different rows read) take 131 us alone and 157
// behind a gradient that is still on its way to memory; with a branch around
// each load 181, with stores that stay in the cache 144.
constexpr int EMB_LOOKUP = 4;

template <class T, bool EVEN>
__global__ __launch_bounds__(EMB_THREADS) void embedding_kernel(
    const T *__restrict__ table, int64_t rs, Tokens tok, int64_t i0, Rows rows,
    T scale, T *__restrict__ out, uint32_t items, FastDivU32 vectors, int D) {
  using RV = RowVec<T>;
  const uint32_t first = blockIdx.x * (EMB_THREADS * EMB_LOOKUP) + threadIdx.x;
  typename RV::V v[EMB_LOOKUP];
  uint32_t row[EMB_LOOKUP];
  int64_t t[EMB_LOOKUP];
  bool has[EMB_LOOKUP];
#pragma unroll
  for (int k = 0; k < EMB_LOOKUP; ++k) {
    row[k] = vectors.div(min(first + k * EMB_THREADS, items - 1));
    t[k] = tok[i0 + row[k]];
  }
#pragma unroll
  for (int k = 0; k < EMB_LOOKUP; ++k) {
    const uint32_t item = min(first + k * EMB_THREADS, items - 1);
    has[k] = rows.has(t[k]);
    // row 0 in place of none, so that the loads need no branches
    v[k] = RowPart<T, EVEN>(item - row[k] * vectors.d, D).load(table + (has[k] ? t[k] : 0) * rs);
  }
#pragma unroll
  for (int k = 0; k < EMB_LOOKUP; ++k) {
    const uint32_t item = first + k * EMB_THREADS;
    if (item < items)
      RowPart<T, EVEN>(item - row[k] * vectors.d, D)
          .template store<false>(out + (i0 + row[k]) * D,
                                 has[k] ? v[k] * scale : typename RV::V{});
  }
}

// Any strides of the table: one element per work-item.
template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_strided_kernel(
    const T *__restrict__ table, int64_t rs, int64_t cs, Tokens tok, int64_t N,
    Rows rows, T scale, T *__restrict__ out, int64_t D) {
  const int64_t total = N * D, stride = int64_t(gridDim.x) * EMB_THREADS;
  for (int64_t e = int64_t(blockIdx.x) * EMB_THREADS + threadIdx.x; e < total;
       e += stride) {
    const int64_t i = e / D, c = e - i * D, t = tok[i];
    out[e] = rows.has(t) ? table[t * rs + c * cs] * scale : T(0);
  }
}

// ------------------------------------------------- gradient, few tokens

constexpr int EMB_SCAN = 256;           // tokens that one scan holds
constexpr int EMB_SEG = EMB_SCAN / 4;   // of them per wave
constexpr int EMB_FLIGHT = 8;           // rows of g in flight per wave

// N <= EMB_SCAN tokens, one launch.  A workgroup owns R rows of dW and 64
// vectors of columns.  Each wave lists the tokens of its quarter that name
// one of the rows, in order; then each wave sums and writes the rows
// wave, wave + 4, ...  Against the sorted form below (us, 1000 x 64, Zipf-like
// tokens): N = 64 7 and 13, N = 256 7.5 and 13.6, N = 1024 12 and 15; but one
// token throughout, which a single wave then sums: N = 256 18 and 12,
// N = 1024 67 and 13.
template <class T, bool ACC, bool EVEN>
__global__ __launch_bounds__(EMB_THREADS) void embedding_scan_kernel(
    const T *__restrict__ g, Tokens tok, int n, int64_t padding, T scale,
    T *__restrict__ dw, int64_t rs, int64_t V, int D, int R, int chunks,
    int *err) {
  using RV = RowVec<T>;
  __shared__ uint32_t list[4][EMB_SEG]; // row in the tile << 8 | token
  __shared__ int count[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t v0 = int64_t(blockIdx.x / chunks) * R;
  const uint32_t c = blockIdx.x % chunks * 64 + lane;
  {
    const int per = ((n + 3) / 4 + 63) / 64 * 64;
    const int beg = wave * per, end = min(n, beg + per);
    int have = 0;
    for (int b = beg; b < end; b += 64) {
      const int i = b + lane;
      int64_t t = -1;
      if (i < end) {
        t = tok[i];
        if ((t < 0 || t >= V) && blockIdx.x == 0)
          *err = NT_ERR_INDEX;
      }
      const bool mine = i < end && t >= v0 && t < v0 + R && t < V && t != padding;
      const uint64_t m = __ballot(mine);
      if (mine)
        list[wave][have + __popcll(m & ((uint64_t(1) << lane) - 1))] =
            uint32_t(t - v0) << 8 | uint32_t(i);
      have += __popcll(m);
    }
    if (lane == 0)
      count[wave] = have;
  }
  __syncthreads();
  const bool in = int64_t(c) * RV::N < D;
  const RowPart<T, EVEN> part(in ? c : 0, D);
  for (int r = wave; r < R && v0 + r < V; r += 4) {
    typename RV::V acc = {};
    bool any = false;
    for (int s = 0; s < 4; ++s) {
      const int have = count[s];
      for (int b = 0; b < have; b += 64) {
        const uint32_t e = b + lane < have ? list[s][b + lane] : ~0u;
        uint64_t m = __ballot(e != ~0u && int(e >> 8) == r);
        any |= m != 0;
        while (m) {
          typename RV::V v[EMB_FLIGHT];
#pragma unroll
          for (int k = 0; k < EMB_FLIGHT; ++k) {
            v[k] = typename RV::V{};
            if (m) {
              const int l = __ffsll((unsigned long long)m) - 1;
              m &= m - 1;
              const int i = int(__builtin_amdgcn_readlane(e, l)) & (EMB_SCAN - 1);
              v[k] = part.load(g + int64_t(i) * D);
            }
          }
#pragma unroll
          for (int k = 0; k < EMB_FLIGHT; ++k)
            acc += v[k];
        }
      }
    }
    if ((ACC && !any) || !in)
      continue;
    part.template store<ACC>(dw + (v0 + r) * rs, acc * scale);
  }
}

// ------------------------------------------------ gradient, many tokens
//
// The tokens are sorted (stably, so a row's terms stay in rising i): up to
// RANK_MOST by counting, more by a radix sort of (key, i) pairs, the key being
// the token, or V where there is no gradient.  The sorted pairs are cut into tiles of 8 or 32.  A work-item
// sums one vector of columns over one tile, run by run.  A run within a tile
// is written to dW; a run that goes on into the next tile leaves one partial
// sum per tile, which a last kernel joins in tile order.  So a token that
// fills a tenth of the batch is spread over the chip like any other.
//
// 65536 tokens into 128000 x 2048 float32: sort 27 us, sums 137 (0.54 GB read,
// 0.17 GB written), joins 15, zero rows 129 (0.89 GB, 6.9 TB/s).  8192 into
// 32000 x 1024: sort and zero rows 20 us, sums 13, joins 4.

constexpr int EMB_DIGIT = 9; // bits of a pass, at most
constexpr int EMB_BINS = 1 << EMB_DIGIT;
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WAVES = SORT_THREADS / WAVE;
constexpr int SORT_ROUNDS = 8; // pairs per lane
constexpr int SORT_MOST = SORT_THREADS * SORT_ROUNDS;

struct Pairs {
  uint32_t *key, *pos;
};

struct SortPlan {
  Tokens tok; // what the first pass reads
  Rows rows;
  uint32_t n, per; // pairs; of them per workgroup, at most SORT_MOST
  int groups, digit, passes;
  uint32_t *table;  // [groups][EMB_BINS] counts
  uint32_t *total;  // [EMB_BINS], or null: then table holds the counts of the groups before
  uint8_t *present; // [V], or null: 1 where a row has a gradient
  Pairs side[2];    // pass k writes side[k & 1]
};

__device__ __forceinline__ uint32_t key_of(const SortPlan &p, uint32_t i) {
  const int64_t t = p.tok[i];
  return p.rows.has(t) ? uint32_t(t) : uint32_t(p.rows.V);
}

// A workgroup's pairs, in registers: each wave takes a contiguous part,
// 64 adjacent pairs a round.
struct SortRegs {
  uint32_t key[SORT_ROUNDS], pos[SORT_ROUNDS];
  uint32_t beg, end; // of the wave

  __device__ __forceinline__ bool in(int r) const {
    return beg + r * WAVE + (threadIdx.x & 63) < end;
  }
  __device__ __forceinline__ void load(const SortPlan &p, int pass) {
    const uint32_t g0 = blockIdx.x * p.per, g1 = min(p.n, g0 + p.per);
    const uint32_t part = ((g1 - g0 + SORT_WAVES - 1) / SORT_WAVES + WAVE - 1) / WAVE * WAVE;
    beg = min(g1, g0 + (threadIdx.x >> 6) * part);
    end = min(g1, beg + part);
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r) {
      const uint32_t i = beg + r * WAVE + (threadIdx.x & 63);
      key[r] = pos[r] = 0;
      if (i < end) {
        if (pass == 0) {
          key[r] = key_of(p, i);
          pos[r] = i;
        } else {
          key[r] = p.side[(pass - 1) & 1].key[i];
          pos[r] = p.side[(pass - 1) & 1].pos[i];
        }
      }
    }
  }
};

struct SortShared {
  uint64_t pair[SORT_MOST];             // sorted by the pass's digit
  uint32_t count[SORT_WAVES][EMB_BINS]; // per wave: pairs of a digit, then their places
  uint32_t out[EMB_BINS];               // what to add to a place for the place among all
  uint32_t sums[SORT_WAVES];
};

// Exclusive sum over the workgroup's threads.
__device__ __forceinline__ uint32_t sum_before(uint32_t v, uint32_t (&sums)[SORT_WAVES]) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t up = v;
  for (int k = 1; k < WAVE; k <<= 1) {
    const uint32_t o = __shfl_up(up, k);
    up += lane >= k ? o : 0;
  }
  __syncthreads();
  if (lane == WAVE - 1)
    sums[wave] = up;
  __syncthreads();
  up -= v;
  for (int w = 0; w < wave; ++w)
    up += sums[w];
  return up;
}

// Sorts the workgroup's pairs by the pass's digit into s.pair.  Each wave
// goes through its rounds once: lanes of equal digit find each other by a
// ballot per bit, take their places in lane order behind the rounds before
// (`count`, per wave and digit), and the last of them moves the count on.
// The counts then become the places where each wave's pairs of a digit start;
// s.out comes from `table`, which has every workgroup's counts.
__device__ __forceinline__ void sort_pass(const SortPlan &p, int pass, const SortRegs &x,
                                          SortShared &s) {
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int shift = pass * p.digit, mask = (1 << p.digit) - 1;
  uint4 *const all = reinterpret_cast<uint4 *>(&s.count[0][0]);
  for (int d = tid; d < SORT_WAVES * EMB_BINS / 4; d += SORT_THREADS)
    all[d] = uint4{0, 0, 0, 0};
  __syncthreads();
  volatile uint32_t *const mine = s.count[wave];
  uint32_t rank[SORT_ROUNDS];
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r) {
    rank[r] = 0;
    if (x.beg + r * WAVE >= x.end)
      break;
    const bool in = x.in(r);
    const uint32_t digit = x.key[r] >> shift & mask;
    uint64_t same = __ballot(in);
#pragma unroll
    for (int b = 0; b < EMB_DIGIT; ++b) {
      const bool one = digit >> b & 1;
      const uint64_t m = __ballot(one);
      same &= one ? m : ~m;
    }
    if (in) {
      const uint32_t have = mine[digit];
      rank[r] = have + __popcll(same & ((uint64_t(1) << lane) - 1));
      __builtin_amdgcn_wave_barrier(); // every lane has read before one writes
      if (same >> lane == 1)
        mine[digit] = have + __popcll(same);
    }
    __builtin_amdgcn_wave_barrier();
  }
  // all workgroups' pairs of a digit, a digit per thread of the first EMB_BINS
  uint32_t total = 0, before = 0;
  if (tid < EMB_BINS) {
    if (p.total) {
      before = p.table[blockIdx.x * EMB_BINS + tid];
      total = p.total[tid];
    } else {
#pragma unroll 8
      for (int b = 0; b < p.groups; ++b) {
        const uint32_t c = p.table[b * EMB_BINS + tid];
        before += b < int(blockIdx.x) ? c : 0;
        total += c;
      }
    }
  }
  __syncthreads();
  uint32_t own = 0;
  if (tid < EMB_BINS) {
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w)
      own += s.count[w][tid];
  }
  const uint32_t first = sum_before(own, s.sums);
  before += sum_before(total, s.sums);
  if (tid < EMB_BINS) {
    uint32_t at = first;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w) {
      const uint32_t c = s.count[w][tid];
      s.count[w][tid] = at;
      at += c;
    }
    s.out[tid] = before - first;
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r)
    if (x.in(r))
      s.pair[s.count[wave][x.key[r] >> shift & mask] + rank[r]] =
          uint64_t(x.key[r]) << 32 | x.pos[r];
  __syncthreads();
}

// s.pair to where the pairs belong; neighbours of a digit stay neighbours.
__device__ __forceinline__ void sort_out(const SortPlan &p, int pass, SortShared &s) {
  const uint32_t n = min(p.per, p.n - blockIdx.x * p.per);
  const Pairs to = p.side[pass & 1];
  for (uint32_t e = threadIdx.x; e < n; e += SORT_THREADS) {
    const uint64_t v = s.pair[e];
    const uint32_t key = uint32_t(v >> 32);
    const uint32_t at = e + s.out[key >> (pass * p.digit) & ((1 << p.digit) - 1)];
    to.key[at] = key;
    to.pos[at] = uint32_t(v);
  }
}

__device__ __forceinline__ void clear_present(const SortPlan &p) {
  if (p.present) { // allocations are multiples of 512 bytes
    uint4 *const at = reinterpret_cast<uint4 *>(p.present);
    for (uint32_t v = blockIdx.x * SORT_THREADS + threadIdx.x; v < (p.rows.V + 15) / 16;
         v += gridDim.x * SORT_THREADS)
      at[v] = uint4{0, 0, 0, 0};
  }
}

__device__ __forceinline__ void set_present(const SortPlan &p, const SortRegs &x) {
  if (p.present)
#pragma unroll
    for (int r = 0; r < SORT_ROUNDS; ++r)
      if (x.in(r) && x.key[r] < p.rows.V)
        p.present[x.key[r]] = 1;
}

// One pass over many workgroups: the counts, then the places.
__global__ __launch_bounds__(SORT_THREADS) void embedding_count_kernel(SortPlan p, int pass) {
  __shared__ uint32_t bin[EMB_BINS];
  for (int d = threadIdx.x; d < EMB_BINS; d += SORT_THREADS)
    bin[d] = 0;
  if (pass == 0)
    clear_present(p);
  SortRegs x;
  x.load(p, pass);
  __syncthreads();
#pragma unroll
  for (int r = 0; r < SORT_ROUNDS; ++r)
    if (x.in(r))
      atomicAdd(&bin[x.key[r] >> (pass * p.digit) & ((1 << p.digit) - 1)], 1u);
  __syncthreads();
  for (int d = threadIdx.x; d < EMB_BINS; d += SORT_THREADS)
    p.table[blockIdx.x * EMB_BINS + d] = bin[d];
}

// Where the groups are many, each count becomes the sum of those of the groups
// before.  A workgroup takes 64 digits, a wave of it a part of the groups.  By
// this and by each workgroup of the places adding up all counts (us, 1000 x
// 16): 1048576 tokens (128 groups) 90 and 84, 4194304 242 and 304, 16777216
// 935 and 2304.
constexpr int SORT_ADDED = 256; // groups up to which they are added up

__global__ __launch_bounds__(SORT_THREADS) void embedding_offsets_kernel(SortPlan p) {
  __shared__ uint32_t sums[SORT_WAVES][WAVE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int digit = blockIdx.x * WAVE + lane;
  const int per = (p.groups + SORT_WAVES - 1) / SORT_WAVES;
  const int beg = min(p.groups, wave * per), end = min(p.groups, beg + per);
  uint32_t *const at = p.table + digit;
  uint32_t sum = 0;
#pragma unroll 16
  for (int b = beg; b < end; ++b)
    sum += at[int64_t(b) * EMB_BINS];
  sums[wave][lane] = sum;
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w)
    before += sums[w][lane];
  if (wave == SORT_WAVES - 1)
    p.total[digit] = before + sum;
#pragma unroll 16
  for (int b = beg; b < end; ++b) {
    const uint32_t c = at[int64_t(b) * EMB_BINS];
    at[int64_t(b) * EMB_BINS] = before;
    before += c;
  }
}

__global__ __launch_bounds__(SORT_THREADS) void embedding_place_kernel(SortPlan p, int pass) {
  __shared__ SortShared s;
  SortRegs x;
  x.load(p, pass);
  if (pass == 0)
    set_present(p, x);
  sort_pass(p, pass, x, s);
  sort_out(p, pass, s);
}

struct SumPlan {
  const uint32_t *key, *pos;
  uint32_t n, V;
  FastDivU32 vectors; // columns in vectors
  int D;
  int64_t rs; // of dW
  uint32_t tile; // pairs of a tile
};

// Partial sums: two vectors for each tile and vector of columns, the first
// for a run that comes from the tile before, the second for one that begins
// here and goes on.
template <class T>
__device__ __forceinline__ T *partial(const SumPlan &p, T *part, uint32_t tile, int which,
                                      uint32_t c) {
  return part + ((int64_t(tile) * 2 + which) * p.vectors.d + c) * RowVec<T>::N;
}

// One tile and vector of columns per work-item.
template <class T, bool ACC, bool EVEN>
__global__ __launch_bounds__(EMB_THREADS) void embedding_sum_kernel(
    const T *__restrict__ g, SumPlan p, T scale, T *__restrict__ dw,
    T *__restrict__ part, uint32_t tile0, uint32_t items) {
  using RV = RowVec<T>;
  const uint32_t item = blockIdx.x * EMB_THREADS + threadIdx.x;
  if (item >= items)
    return;
  uint32_t tile = p.vectors.div(item);
  const uint32_t c = item - tile * p.vectors.d;
  tile += tile0;
  const uint32_t beg = tile * p.tile, end = min(p.n, beg + p.tile);
  const RowPart<T, EVEN> part_of(c, p.D);
  uint32_t key = p.key[beg];
  bool carried = beg > 0 && p.key[beg - 1] == key;
  typename RV::V acc = {};
  for (uint32_t b = beg; b < end; b += EMB_FLIGHT) {
    typename RV::V v[EMB_FLIGHT];
    uint32_t k[EMB_FLIGHT], pos[EMB_FLIGHT];
#pragma unroll
    for (int j = 0; j < EMB_FLIGHT; ++j) {
      k[j] = p.key[min(b + j, end - 1)];
      pos[j] = p.pos[min(b + j, end - 1)];
    }
#pragma unroll
    for (int j = 0; j < EMB_FLIGHT; ++j)
      v[j] = part_of.template load<true>(g + int64_t(pos[j]) * p.D);
#pragma unroll
    for (int j = 0; j < EMB_FLIGHT; ++j) {
      if (b + j >= end)
        break;
      if (k[j] != key) {
        if (carried)
          RV::store(partial(p, part, tile, 0, c), acc);
        else
          part_of.template store<ACC>(dw + key * p.rs, acc * scale); // keys rise: not yet V
        carried = false;
        key = k[j];
        acc = typename RV::V{};
      }
      acc += v[j];
    }
  }
  if (key >= p.V)
    return;
  if (carried)
    RV::store(partial(p, part, tile, 0, c), acc);
  else if (end < p.n && p.key[end] == key)
    RV::store(partial(p, part, tile, 1, c), acc);
  else
    part_of.template store<ACC>(dw + key * p.rs, acc * scale);
}

// Zeros into the rows that no token names.
constexpr int EMB_FILL = 4; // vectors per work-item

template <class T, bool EVEN>
__global__ __launch_bounds__(EMB_THREADS) void embedding_fill_kernel(
    SumPlan p, T *__restrict__ dw, const uint8_t *present, uint32_t row0, uint32_t items) {
  const uint32_t first = blockIdx.x * (EMB_THREADS * EMB_FILL) + threadIdx.x;
#pragma unroll
  for (int k = 0; k < EMB_FILL; ++k) {
    const uint32_t item = first + k * EMB_THREADS;
    if (item >= items)
      return;
    const uint32_t row = p.vectors.div(item);
    if (!present[row0 + row])
      RowPart<T, EVEN>(item - row * p.vectors.d, p.D)
          .template store<false, false>(dw + (row0 + row) * p.rs, typename RowVec<T>::V{});
  }
}

// Up to RANK_MOST tokens are sorted in one launch: a workgroup takes 64 of
// them, one per lane, and each of its waves counts, in its part of all
// tokens, those that come before (smaller ones, and equal ones of smaller i).
// The further workgroups write the zero rows meanwhile: each looks which of
// its rows the tokens name.  n^2 comparisons over the chip: 9000 tokens into
// 1000 x 64 take 27 us in all, by the radix sort 36; at 16384 both take 39 and
// 37, into 32000 x 1024 both 65.
constexpr int RANK_MOST = 16384;
constexpr int RANK_ROWS = 1024; // rows of a filling workgroup, at most

template <class T, bool EVEN>
__global__ __launch_bounds__(SORT_THREADS) void embedding_rank_kernel(
    SortPlan p, uint32_t ranking, uint32_t R, FastDivU32 vectors, int D, int64_t rs,
    T *__restrict__ dw) {
  __shared__ __align__(16) uint32_t key[RANK_MOST];
  __shared__ uint32_t part[SORT_WAVES][WAVE];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  if (blockIdx.x >= ranking) {
    const uint32_t v0 = (blockIdx.x - ranking) * R, rows = min(R, uint32_t(p.rows.V) - v0);
    for (uint32_t v = tid; v < rows; v += SORT_THREADS)
      key[v] = 0;
    __syncthreads();
    for (uint32_t i = tid; i < p.n; i += SORT_THREADS) {
      const int64_t t = p.tok[i];
      if (t >= v0 && t < int64_t(v0) + rows && t != p.rows.padding)
        key[t - v0] = 1;
    }
    __syncthreads();
    if (vectors.d >= WAVE) { // a row per wave
      for (uint32_t row = wave; row < rows; row += SORT_WAVES)
        if (!key[row])
          for (uint32_t c = lane; c < vectors.d; c += WAVE)
            RowPart<T, EVEN>(c, D).template store<false, false>(dw + (v0 + row) * rs,
                                                                typename RowVec<T>::V{});
      return;
    }
    const uint32_t items = rows * vectors.d;
    for (uint32_t e = tid; e < items; e += SORT_THREADS) {
      const uint32_t row = vectors.div(e);
      if (!key[row])
        RowPart<T, EVEN>(e - row * vectors.d, D)
            .template store<false, false>(dw + (v0 + row) * rs, typename RowVec<T>::V{});
    }
    return;
  }
  const uint32_t padded = (p.n + 63) / 64 * 64;
  for (uint32_t i = tid; i < padded; i += SORT_THREADS)
    key[i] = i < p.n ? key_of(p, i) : ~0u; // past the end: before nothing
  __syncthreads();
  const uint32_t i0 = blockIdx.x * WAVE, i = i0 + lane;
  const uint32_t mine = key[i];
  const uint32_t per = (padded / WAVE + SORT_WAVES - 1) / SORT_WAVES * WAVE;
  const uint32_t beg = min(padded, wave * per), end = min(padded, beg + per);
  uint32_t n = 0;
  const auto count = [&](uint32_t from, uint32_t to, uint32_t below) {
    for (uint32_t j = from; j < to; j += 16) {
      uint4 k[4];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        k[q] = reinterpret_cast<const uint4 *>(key + j)[q];
#pragma unroll
      for (int q = 0; q < 4; ++q)
        n += (k[q].x < below) + (k[q].y < below) + (k[q].z < below) + (k[q].w < below);
    }
  };
  count(beg, min(end, i0), mine + 1);
  if (i0 >= beg && i0 < end)
    for (int j = 0; j < WAVE; ++j)
      n += key[i0 + j] < mine + (j < lane);
  count(max(beg, i0 + WAVE), end, mine);
  part[wave][lane] = n;
  __syncthreads();
  if (wave == 0 && i < p.n) {
    uint32_t at = 0;
#pragma unroll
    for (int w = 0; w < SORT_WAVES; ++w)
      at += part[w][lane];
    p.side[0].key[at] = mine;
    p.side[0].pos[at] = i;
  }
}

// Runs over several tiles, by the tile that they begin in.  A run of up to
// EMB_JOIN tiles more is joined by one work-item per vector of columns.  The
// further workgroups take the longer ones: each looks through 64 tiles, and
// its waves add every fourth group of EMB_JOIN tiles of a run and then each
// other's sums, in their order.
constexpr int EMB_JOIN = 16;

// Whether a run begins in the tile and goes on; its key.
__device__ __forceinline__ bool run_begins(const SumPlan &p, uint32_t tile, uint32_t &key) {
  const uint32_t beg = tile * p.tile, end = beg + p.tile;
  if (end >= p.n)
    return false;
  key = p.key[end - 1];
  return key < p.V && p.key[end] == key && !(beg > 0 && p.key[beg - 1] == key);
}

// Adds the sums that the EMB_JOIN tiles from `tile` on carry of the key's run.
template <class T>
__device__ __forceinline__ typename RowVec<T>::V
add_group(const SumPlan &p, T *part, uint32_t tile, uint32_t key, uint32_t c,
          typename RowVec<T>::V acc) {
  using RV = RowVec<T>;
  typename RV::V v[EMB_JOIN];
  bool same[EMB_JOIN];
#pragma unroll
  for (int j = 0; j < EMB_JOIN; ++j) {
    const uint32_t b = (tile + j) * p.tile;
    same[j] = (b < p.n) & (p.key[min(b, p.n - 1)] == key);
  }
#pragma unroll
  for (int j = 0; j < EMB_JOIN; ++j)
    if (same[j])
      v[j] = RV::load(partial(p, part, tile + j, 0, c));
#pragma unroll
  for (int j = 0; j < EMB_JOIN; ++j)
    acc = same[j] ? acc + v[j] : acc;
  return acc;
}

template <class T, bool ACC, bool EVEN>
__global__ __launch_bounds__(EMB_THREADS) void embedding_join_kernel(
    SumPlan p, T scale, T *__restrict__ dw, T *part, uint32_t tile0, uint32_t tiles,
    uint32_t joining, uint32_t chunks) {
  using RV = RowVec<T>;
  if (blockIdx.x < joining) {
    const uint32_t item = blockIdx.x * EMB_THREADS + threadIdx.x;
    const uint32_t tile = p.vectors.div(item), c = item - tile * p.vectors.d;
    uint32_t key;
    if (tile >= tiles || !run_begins(p, tile0 + tile, key))
      return;
    const uint32_t b = (tile0 + tile + 1) * p.tile;
    if (b + EMB_JOIN * p.tile < p.n && p.key[b + EMB_JOIN * p.tile] == key)
      return; // a longer one
    const typename RV::V acc = RV::load(partial(p, part, tile0 + tile, 1, c));
    RowPart<T, EVEN>(c, p.D).template store<ACC>(
        dw + key * p.rs, add_group(p, part, tile0 + tile + 1, key, c, acc) * scale);
    return;
  }
  constexpr int WAVES = EMB_THREADS / WAVE;
  __shared__ typename RV::V sums[WAVES][WAVE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint32_t block = blockIdx.x - joining, t64 = block / chunks * WAVE;
  const uint32_t c = block % chunks * WAVE + lane, at_c = min(c, p.vectors.d - 1);
  uint32_t mine = 0;
  const uint32_t next = (tile0 + t64 + lane + 1) * p.tile;
  const bool longer = t64 + lane < tiles && run_begins(p, tile0 + t64 + lane, mine) &&
                      next + EMB_JOIN * p.tile < p.n && p.key[next + EMB_JOIN * p.tile] == mine;
  uint64_t m = __ballot(longer); // the same in every wave
  while (m) {
    const int l = __ffsll((unsigned long long)m) - 1;
    m &= m - 1;
    const uint32_t tile = tile0 + t64 + l, key = __builtin_amdgcn_readlane(mine, l);
    typename RV::V acc = {};
    if (wave == 0)
      acc = RV::load(partial(p, part, tile, 1, at_c));
    for (uint32_t t = tile + 1 + wave * EMB_JOIN; t * p.tile < p.n && p.key[t * p.tile] == key;
         t += WAVES * EMB_JOIN)
      acc = add_group(p, part, t, key, at_c, acc);
    __syncthreads(); // the sums of the run before have been read
    sums[wave][lane] = acc;
    __syncthreads();
    if (wave == 0 && c < p.vectors.d) {
#pragma unroll
      for (int w = 1; w < WAVES; ++w)
        acc += sums[w][lane];
      RowPart<T, EVEN>(c, p.D).template store<ACC>(dw + key * p.rs, acc * scale);
    }
  }
}

namespace {

// Calls f(first row, rows) over `rows` rows of `vectors` work-items each, in
// launches of less than 2^30 work-items.
template <class F> void in_launches(int64_t rows, int64_t vectors, F &&f) {
  const int64_t most = std::max<int64_t>(1, ((int64_t(1) << 30) - 1) / vectors);
  for (int64_t r = 0; r < rows; r += most)
    f(r, std::min(most, rows - r));
}

template <class T> uint32_t row_vectors(int64_t D) {
  return uint32_t((D + RowVec<T>::N - 1) / RowVec<T>::N);
}

unsigned blocks_for(int64_t items, int per) { return unsigned((items + per - 1) / per); }

template <class T, bool EVEN>
void run_embedding(const nt_view *table, const Tokens &tok, int64_t N,
                   int64_t padding, double scale, const nt_view *out) {
  const int64_t V = table->shape[0], D = table->shape[1];
  if (N == 0 || D == 0)
    return;
  const Rows rows{V, padding, deferred_error_word()};
  const T *from = typed_ptr<const T>(table);
  T *to = typed_ptr<T>(out);
  if (V == 0 || (D > 1 && table->strides[1] != 1)) {
    const int64_t blocks = std::min<int64_t>((N * D + EMB_THREADS - 1) / EMB_THREADS,
                                             int64_t(1) << 22);
    embedding_strided_kernel<T><<<dim3(unsigned(blocks)), EMB_THREADS, 0, stream()>>>(
        from, table->strides[0], table->strides[1], tok, N, rows, T(scale), to, D);
    NT_LAUNCH_CHECK();
    return;
  }
  const uint32_t vectors = row_vectors<T>(D);
  in_launches(N, vectors, [&](int64_t i0, int64_t n) {
    const int64_t items = n * vectors;
    embedding_kernel<T, EVEN>
        <<<dim3(blocks_for(items, EMB_THREADS * EMB_LOOKUP)), EMB_THREADS, 0, stream()>>>(
            from, table->strides[0], tok, i0, rows, T(scale), to, uint32_t(items),
            FastDivU32(vectors), int(D));
    NT_LAUNCH_CHECK();
  });
}

template <class T, bool ACC, bool EVEN>
void run_scan(const nt_view *g, const Tokens &tok, int64_t padding, T scale,
              const nt_view *dw) {
  const int64_t D = g->shape[1], V = dw->shape[0];
  const int64_t chunks = (D + 64 * RowVec<T>::N - 1) / (64 * RowVec<T>::N);
  // few rows per workgroup while that fills the chip; a row takes 20 bits of
  // a list entry
  int R = 4;
  while (R < 1 << 20 && (V + R - 1) / R * chunks > (R < 64 ? 2048 : int64_t(1) << 22))
    R *= 2;
  const int64_t blocks = (V + R - 1) / R * chunks;
  if (blocks >= int64_t(1) << 24)
    fail(NT_ERR_VALUE, "embedding_bwd: table too large");
  embedding_scan_kernel<T, ACC, EVEN><<<dim3(unsigned(blocks)), EMB_THREADS, 0, stream()>>>(
      typed_ptr<const T>(g), tok, int(g->shape[0]), padding, scale, typed_ptr<T>(dw),
      dw->strides[0], V, int(D), R, int(chunks), deferred_error_word());
  NT_LAUNCH_CHECK();
}

template <class T, bool ACC, bool EVEN>
void run_sorted(const nt_view *g, const Tokens &tok, int64_t padding, T scale,
                const nt_view *dw) {
  const int64_t N = g->shape[0], D = g->shape[1], V = dw->shape[0];
  hipStream_t s = stream();
  int bits = 1;
  while (V >> bits)
    ++bits; // keys 0 .. V
  SortPlan p{};
  p.tok = tok;
  p.rows = Rows{V, padding, deferred_error_word()};
  p.n = uint32_t(N);
  p.passes = (bits + EMB_DIGIT - 1) / EMB_DIGIT;
  p.digit = (bits + p.passes - 1) / p.passes;
  const uint32_t vectors = row_vectors<T>(D);
  T *const to = typed_ptr<T>(dw);
  // a filling workgroup's rows: 512 workgroups, but 2^12 to 2^15 vectors each,
  // which take longer to write than the tokens to read, and at most RANK_ROWS
  // rows.  Those bound tall narrow tables, whose many workgroups each read all
  // tokens (us by ranks and by the radix sort: 1000000 x 4, 1024 tokens 14 and
  // 45, 16384 54 and 64; 10000000 x 4, 1024 36 and 122, 9000 96 and 103, but
  // 16384 145 and 107).
  const int64_t fill = std::clamp<int64_t>((V * vectors + 511) / 512, 1 << 12, 1 << 15);
  const uint32_t R = uint32_t(std::clamp<int64_t>(fill / vectors, 1, RANK_ROWS));
  const bool ranked = N <= RANK_MOST && (ACC || (V + R - 1) / R < int64_t(1) << 20);
  DeviceScratch pairs(size_t(N) * (ranked ? 8 : 16));
  uint32_t *const base = pairs.get<uint32_t>();
  p.side[0] = {base, base + N};
  if (!ranked)
    p.side[1] = {base + 2 * N, base + 3 * N};
  // up to 64 workgroups of at least 2048 pairs; more once those are full
  const int64_t per = std::clamp<int64_t>((N + 63) / 64, 2048, SORT_MOST);
  p.per = uint32_t((per + SORT_THREADS - 1) / SORT_THREADS * SORT_THREADS);
  p.groups = int((N + p.per - 1) / p.per);
  const bool added = p.groups <= SORT_ADDED;
  DeviceScratch table(ranked ? 0 : size_t(p.groups + !added) * EMB_BINS * 4),
      present(ACC || ranked ? 0 : size_t(V));
  p.table = table.get<uint32_t>();
  p.total = added ? nullptr : p.table + int64_t(p.groups) * EMB_BINS;
  p.present = present.get<uint8_t>();
  if (ranked) {
    p.passes = 1;
    const uint32_t ranking = uint32_t((N + WAVE - 1) / WAVE);
    const uint32_t filling = ACC ? 0 : uint32_t((V + R - 1) / R);
    embedding_rank_kernel<T, EVEN><<<dim3(ranking + filling), SORT_THREADS, 0, s>>>(
        p, ranking, R, FastDivU32(vectors), int(D), dw->strides[0], to);
    NT_LAUNCH_CHECK();
  } else {
    for (int k = 0; k < p.passes; ++k) {
      embedding_count_kernel<<<dim3(unsigned(p.groups)), SORT_THREADS, 0, s>>>(p, k);
      NT_LAUNCH_CHECK();
      if (!added) {
        embedding_offsets_kernel<<<dim3(EMB_BINS / WAVE), SORT_THREADS, 0, s>>>(p);
        NT_LAUNCH_CHECK();
      }
      embedding_place_kernel<<<dim3(unsigned(p.groups)), SORT_THREADS, 0, s>>>(p, k);
      NT_LAUNCH_CHECK();
    }
  }
  // Few tokens: small tiles, since the chip is not full and a tile's loads
  // follow each other (us for 8 and 32 a tile, Zipf-like tokens: 50000 x 129,
  // N = 1500 16 and 25, N = 4000 22 and 28; 1000 x 64, N = 4000 18.5 and
  // 18.7, N = 8192 27 and 25).  One token throughout, whose sums the join
  // adds up, takes longer (N = 4000 28 and 19; N = 16384 91 and 47).
  const uint32_t tile = N <= 4096 ? 8 : 32;
  const int64_t tiles = (N + tile - 1) / tile;
  const Pairs &sorted = p.side[(p.passes - 1) & 1];
  const SumPlan q{sorted.key, sorted.pos, p.n, uint32_t(V), FastDivU32(vectors), int(D),
                  dw->strides[0], tile};
  if (!ACC && !ranked)
    in_launches(V, vectors, [&](int64_t r0, int64_t n) {
      embedding_fill_kernel<T, EVEN>
          <<<dim3(blocks_for(n * vectors, EMB_THREADS * EMB_FILL)), EMB_THREADS, 0, s>>>(
              q, to, p.present, uint32_t(r0), uint32_t(n * vectors));
      NT_LAUNCH_CHECK();
    });
  DeviceScratch part(size_t(2 * tiles * vectors) * 16);
  in_launches(tiles, vectors, [&](int64_t t0, int64_t n) {
    embedding_sum_kernel<T, ACC, EVEN>
        <<<dim3(blocks_for(n * vectors, EMB_THREADS)), EMB_THREADS, 0, s>>>(
            typed_ptr<const T>(g), q, scale, to, part.get<T>(), uint32_t(t0),
            uint32_t(n * vectors));
    NT_LAUNCH_CHECK();
  });
  const uint32_t chunks = (vectors + WAVE - 1) / WAVE;
  in_launches(tiles, vectors, [&](int64_t t0, int64_t n) {
    const unsigned joining = blocks_for(n * vectors, EMB_THREADS);
    const unsigned longer = unsigned((n + WAVE - 1) / WAVE * chunks);
    embedding_join_kernel<T, ACC, EVEN><<<dim3(joining + longer), EMB_THREADS, 0, s>>>(
        q, scale, to, part.get<T>(), uint32_t(t0), uint32_t(n), joining, chunks);
    NT_LAUNCH_CHECK();
  });
}

template <class T, bool ACC, bool EVEN>
void run_embedding_bwd(const nt_view *g, const Tokens &tok, int64_t padding, T scale,
                       const nt_view *dw) {
  if (dw->shape[0] == 0 || g->shape[1] == 0)
    return;
  if (g->shape[0] <= EMB_SCAN)
    run_scan<T, ACC, EVEN>(g, tok, padding, scale, dw);
  else
    run_sorted<T, ACC, EVEN>(g, tok, padding, scale, dw);
}

// f.operator()<flag>() for a flag known at run time.
template <class F> void with_flag(bool flag, F &&f) {
  flag ? f.template operator()<true>() : f.template operator()<false>();
}

template <class T> bool even_rows(int64_t D) { return D % RowVec<T>::N == 0; }

void check_size(int64_t N, int64_t V, int64_t D, const char *fname) {
  const int64_t most = int64_t(1) << 30;
  if (N >= most || V >= most || D >= most)
    fail(NT_ERR_VALUE, std::string(fname) +
                           ": tokens, rows and columns must be fewer than 2^30 each");
}

} // namespace
} // namespace nt

using namespace nt;

extern "C" {

int nt_embedding(const nt_view *table, const nt_view *tokens, double scale,
                 int64_t padding, const nt_view *out) {
  return guard([&] {
    check_view(table, "embedding");
    check_view(out, "embedding");
    const Tokens tok = token_view(tokens, "embedding");
    require_same_dtype(table, out, "embedding");
    if (table->ndim != 2 || out->ndim != 2 || out->shape[0] != tokens->shape[0] ||
        out->shape[1] != table->shape[1])
      fail(NT_ERR_RUNTIME, "embedding: expected [V, D], [N] and [N, D]");
    if (!is_contiguous(out))
      fail(NT_ERR_RUNTIME, "embedding: out must be contiguous");
    check_size(tokens->shape[0], table->shape[0], table->shape[1], "embedding");
    dispatch_float(table->dtype, [&]<class T>() {
      with_flag(even_rows<T>(table->shape[1]), [&]<bool EVEN>() {
        run_embedding<T, EVEN>(table, tok, tokens->shape[0], padding, scale, out);
      });
    });
  });
}

int nt_embedding_bwd(const nt_view *g, const nt_view *tokens, double scale,
                     int64_t padding, const nt_view *dtable, int32_t accumulate) {
  return guard([&] {
    check_view(g, "embedding_bwd");
    check_view(dtable, "embedding_bwd");
    const Tokens tok = token_view(tokens, "embedding_bwd");
    require_same_dtype(g, dtable, "embedding_bwd");
    if (g->ndim != 2 || dtable->ndim != 2 || g->shape[0] != tokens->shape[0] ||
        g->shape[1] != dtable->shape[1])
      fail(NT_ERR_RUNTIME, "embedding_bwd: expected [N, D], [N] and [V, D]");
    if (!is_contiguous(g) || (dtable->shape[1] > 1 && dtable->strides[1] != 1))
      fail(NT_ERR_RUNTIME, "embedding_bwd: g must be contiguous, and so must be "
                           "each row of the table's gradient");
    check_size(g->shape[0], dtable->shape[0], g->shape[1], "embedding_bwd");
    dispatch_float(g->dtype, [&]<class T>() {
      with_flag(accumulate != 0, [&]<bool ACC>() {
        with_flag(even_rows<T>(g->shape[1]), [&]<bool EVEN>() {
          run_embedding_bwd<T, ACC, EVEN>(g, tok, padding, T(scale), dtable);
        });
      });
    });
  });
}

} // extern "C"

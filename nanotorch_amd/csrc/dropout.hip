// Dropout whose mask is a function of the element's index, never stored:
//
//   y_i = x_i * 1/(1-p)  where r_i >= T, else 0,   T = round(p * 2^32)
//
// r_i is word i mod 4 of Philox4x32-10 under the 64-bit key `seed` at the
// 128-bit counter (i div 4, offset); i is the row-major index, so a view and
// its copy lose the same elements, and the backward pass is the same call on
// the gradient.  Philox: J. Salmon, M. Moraes, R. Dror, D. Shaw, "Parallel
// random numbers: as easy as 1, 2, 3", SC 2011.  A dropped element is 0
// whatever x holds there (infinities and NaN included).
#include "ew_engine.h"
#include "tokens.h"

namespace nt {

struct DropoutPlan {
  uint32_t threshold; // keeps words that are no smaller
  uint32_t none;      // p = 1: keeps nothing
  uint64_t seed, offset;
  double scale;

  __device__ __forceinline__ bool keeps(uint32_t w) const {
    return w >= threshold && !none;
  }
};

// The four words of the counter (group, offset).
__device__ __forceinline__ void philox(uint64_t group, const DropoutPlan &p,
                                       uint32_t (&w)[4]) {
  uint32_t c0 = uint32_t(group), c1 = uint32_t(group >> 32);
  uint32_t c2 = uint32_t(p.offset), c3 = uint32_t(p.offset >> 32);
  uint32_t k0 = uint32_t(p.seed), k1 = uint32_t(p.seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t a = uint64_t(c0) * 0xD2511F53u;
    const uint64_t b = uint64_t(c2) * 0xCD9E8D57u;
    c0 = uint32_t(b >> 32) ^ c1 ^ k0;
    c1 = uint32_t(b);
    c2 = uint32_t(a >> 32) ^ c3 ^ k1;
    c3 = uint32_t(a);
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0, w[1] = c1, w[2] = c2, w[3] = c3;
}

constexpr int DROP_THREADS = 256;

// A counter's four elements, 16 bytes at a time.
template <class T> struct Four {
  using RV = RowVec<T>;
  static constexpr int PARTS = 4 / RV::N;
  typename RV::V v[PARTS];

  __device__ __forceinline__ T get(int j) const { return v[j / RV::N][j % RV::N]; }
  __device__ __forceinline__ void set(int j, T x) { v[j / RV::N][j % RV::N] = x; }
  template <bool STREAM> __device__ __forceinline__ void load(const T *p) {
#pragma unroll
    for (int k = 0; k < PARTS; ++k)
      v[k] = RV::template load<STREAM>(p + k * RV::N);
  }
  template <bool STREAM> __device__ __forceinline__ void store(T *p) const {
#pragma unroll
    for (int k = 0; k < PARTS; ++k)
      RV::template store<STREAM>(p + k * RV::N, v[k]);
  }
};

// Contiguous operands: 16 bytes per work-item (two work-items share a counter
// in float64, each drawing it); the last, partial vector is taken element by
// element.  Bound by memory: 8192 x 4096 float32 takes 42 us (6.4 TB/s), with
// two or four vectors per work-item no less.
template <class T, bool ACC>
__global__ __launch_bounds__(DROP_THREADS) void dropout_flat_kernel(
    const T *__restrict__ x, T *__restrict__ y, int64_t n, int64_t vec0, DropoutPlan p) {
  using RV = RowVec<T>;
  constexpr int N = RV::N;
  const int64_t vec = vec0 + int64_t(blockIdx.x) * DROP_THREADS + threadIdx.x, i = N * vec;
  if (i >= n)
    return;
  const bool whole = i + N <= n;
  typename RV::V v = {}, old = {};
  if (whole) {
    v = RV::template load<true>(x + i);
    if (ACC)
      old = RV::template load<true>(y + i);
  } else {
#pragma unroll
    for (int j = 0; j < N - 1; ++j) {
      const int64_t at = min(i + j, n - 1);
      v[j] = x[at];
      if (ACC)
        old[j] = y[at];
    }
  }
  uint32_t w[4];
  philox(uint64_t(i) >> 2, p, w);
  if constexpr (N == 2) { // of an odd vector, the counter's words 2 and 3
    w[0] = vec & 1 ? w[2] : w[0];
    w[1] = vec & 1 ? w[3] : w[1];
  }
  const T scale = T(p.scale);
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const T r = p.keeps(w[j]) ? v[j] * scale : T(0);
    v[j] = ACC ? old[j] + r : r;
  }
  if (whole) {
    RV::template store<true>(y + i, v);
  } else {
#pragma unroll
    for (int j = 0; j < N - 1; ++j)
      if (i + j < n)
        y[i + j] = v[j];
  }
}

// x [R, C] stored by columns (adjacent elements along R), y by rows: tiles
// of 64 x 64 through LDS.  Reading, a wave takes a column's 64 elements;
// writing, a work-item takes a counter's four elements of a row, of which
// those at the tile's edge may belong to the next tile (C need not be a
// multiple of 4).
constexpr int DROP_TILE = 64;

template <class T, bool ACC>
__global__ __launch_bounds__(DROP_THREADS) void dropout_tile_kernel(
    const T *__restrict__ x, int64_t sx, T *__restrict__ y, int64_t sy, int64_t R, int64_t C,
    int64_t tiles_c, DropoutPlan p) {
  __shared__ T tile[DROP_TILE][DROP_TILE + 1];
  const int64_t r0 = blockIdx.x / tiles_c * DROP_TILE, c0 = blockIdx.x % tiles_c * DROP_TILE;
  const int rows = int(min(int64_t(DROP_TILE), R - r0)), cols = int(min(int64_t(DROP_TILE), C - c0));
  {
    const int r = threadIdx.x & 63, first = threadIdx.x >> 6;
    T v[DROP_TILE / 4];
#pragma unroll
    for (int k = 0; k < DROP_TILE / 4; ++k) {
      const int c = first + 4 * k;
      v[k] = x[(c0 + min(c, cols - 1)) * sx + r0 + min(r, rows - 1)];
    }
#pragma unroll
    for (int k = 0; k < DROP_TILE / 4; ++k)
      tile[r][first + 4 * k] = v[k];
  }
  __syncthreads();
  constexpr int PER = DROP_TILE / 4 + 1; // counters that a row of the tile may touch
  const T scale = T(p.scale);
  for (int q = threadIdx.x; q < DROP_TILE * PER; q += DROP_THREADS) {
    const int r = q / PER;
    const int64_t i0 = (r0 + r) * C + c0; // the tile's first element of the row
    const int64_t g = (i0 >> 2) + q % PER;
    const int c = int(4 * g - i0); // of the counter's first element, from c0
    if (r >= rows || c >= cols)
      continue;
    uint32_t w[4];
    philox(uint64_t(g), p, w);
    T *const to = y + (r0 + r) * sy + c0 + c;
    const bool whole = c >= 0 && c + 4 <= cols;
    Four<T> o;
    if (ACC && whole)
      o.template load<false>(to);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T u = p.keeps(w[j]) ? tile[r][min(max(c + j, 0), DROP_TILE - 1)] * scale : T(0);
      if (whole)
        o.set(j, ACC ? o.get(j) + u : u);
      else if (c + j >= 0 && c + j < cols)
        to[j] = ACC ? to[j] + u : u;
    }
    if (whole)
      o.template store<false>(to);
  }
}

struct DropoutViews {
  int ndim;
  int64_t shape[NT_MAX_DIMS], sx[NT_MAX_DIMS], sy[NT_MAX_DIMS];
};

// Any strides: a work-item takes one element.
template <class T, bool ACC>
__global__ __launch_bounds__(DROP_THREADS) void dropout_strided_kernel(
    const T *__restrict__ x, T *__restrict__ y, int64_t n, DropoutViews v,
    DropoutPlan p) {
  const int64_t stride = int64_t(gridDim.x) * DROP_THREADS;
  const T scale = T(p.scale);
  for (int64_t i = int64_t(blockIdx.x) * DROP_THREADS + threadIdx.x; i < n;
       i += stride) {
    int64_t rem = i, ox = 0, oy = 0;
    for (int d = v.ndim - 1; d >= 0; --d) {
      const int64_t q = rem / v.shape[d], c = rem - q * v.shape[d];
      rem = q;
      ox += c * v.sx[d];
      oy += c * v.sy[d];
    }
    uint32_t w[4];
    philox(uint64_t(i) >> 2, p, w);
    const int j = int(i & 3);
    const uint32_t r = j == 0 ? w[0] : j == 1 ? w[1] : j == 2 ? w[2] : w[3];
    const T u = p.keeps(r) ? x[ox] * scale : T(0);
    y[oy] = ACC ? y[oy] + u : u;
  }
}

namespace {

template <class T, bool ACC>
void run_dropout(const nt_view *x, const nt_view *y, const DropoutPlan &p) {
  const int64_t n = numel(x);
  if (n == 0)
    return;
  const ByteRange rd[2] = {view_bytes(x), view_bytes(y)}, wr[1] = {view_bytes(y)};
  const uint32_t flags = ew_launch_flags(rd, ACC ? 2 : 1, wr, 1);
  const nt_view *ops[2] = {x, y};
  const JointLayout L = coalesce(ops, 2);
  const T *px = typed_ptr<const T>(x);
  T *py = typed_ptr<T>(y);
  const bool flat = L.ndim == 0 ||
                    (L.ndim == 1 && L.strides[0][0] == 1 && L.strides[1][0] == 1);
  if (flat) {
    const int64_t vecs = (n + RowVec<T>::N - 1) / RowVec<T>::N;
    const int64_t most = int64_t(DROP_THREADS) << 22;
    for (int64_t v = 0; v < vecs; v += most) {
      const dim3 grid{unsigned((std::min(most, vecs - v) + DROP_THREADS - 1) / DROP_THREADS)};
      ew_launch(dropout_flat_kernel<T, ACC>, grid, DROP_THREADS, stream(), flags, px, py, n,
                v, p);
    }
    return;
  }
  if (L.ndim == 2 && L.strides[0][0] == 1 && L.strides[1][1] == 1) {
    const int64_t tr = (L.shape[0] + DROP_TILE - 1) / DROP_TILE,
                  tc = (L.shape[1] + DROP_TILE - 1) / DROP_TILE;
    if (tr * tc < int64_t(1) << 24) {
      ew_launch(dropout_tile_kernel<T, ACC>, dim3(unsigned(tr * tc)), DROP_THREADS, stream(),
                flags, px, L.strides[0][1], py, L.strides[1][0], L.shape[0], L.shape[1], tc,
                p);
      return;
    }
  }
  const dim3 grid{unsigned(std::min<int64_t>((n + DROP_THREADS - 1) / DROP_THREADS,
                                             int64_t(1) << 22))};
  DropoutViews v{};
  v.ndim = L.ndim;
  for (int d = 0; d < L.ndim; ++d) {
    v.shape[d] = L.shape[d];
    v.sx[d] = L.strides[0][d];
    v.sy[d] = L.strides[1][d];
  }
  ew_launch(dropout_strided_kernel<T, ACC>, grid, DROP_THREADS, stream(), flags, px, py,
            n, v, p);
}

} // namespace
} // namespace nt

using namespace nt;

extern "C" {

int nt_dropout(const nt_view *x, double p, uint64_t seed, uint64_t offset,
               const nt_view *y, int32_t accumulate) {
  return guard_ew([&] {
    check_view(x, "dropout");
    check_view(y, "dropout");
    require_same_shape(x, y, "dropout");
    require_same_dtype(x, y, "dropout");
    if (!(p >= 0.0 && p <= 1.0))
      fail(NT_ERR_VALUE, "dropout: p must lie in [0, 1]");
    DropoutPlan plan;
    const uint64_t threshold = uint64_t(std::nearbyint(p * 4294967296.0));
    plan.none = threshold >> 32 != 0;
    plan.threshold = uint32_t(threshold);
    plan.seed = seed;
    plan.offset = offset;
    plan.scale = p < 1.0 ? 1.0 / (1.0 - p) : 0.0;
    dispatch_float(x->dtype, [&]<class T>() {
      if (accumulate)
        run_dropout<T, true>(x, y, plan);
      else
        run_dropout<T, false>(x, y, plan);
    });
  });
}

} // extern "C"

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

// x [B, R, C] stored by columns (adjacent elements along R), y by rows: tiles
// of 64 x 64 through LDS.  Reading, a wave takes a column's 64 elements;
// writing, a work-item takes a counter's four elements of a row, of which
// those at the tile's edge may belong to the next tile (C need not be a
// multiple of 4).  [64, 512, 1024] with its last axes exchanged takes 44.5 us
// (6.0 TB/s).
constexpr int DROP_TILE = 64;

template <class T, bool ACC>
__global__ __launch_bounds__(DROP_THREADS) void dropout_tile_kernel(
    const T *__restrict__ x, int64_t bx, int64_t sx, T *__restrict__ y, int64_t by, int64_t sy,
    int64_t R, int64_t C, uint32_t tiles, uint32_t tiles_c, DropoutPlan p) {
  __shared__ T tile[DROP_TILE][DROP_TILE + 1];
  const uint32_t b = blockIdx.x / tiles, at = blockIdx.x % tiles;
  const int64_t r0 = int64_t(at / tiles_c) * DROP_TILE, c0 = int64_t(at % tiles_c) * DROP_TILE;
  x += b * bx;
  y += b * by;
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
    const int64_t i0 = (b * R + r0 + r) * C + c0; // the tile's first element of the row
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

// Quotients by a view's sizes: of indexes below 2^32, and of any.
struct Size64 {
  uint64_t d;
  Size64() : d(1) {}
  explicit Size64(uint64_t n) : d(n) {}
  __device__ __forceinline__ uint64_t div(uint64_t n) const { return n / d; }
};

template <class Size> struct DropoutViews {
  int ndim;
  Size shape[NT_MAX_DIMS];
  int64_t sx[NT_MAX_DIMS], sy[NT_MAX_DIMS];

  // The offsets of element i; its position in the innermost dimension.
  template <class I> __device__ __forceinline__ I find(I i, int64_t &ox, int64_t &oy) const {
    ox = oy = 0;
    I at = 0;
    for (int d = ndim - 1; d >= 0; --d) {
      const I q = shape[d].div(i), c = i - q * I(shape[d].d);
      i = q;
      at = d == ndim - 1 ? c : at;
      ox += int64_t(c) * sx[d];
      oy += int64_t(c) * sy[d];
    }
    return at;
  }
};

// Any strides: a work-item takes a counter's four elements, side by side
// where they lie in one row of the innermost dimension (ROWS: its elements
// are adjacent in both operands).  Bound by memory: 2048 columns of 8192 x 4096
// float32 take 23.6 us (5.7 TB/s; with an element per work-item, each drawing
// its counter, 68.9), [64, 512, 16, 64] with its middle axes exchanged 44.7
// (6.0 TB/s; 187), every second column of 8192 x 4096 33 (54).
template <class T, bool ACC, bool ROWS, class Size, class I>
__global__ __launch_bounds__(DROP_THREADS) void dropout_strided_kernel(
    const T *__restrict__ x, T *__restrict__ y, int64_t n, int64_t group0,
    DropoutViews<Size> v, DropoutPlan p) {
  const int64_t group = group0 + int64_t(blockIdx.x) * DROP_THREADS + threadIdx.x, i = 4 * group;
  if (i >= n)
    return;
  int64_t ox, oy;
  const I c = v.find(I(i), ox, oy), C = I(v.shape[v.ndim - 1].d);
  uint32_t w[4];
  philox(uint64_t(group), p, w);
  const T scale = T(p.scale);
  if (C - c >= 4) {
    const int64_t sx = v.sx[v.ndim - 1], sy = v.sy[v.ndim - 1];
    Four<T> in, old;
    if constexpr (ROWS) {
      in.template load<true>(x + ox);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        in.set(j, x[ox + j * sx]);
    }
    if constexpr (ACC) {
      if (ROWS || sy == 1) {
        old.template load<false>(y + oy);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          old.set(j, y[oy + j * sy]);
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const T u = p.keeps(w[j]) ? in.get(j) * scale : T(0);
      in.set(j, ACC ? old.get(j) + u : u);
    }
    if (ROWS || sy == 1) {
      in.template store<true>(y + oy);
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        y[oy + j * sy] = in.get(j);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (i + j >= n)
      break;
    v.find(I(i + j), ox, oy);
    const T u = p.keeps(w[j]) ? x[ox] * scale : T(0);
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
  const int k = L.ndim - 2; // of the rows, from where there are two dimensions or three
  if ((k == 0 || k == 1) && L.strides[0][k] == 1 && L.strides[1][k + 1] == 1) {
    const int64_t R = L.shape[k], C = L.shape[k + 1], B = k ? L.shape[0] : 1;
    const int64_t tr = (R + DROP_TILE - 1) / DROP_TILE, tc = (C + DROP_TILE - 1) / DROP_TILE;
    if (B * tr * tc < int64_t(1) << 24) {
      ew_launch(dropout_tile_kernel<T, ACC>, dim3(unsigned(B * tr * tc)), DROP_THREADS, stream(),
                flags, px, L.strides[0][0], L.strides[0][k + 1], py, L.strides[1][0],
                L.strides[1][k], R, C, uint32_t(tr * tc), uint32_t(tc), p);
      return;
    }
  }
  const auto strided = [&]<bool ROWS, class Size, class I>() {
    DropoutViews<Size> v{};
    v.ndim = L.ndim;
    for (int d = 0; d < L.ndim; ++d) {
      v.shape[d] = Size(L.shape[d]);
      v.sx[d] = L.strides[0][d];
      v.sy[d] = L.strides[1][d];
    }
    const int64_t groups = (n + 3) / 4, most = int64_t(DROP_THREADS) << 22;
    for (int64_t g = 0; g < groups; g += most) {
      const dim3 grid{unsigned((std::min(most, groups - g) + DROP_THREADS - 1) / DROP_THREADS)};
      ew_launch(dropout_strided_kernel<T, ACC, ROWS, Size, I>, grid, DROP_THREADS, stream(),
                flags, px, py, n, g, v, p);
    }
  };
  const bool rows = L.strides[0][L.ndim - 1] == 1 && L.strides[1][L.ndim - 1] == 1;
  if (n < int64_t(1) << 32)
    rows ? strided.template operator()<true, FastDivU32, uint32_t>()
         : strided.template operator()<false, FastDivU32, uint32_t>();
  else
    rows ? strided.template operator()<true, Size64, uint64_t>()
         : strided.template operator()<false, Size64, uint64_t>();
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

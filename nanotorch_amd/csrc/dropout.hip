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
  uint64_t threshold; // keeps r >= threshold, 0 <= threshold <= 2^32
  uint64_t seed, offset;
  double scale;
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

// Contiguous operands: a work-item takes a counter's four elements.
template <class T, bool ACC>
__global__ __launch_bounds__(DROP_THREADS) void dropout_flat_kernel(
    const T *__restrict__ x, T *__restrict__ y, int64_t n, DropoutPlan p) {
  const int64_t groups = (n + 3) / 4;
  const int64_t stride = int64_t(gridDim.x) * DROP_THREADS;
  const T scale = T(p.scale);
  for (int64_t g = int64_t(blockIdx.x) * DROP_THREADS + threadIdx.x; g < groups;
       g += stride) {
    uint32_t w[4];
    philox(uint64_t(g), p, w);
    for (int j = 0; j < 4; ++j) {
      const int64_t i = 4 * g + j;
      if (i >= n)
        break;
      const T v = uint64_t(w[j]) >= p.threshold ? x[i] * scale : T(0);
      y[i] = ACC ? y[i] + v : v;
    }
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
    const T u = uint64_t(r) >= p.threshold ? x[ox] * scale : T(0);
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
  const int64_t items = flat ? (n + 3) / 4 : n;
  const dim3 grid{unsigned(std::min<int64_t>((items + DROP_THREADS - 1) / DROP_THREADS,
                                             int64_t(1) << 22))};
  if (flat) {
    ew_launch(dropout_flat_kernel<T, ACC>, grid, DROP_THREADS, stream(), flags, px, py,
              n, p);
    return;
  }
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
    plan.threshold = uint64_t(std::nearbyint(p * 4294967296.0));
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

// The AdamW step (Loshchilov and Hutter, "Decoupled weight decay
// regularization", 2019) over many parameters in one launch:
//
//   m = b1 m + (1 - b1) g          v = b2 v + (1 - b2) g^2
//   p = p - lr wd p - lr (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps)
//
// Seven streams of the parameters' size (p, g, m, v read, p, m, v written)
// and some 60 instructions an element: bound by HBM from a few million
// elements on, by the launch below.  184 million in 122 parameters take 905 us,
// 287 million in 12 1375: 5.7 and 5.85 TB/s.  (Two 16-byte pieces of each stream to a
// work-item, or eight, or workgroups of 512 took 2 to 5% longer, loads and stores
// without the streaming hint 8%.)  Coefficients are formed on the host in
// 64 bits and rounded once; the element's own arithmetic is in its type.  The decay
// is added to the update before p is rounded, once: 1 - lr wd in float32, a multiple of
// 2^-24 and the same in every step, would decay by 19% too much at lr wd = 1e-7 and
// not at all below 3e-8.
#include <algorithm>
#include <cmath>

#include "tokens.h"

namespace nt {

// Parameters of one launch: pointers travel in the kernel's arguments (4 KB
// at most), so a step with new gradients needs no copy to the device.
constexpr int AW_TENSORS = 96;
constexpr int AW_THREADS = 256;
// 16-byte loads of each stream in flight per work-item.
constexpr int AW_VECS = 4;

template <class T> struct AdamwArgs {
  T *p[AW_TENSORS];
  const T *g[AW_TENSORS];
  int64_t state[AW_TENSORS];      // where the tensor's moments begin
  int64_t n[AW_TENSORS];
  uint32_t first[AW_TENSORS + 1]; // its first workgroup
  T *m, *v;
  int count;
  T b1, c1, b2, c2;   // c = 1 - b
  T decay;            // lr wd
  T rate;             // lr / (1 - b1^t)
  T root;             // 1 / sqrt(1 - b2^t)
  T eps;
};

template <class T>
__device__ __forceinline__ void adamw_element(const AdamwArgs<T> &a, T &p, T g, T &m, T &v) {
  m = fma(a.b1, m, a.c1 * g);
  v = fma(a.b2, v, a.c2 * g * g);
  T step = a.rate * m / fma(sqrt(v), a.root, a.eps);
  if (a.decay != T(0)) // (0 times an infinite p would be NaN)
    step = fma(a.decay, p, step);
  p -= step;
}

template <class T>
__global__ __launch_bounds__(AW_THREADS) void adamw_kernel(const AdamwArgs<T> a) {
  using R = RowVec<T>;
  constexpr int CHUNK = AW_THREADS * AW_VECS * R::N;
  // the tensor whose workgroups hold this one; uniform, a few scalar loads
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (a.first[mid] <= blockIdx.x)
      lo = mid;
    else
      hi = mid - 1;
  }
  const int64_t at = int64_t(blockIdx.x - a.first[lo]) * CHUNK;
  const int64_t left = a.n[lo] - at;
  T *p = a.p[lo] + at;
  const T *g = a.g[lo] + at;
  T *m = a.m + a.state[lo] + at, *v = a.v + a.state[lo] + at;
  if (left >= CHUNK) {
    typename R::V vp[AW_VECS], vg[AW_VECS], vm[AW_VECS], vv[AW_VECS];
#pragma unroll
    for (int i = 0; i < AW_VECS; ++i) {
      const int e = (i * AW_THREADS + int(threadIdx.x)) * R::N;
      vp[i] = R::template load<true>(p + e);
      vg[i] = R::template load<true>(g + e);
      vm[i] = R::template load<true>(m + e);
      vv[i] = R::template load<true>(v + e);
    }
#pragma unroll
    for (int i = 0; i < AW_VECS; ++i) {
      const int e = (i * AW_THREADS + int(threadIdx.x)) * R::N;
#pragma unroll
      for (int j = 0; j < R::N; ++j) {
        T x = vp[i][j], y = vm[i][j], z = vv[i][j];
        adamw_element(a, x, T(vg[i][j]), y, z);
        vp[i][j] = x, vm[i][j] = y, vv[i][j] = z;
      }
      R::template store<true>(p + e, vp[i]);
      R::template store<true>(m + e, vm[i]);
      R::template store<true>(v + e, vv[i]);
    }
    return;
  }
  for (int64_t e = threadIdx.x; e < left; e += AW_THREADS) {
    T x = p[e], y = m[e], z = v[e];
    adamw_element(a, x, g[e], y, z);
    p[e] = x, m[e] = y, v[e] = z;
  }
}

namespace {

// No parameter may share memory with another one or with any gradient: the
// launch updates all of them in no particular order.
void check_apart(const nt_adamw_tensor *t, int64_t count, size_t item) {
  struct Span {
    uintptr_t lo, hi;
    bool written;
  };
  std::vector<Span> spans;
  spans.reserve(size_t(2 * count));
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].n == 0)
      continue;
    const auto p = reinterpret_cast<uintptr_t>(t[i].p), g = reinterpret_cast<uintptr_t>(t[i].g);
    spans.push_back({p, p + uintptr_t(t[i].n) * item, true});
    spans.push_back({g, g + uintptr_t(t[i].n) * item, false});
  }
  std::sort(spans.begin(), spans.end(),
            [](const Span &a, const Span &b) { return a.lo < b.lo; });
  uintptr_t end = 0, written = 0; // of all spans so far, and of the written ones
  for (const Span &s : spans) {
    if (s.lo < (s.written ? end : written))
      fail(NT_ERR_RUNTIME, "adamw: parameters that share memory with one another or with "
                           "gradients cannot be updated together");
    end = std::max(end, s.hi);
    if (s.written)
      written = std::max(written, s.hi);
  }
}

template <class T>
void run_adamw(const nt_adamw_tensor *t, int64_t count, const nt_view *m, const nt_view *v,
               double lr, double b1, double b2, double eps, double wd, int64_t step) {
  AdamwArgs<T> a;
  a.m = typed_ptr<T>(m);
  a.v = typed_ptr<T>(v);
  a.b1 = T(b1), a.c1 = T(1.0 - b1);
  a.b2 = T(b2), a.c2 = T(1.0 - b2);
  a.decay = T(lr * wd);
  // 1 - b^t without cancellation where b is next to 1; log(0) = -inf gives 1
  a.rate = T(lr / -std::expm1(double(step) * std::log(b1)));
  a.root = T(1.0 / std::sqrt(-std::expm1(double(step) * std::log(b2))));
  a.eps = T(eps);
  constexpr int64_t CHUNK = AW_THREADS * AW_VECS * RowVec<T>::N;
  int64_t groups = 0;
  a.count = 0;
  auto launch = [&] {
    if (a.count == 0)
      return;
    a.first[a.count] = uint32_t(groups);
    adamw_kernel<T><<<dim3(uint32_t(groups)), AW_THREADS, 0, stream()>>>(a);
    NT_LAUNCH_CHECK();
    a.count = 0;
    groups = 0;
  };
  for (int64_t i = 0; i < count; ++i) {
    if (t[i].n == 0)
      continue;
    const int64_t need = (t[i].n + CHUNK - 1) / CHUNK;
    if (a.count == AW_TENSORS || groups + need >= (int64_t(1) << 31) / AW_THREADS)
      launch();
    a.p[a.count] = static_cast<T *>(t[i].p);
    a.g[a.count] = static_cast<const T *>(t[i].g);
    a.state[a.count] = t[i].state;
    a.n[a.count] = t[i].n;
    a.first[a.count++] = uint32_t(groups);
    groups += need;
  }
  launch();
}

} // namespace

} // namespace nt

using namespace nt;

extern "C" {

int nt_adamw_step(const nt_adamw_tensor *tensors, int64_t count, const nt_view *m,
                  const nt_view *v, double lr, double beta1, double beta2, double eps,
                  double weight_decay, int64_t step) {
  return guard([&] {
    if (count < 0 || (count && tensors == nullptr))
      fail(NT_ERR_RUNTIME, "adamw: null tensors");
    check_view(m, "adamw");
    check_view(v, "adamw");
    require_same_shape(m, v, "adamw");
    require_same_dtype(m, v, "adamw");
    if (m->ndim != 1 || !is_contiguous(m) || !is_contiguous(v))
      fail(NT_ERR_RUNTIME, "adamw: the moments are two contiguous vectors");
    if (!(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0) || step < 1)
      fail(NT_ERR_VALUE, "adamw: 0 <= beta < 1 and step >= 1");
    dispatch_float(m->dtype, [&]<class T>() {
      constexpr int64_t CHUNK = AW_THREADS * AW_VECS * RowVec<T>::N;
      int64_t end = 0;
      for (int64_t i = 0; i < count; ++i) {
        const nt_adamw_tensor &t = tensors[i];
        // in rising order, so no two tensors have one moment
        if (t.n < 0 || t.state < end || t.n > m->shape[0] || t.state > m->shape[0] - t.n)
          fail(NT_ERR_RUNTIME, "adamw: a tensor's moments lie outside the vectors or in another's");
        if (t.n / CHUNK >= (int64_t(1) << 31) / AW_THREADS - 1)
          fail(NT_ERR_RUNTIME, "adamw: a tensor is too large");
        if (t.n && (t.p == nullptr || t.g == nullptr))
          fail(NT_ERR_RUNTIME, "adamw: null tensor");
        end = t.state + t.n;
      }
      check_apart(tensors, count, sizeof(T));
      run_adamw<T>(tensors, count, m, v, lr, beta1, beta2, eps, weight_decay, step);
    });
  });
}

} // extern "C"

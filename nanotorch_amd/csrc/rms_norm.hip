// Root-mean-square norm of rows, with a residual's addition before it, and its
// gradients:
//
//   s = x + residual (or x)    r = (mean s^2 + eps)^-1/2    y = s r w
//   ds = gs + r (g w - n mean(g w n)),  n = s r;      dw = sum over rows of g n
//
// (gs: the gradient of s itself, which the next residual hands back.)  Forward
// and backward each read and write every array once: a row lives in the
// registers of one to sixteen waves, as many as its length needs at up to four
// 16-byte pieces a lane, between the sum over it and its use.  The sums
// are held in the row's type.  Rows longer than that are read twice, the
// second time mostly from the L2, and three times backward, the third for dw.  HBM
// bound: 8192 x 4096 with a residual takes 92 us forward and 82 backward, 537 MB each
// (5.8 and 6.5 TB/s).
//
// dw: every workgroup takes rows w, w + groups, ... and keeps the sums of its
// columns in registers; its partial sums are one row of a workspace, which a
// second kernel adds up in order.  Which rows a workgroup has is a function of
// the shape alone, so dw comes out the same every time.
#include <algorithm>

#include "tokens.h"

namespace nt {

constexpr int RN_MAX_THREADS = 1024;

template <class T> struct NormArgs {
  const T *x, *res, *w; // res and w may be null
  int64_t x_stride, res_stride;
  T *y, *s, *rstd; // s and rstd may be null
  int64_t rows;
  int64_t D;
  T eps;
};

template <class T> struct NormBackArgs {
  const T *s, *w, *rstd, *g, *gs; // w, g and gs may be null
  int64_t s_stride, g_stride, gs_stride;
  T *ds, *part; // either may be null; part: [workgroups, D]
  int64_t rows;
  int64_t D;
};

template <class T> __device__ __forceinline__ T wave_sum(T v) {
#pragma unroll
  for (int o = 32; o; o >>= 1)
    v += __shfl_xor(v, o);
  return v;
}

// The sum over the TPR work-items of a row; every one of them gets it.  `slots`
// alternates between two halves, so that one barrier per row is enough.
template <class T, int TPR> __device__ __forceinline__ T row_sum(T v, T *slots) {
  v = wave_sum(v);
  if constexpr (TPR > WAVE) {
    constexpr int W = TPR / WAVE;
    if ((threadIdx.x & 63) == 0)
      slots[threadIdx.x >> 6] = v;
    __syncthreads();
    v = slots[0];
#pragma unroll
    for (int i = 1; i < W; ++i)
      v += slots[i];
  }
  return v;
}

// A row's piece i of this lane: elements [at, at + N), as many as are left.
template <class T> struct RowPiece {
  using R = RowVec<T>;
  template <bool STREAM = false>
  static __device__ __forceinline__ typename R::V load(const T *p, int64_t at, int64_t D) {
    if (at + R::N <= D)
      return R::template load<STREAM>(p + at);
    typename R::V v{};
#pragma unroll
    for (int j = 0; j < R::N; ++j)
      if (at + j < D)
        v[j] = p[at + j];
    return v;
  }
  template <bool STREAM = false>
  static __device__ __forceinline__ void store(T *p, int64_t at, int64_t D, typename R::V v) {
    if (at + R::N <= D)
      return R::template store<STREAM>(p + at, v);
#pragma unroll
    for (int j = 0; j < R::N; ++j)
      if (at + j < D)
        p[at + j] = v[j];
  }
};

// TPR work-items to a row, PIECES 16-byte pieces to each; a workgroup of
// max(TPR, 256) holds 256 / TPR rows where TPR is less.
template <class T, int TPR, int PIECES>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_kernel(const NormArgs<T> a) {
  constexpr int ROWS = TPR < 256 ? 256 / TPR : 1, N = RowVec<T>::N;
  using P = RowPiece<T>;
  __shared__ T slots[RN_MAX_THREADS / WAVE];
  const int lane = int(threadIdx.x) % TPR;
  const int64_t row = int64_t(blockIdx.x) * ROWS + int(threadIdx.x) / TPR;
  if (row >= a.rows)
    return; // whole waves: rows of several waves have the workgroup to themselves
  const T *x = a.x + row * a.x_stride;
  const T *res = a.res ? a.res + row * a.res_stride : nullptr;
  typename RowVec<T>::V v[PIECES], u[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
    v[i] = P::template load<true>(x, (int64_t(i) * TPR + lane) * N, a.D);
  if (res) {
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
      u[i] = P::template load<true>(res, (int64_t(i) * TPR + lane) * N, a.D);
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[i][j] += u[i][j];
  }
  T sum = 0;
#pragma unroll
  for (int i = 0; i < PIECES; ++i)
#pragma unroll
    for (int j = 0; j < N; ++j)
      sum = fma(v[i][j], v[i][j], sum);
  sum = row_sum<T, TPR>(sum, slots);
  const T r = T(1) / sqrt(sum / T(a.D) + a.eps);
  if (a.rstd && lane == 0)
    a.rstd[row] = r;
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    const int64_t at = (int64_t(i) * TPR + lane) * N;
    if (at >= a.D)
      break;
    if (a.s)
      P::store(a.s + row * a.D, at, a.D, v[i]);
    if (a.w)
      u[i] = P::load(a.w, at, a.D);
#pragma unroll
    for (int j = 0; j < N; ++j)
      v[i][j] = a.w ? v[i][j] * r * u[i][j] : v[i][j] * r;
    P::store(a.y + row * a.D, at, a.D, v[i]);
  }
}

// Rows that no workgroup's registers hold: the sum is read again.
template <class T>
__global__ __launch_bounds__(RN_MAX_THREADS) void rms_norm_long_kernel(const NormArgs<T> a) {
  constexpr int N = RowVec<T>::N;
  using P = RowPiece<T>;
  __shared__ T slots[RN_MAX_THREADS / WAVE];
  const int64_t row = blockIdx.x;
  const T *x = a.x + row * a.x_stride;
  const T *res = a.res ? a.res + row * a.res_stride : nullptr;
  auto read = [&](int64_t at) {
    auto v = P::load(x, at, a.D);
    if (res) {
      const auto u = P::load(res, at, a.D);
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[j] += u[j];
    }
    return v;
  };
  T sum = 0;
  for (int64_t at = int64_t(threadIdx.x) * N; at < a.D; at += RN_MAX_THREADS * N) {
    const auto v = read(at);
#pragma unroll
    for (int j = 0; j < N; ++j)
      sum = fma(v[j], v[j], sum);
  }
  sum = row_sum<T, RN_MAX_THREADS>(sum, slots);
  const T r = T(1) / sqrt(sum / T(a.D) + a.eps);
  if (a.rstd && threadIdx.x == 0)
    a.rstd[row] = r;
  for (int64_t at = int64_t(threadIdx.x) * N; at < a.D; at += RN_MAX_THREADS * N) {
    auto v = read(at);
    if (a.s)
      P::store(a.s + row * a.D, at, a.D, v);
    if (a.w) {
      const auto u = P::load(a.w, at, a.D);
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[j] = v[j] * r * u[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[j] *= r;
    }
    P::store(a.y + row * a.D, at, a.D, v);
  }
}

// Both gradients; a workgroup walks its rows and keeps its columns' part of dw.
template <class T, int TPR, int PIECES>
__global__ __launch_bounds__(TPR < 256 ? 256 : TPR) void rms_norm_bwd_kernel(
    const NormBackArgs<T> a) {
  constexpr int ROWS = TPR < 256 ? 256 / TPR : 1, N = RowVec<T>::N;
  using P = RowPiece<T>;
  using V = typename RowVec<T>::V;
  __shared__ T slots[2][RN_MAX_THREADS / WAVE];
  const int lane = int(threadIdx.x) % TPR, sub = int(threadIdx.x) / TPR;
  V w[PIECES], dw[PIECES];
#pragma unroll
  for (int i = 0; i < PIECES; ++i) {
    dw[i] = V{};
    if (a.w) {
      w[i] = P::load(a.w, (int64_t(i) * TPR + lane) * N, a.D);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        w[i][j] = T(1);
    }
  }
  int turn = 0;
  for (int64_t row = int64_t(blockIdx.x) * ROWS + sub; row < a.rows;
       row += int64_t(gridDim.x) * ROWS, turn ^= 1) {
    const T *s = a.s + row * a.s_stride;
    V n[PIECES], g[PIECES], gs[PIECES];
    const T r = a.rstd[row];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int64_t at = (int64_t(i) * TPR + lane) * N;
      n[i] = P::template load<true>(s, at, a.D);
      g[i] = a.g ? P::template load<true>(a.g + row * a.g_stride, at, a.D) : V{};
    }
    if (a.gs)
#pragma unroll
      for (int i = 0; i < PIECES; ++i)
        gs[i] = P::template load<true>(a.gs + row * a.gs_stride, (int64_t(i) * TPR + lane) * N,
                                       a.D);
    T dot = 0;
#pragma unroll
    for (int i = 0; i < PIECES; ++i)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        n[i][j] *= r;
        dw[i][j] = fma(g[i][j], n[i][j], dw[i][j]);
        g[i][j] *= w[i][j];
        dot = fma(g[i][j], n[i][j], dot);
      }
    if (a.ds == nullptr)
      continue;
    const T mean = row_sum<T, TPR>(dot, slots[turn]) / T(a.D);
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int64_t at = (int64_t(i) * TPR + lane) * N;
      if (at >= a.D)
        break;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const T d = r * (g[i][j] - n[i][j] * mean);
        g[i][j] = a.gs ? gs[i][j] + d : d;
      }
      P::store(a.ds + row * a.D, at, a.D, g[i]);
    }
  }
  if (a.part == nullptr)
    return;
  if constexpr (ROWS > 1) { // the rows' groups one after the other
    __shared__ V join[(ROWS - 1) * TPR];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      if (i)
        __syncthreads();
      if (sub)
        join[(sub - 1) * TPR + lane] = dw[i];
      __syncthreads();
      if (sub == 0)
#pragma unroll
        for (int k = 0; k < ROWS - 1; ++k)
#pragma unroll
          for (int j = 0; j < N; ++j)
            dw[i][j] += join[k * TPR + lane][j];
    }
  }
  if (sub == 0)
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
      const int64_t at = (int64_t(i) * TPR + lane) * N;
      if (at < a.D)
        P::store(a.part + int64_t(blockIdx.x) * a.D, at, a.D, dw[i]);
    }
}

// ds of long rows; their dw is the next kernel's.
template <class T>
__global__ __launch_bounds__(RN_MAX_THREADS) void rms_norm_bwd_long_kernel(
    const NormBackArgs<T> a) {
  constexpr int N = RowVec<T>::N;
  using P = RowPiece<T>;
  __shared__ T slots[RN_MAX_THREADS / WAVE];
  const int64_t row = blockIdx.x;
  const T *s = a.s + row * a.s_stride;
  const T *g = a.g ? a.g + row * a.g_stride : nullptr;
  const T r = a.rstd[row];
  typename RowVec<T>::V vs, vg;
  auto read = [&](int64_t at) { // n and g w
    vs = P::load(s, at, a.D);
    vg = g ? P::load(g, at, a.D) : typename RowVec<T>::V{};
    const auto w = a.w ? P::load(a.w, at, a.D) : typename RowVec<T>::V{};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      vs[j] *= r;
      if (a.w)
        vg[j] *= w[j];
    }
  };
  T dot = 0;
  for (int64_t at = int64_t(threadIdx.x) * N; at < a.D; at += RN_MAX_THREADS * N) {
    read(at);
#pragma unroll
    for (int j = 0; j < N; ++j)
      dot = fma(vg[j], vs[j], dot);
  }
  const T mean = row_sum<T, RN_MAX_THREADS>(dot, slots) / T(a.D);
  for (int64_t at = int64_t(threadIdx.x) * N; at < a.D; at += RN_MAX_THREADS * N) {
    read(at);
    const auto gs =
        a.gs ? P::load(a.gs + row * a.gs_stride, at, a.D) : typename RowVec<T>::V{};
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const T d = r * (vg[j] - vs[j] * mean);
      vg[j] = a.gs ? gs[j] + d : d;
    }
    P::store(a.ds + row * a.D, at, a.D, vg);
  }
}

// dw of long rows: each work-item one column of a run of rows.
template <class T>
__global__ __launch_bounds__(256) void rms_norm_dw_long_kernel(const NormBackArgs<T> a,
                                                               int64_t run) {
  const int64_t col = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (col >= a.D)
    return;
  T sum = 0;
  if (a.g)
    for (int64_t row = blockIdx.y * run; row < min(a.rows, (blockIdx.y + 1) * run); ++row)
      sum = fma(a.g[row * a.g_stride + col], a.s[row * a.s_stride + col] * a.rstd[row], sum);
  a.part[blockIdx.y * a.D + col] = sum;
}

// dw = the partial sums [parts, D] added up in order, for `cols` columns: 32 columns to a workgroup, each half wave
// a 32nd of the parts, eight loads of it on their way at a time.
template <class T>
__global__ __launch_bounds__(1024) void rms_norm_dw_kernel(const T *part, T *dw, int parts,
                                                           int64_t D, int64_t cols) {
  __shared__ T sums[32][32];
  const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
  const int64_t col = int64_t(blockIdx.x) * 32 + lane;
  const int run = (parts + 31) / 32, end = min(parts, (group + 1) * run);
  T sum = 0;
  if (col < cols) {
    int i = group * run;
    for (; i + 8 <= end; i += 8) {
      T v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        v[k] = part[int64_t(i + k) * D + col];
#pragma unroll
      for (int k = 0; k < 8; ++k)
        sum += v[k];
    }
    for (; i < end; ++i)
      sum += part[int64_t(i) * D + col];
  }
  sums[group][lane] = sum;
  __syncthreads();
  if (group || col >= cols)
    return;
#pragma unroll
  for (int k = 1; k < 32; ++k)
    sum += sums[k][lane];
  dw[col] = sum;
}

namespace {

// The fewest work-items whose registers hold a row of D elements, at 4 pieces
// each; false: none do.
template <class T, class F> bool norm_shape(int64_t D, F &&f) {
  const int64_t pieces = (D + RowVec<T>::N - 1) / RowVec<T>::N;
  if (pieces <= 64)
    f.template operator()<64, 1>();
  else if (pieces <= 128)
    f.template operator()<64, 2>();
  else if (pieces <= 256)
    f.template operator()<64, 4>();
  else if (pieces <= 512)
    f.template operator()<256, 2>();
  else if (pieces <= 1024)
    f.template operator()<256, 4>();
  else if (pieces <= 2048)
    f.template operator()<512, 4>();
  else if (pieces <= 4096)
    f.template operator()<1024, 4>();
  else
    return false;
  return true;
}

template <class T> T *rows_of(const nt_view *v, int64_t rows, int64_t D, int dt, int64_t &stride,
                              const char *what) {
  check_view(v, what);
  if (v->dtype != dt)
    fail(NT_ERR_VALUE, std::string("rms_norm: ") + what + " has another dtype");
  if (v->ndim != 2 || v->shape[0] != rows || v->shape[1] != D)
    fail(NT_ERR_RUNTIME, std::string("rms_norm: ") + what + " has another shape");
  if (D > 1 && v->strides[1] != 1)
    fail(NT_ERR_RUNTIME, std::string("rms_norm: rows of ") + what + " need adjacent elements");
  stride = v->strides[0];
  return typed_ptr<T>(v);
}

template <class T> T *dense_of(const nt_view *v, int64_t rows, int64_t D, int dt,
                               const char *what) {
  int64_t stride;
  T *p = rows_of<T>(v, rows, D, dt, stride, what);
  if (rows > 1 && stride != D)
    fail(NT_ERR_RUNTIME, std::string("rms_norm: ") + what + " must be contiguous");
  return p;
}

template <class T> T *vector_of(const nt_view *v, int64_t n, int dt, const char *what) {
  check_view(v, what);
  if (v->dtype != dt)
    fail(NT_ERR_VALUE, std::string("rms_norm: ") + what + " has another dtype");
  if (v->ndim != 1 || v->shape[0] != n || !is_contiguous(v))
    fail(NT_ERR_RUNTIME, std::string("rms_norm: ") + what + " must be a contiguous vector of " +
                             std::to_string(n));
  return typed_ptr<T>(v);
}

void check_rows(const nt_view *x) {
  check_view(x, "rms_norm");
  if (x->ndim != 2)
    fail(NT_ERR_RUNTIME, "rms_norm: expects [rows, D]");
  if (x->shape[1] < 1 || x->shape[1] >= (int64_t(1) << 30) || x->shape[0] >= (int64_t(1) << 30))
    fail(NT_ERR_VALUE, "rms_norm: rows of 1 to 2^30 - 1 elements, fewer than 2^30 of them");
}

// Rows of one launch, whose work-items (up to 1024 a row) are counted in 32 bits.
constexpr int64_t RN_MOST_ROWS = int64_t(1) << 21;
constexpr int64_t RN_MOST_COLUMNS = int64_t(1) << 26; // of rms_norm_dw_kernel: 32 a column

template <class T> void launch_norm(const NormArgs<T> &a) {
  const bool held = norm_shape<T>(a.D, [&]<int TPR, int PIECES>() {
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1;
    rms_norm_kernel<T, TPR, PIECES>
        <<<dim3(uint32_t((a.rows + ROWS - 1) / ROWS)), TPR < 256 ? 256 : TPR, 0, stream()>>>(a);
  });
  if (!held)
    rms_norm_long_kernel<T><<<dim3(uint32_t(a.rows)), RN_MAX_THREADS, 0, stream()>>>(a);
  NT_LAUNCH_CHECK();
}

template <class T> void run_norm(const NormArgs<T> &a) {
  for (int64_t at = 0; at < a.rows; at += RN_MOST_ROWS) {
    NormArgs<T> b = a;
    b.rows = std::min(RN_MOST_ROWS, a.rows - at);
    b.x += at * a.x_stride;
    b.y += at * a.D;
    if (a.res)
      b.res += at * a.res_stride;
    if (a.s)
      b.s += at * a.D;
    if (a.rstd)
      b.rstd += at;
    launch_norm(b);
  }
}

template <class T> void run_norm_bwd(NormBackArgs<T> a, T *dw) {
  // Workgroups that walk rows: two waves to a SIMD (of 1024 work-items one workgroup to
  // a CU, four), which fill the chip with loads (8192 x 4096, both passes: 180 us, 184
  // with four and 191 with eight, whose parts of dw are as many more).
  int64_t parts = 0;
  auto add_up = [&] {
    for (int64_t at = 0; dw && at < a.D; at += RN_MOST_COLUMNS) {
      const int64_t cols = std::min(RN_MOST_COLUMNS, a.D - at);
      rms_norm_dw_kernel<T><<<dim3(uint32_t((cols + 31) / 32)), 1024, 0, stream()>>>(
          a.part + at, dw + at, int(parts), a.D, cols);
      NT_LAUNCH_CHECK();
    }
  };
  const bool held = norm_shape<T>(a.D, [&]<int TPR, int PIECES>() {
    constexpr int ROWS = TPR < 256 ? 256 / TPR : 1, THREADS = TPR < 256 ? 256 : TPR;
    parts = std::min<int64_t>((a.rows + ROWS - 1) / ROWS,
                              int64_t(device_cu_count()) * std::max(512 / THREADS, 1));
    DeviceScratch part(dw && parts > 1 ? size_t(parts) * size_t(a.D) * sizeof(T) : 0);
    a.part = parts > 1 ? part.get<T>() : dw; // one workgroup's part is the whole
    rms_norm_bwd_kernel<T, TPR, PIECES><<<dim3(uint32_t(parts)), THREADS, 0, stream()>>>(a);
    NT_LAUNCH_CHECK();
    if (parts > 1)
      add_up();
  });
  if (held)
    return;
  for (int64_t at = 0; a.ds && at < a.rows; at += RN_MOST_ROWS) {
    NormBackArgs<T> b = a;
    b.s += at * a.s_stride;
    b.rstd += at;
    b.ds += at * a.D;
    if (a.g)
      b.g += at * a.g_stride;
    if (a.gs)
      b.gs += at * a.gs_stride;
    rms_norm_bwd_long_kernel<T><<<dim3(uint32_t(std::min(RN_MOST_ROWS, a.rows - at))),
                                  RN_MAX_THREADS, 0, stream()>>>(b);
    NT_LAUNCH_CHECK();
  }
  if (dw) {
    parts = std::min<int64_t>(a.rows, 64);
    DeviceScratch part(size_t(parts) * size_t(a.D) * sizeof(T));
    a.part = part.get<T>();
    rms_norm_dw_long_kernel<T>
        <<<dim3(uint32_t((a.D + 255) / 256), uint32_t(parts)), 256, 0, stream()>>>(
            a, (a.rows + parts - 1) / parts);
    NT_LAUNCH_CHECK();
    add_up();
  }
}

} // namespace

} // namespace nt

using namespace nt;

extern "C" {

int nt_rms_norm(const nt_view *x, const nt_view *residual, const nt_view *weight, double eps,
                const nt_view *y, const nt_view *sum, const nt_view *rstd) {
  return guard([&] {
    check_rows(x);
    const int64_t rows = x->shape[0], D = x->shape[1];
    const int dt = x->dtype;
    dispatch_float(dt, [&]<class T>() {
      NormArgs<T> a{};
      a.rows = rows;
      a.D = D;
      a.eps = T(eps);
      a.x = rows_of<const T>(x, rows, D, dt, a.x_stride, "x");
      if (residual)
        a.res = rows_of<const T>(residual, rows, D, dt, a.res_stride, "residual");
      if (weight)
        a.w = vector_of<const T>(weight, D, dt, "weight");
      a.y = dense_of<T>(y, rows, D, dt, "y");
      if (sum)
        a.s = dense_of<T>(sum, rows, D, dt, "sum");
      if (rstd)
        a.rstd = vector_of<T>(rstd, rows, dt, "rstd");
      if (rows)
        run_norm(a);
    });
  });
}

int nt_rms_norm_bwd(const nt_view *sum, const nt_view *weight, const nt_view *rstd,
                    const nt_view *g, const nt_view *g_sum, const nt_view *d_sum,
                    const nt_view *d_weight) {
  return guard([&] {
    check_rows(sum);
    const int64_t rows = sum->shape[0], D = sum->shape[1];
    const int dt = sum->dtype;
    dispatch_float(dt, [&]<class T>() {
      NormBackArgs<T> a{};
      a.rows = rows;
      a.D = D;
      a.s = rows_of<const T>(sum, rows, D, dt, a.s_stride, "sum");
      if (weight)
        a.w = vector_of<const T>(weight, D, dt, "weight");
      a.rstd = vector_of<const T>(rstd, rows, dt, "rstd");
      if (g)
        a.g = rows_of<const T>(g, rows, D, dt, a.g_stride, "g");
      if (g_sum)
        a.gs = rows_of<const T>(g_sum, rows, D, dt, a.gs_stride, "g_sum");
      if (d_sum)
        a.ds = dense_of<T>(d_sum, rows, D, dt, "d_sum");
      T *dw = d_weight ? vector_of<T>(d_weight, D, dt, "d_weight") : nullptr;
      if (dw && rows == 0) {
        if (int rc = nt_fill(dw, dt, D, 0.0))
          fail(rc, nt_last_error());
        return;
      }
      if (rows && (a.ds || dw))
        run_norm_bwd(a, dw);
    });
  });
}

} // extern "C"

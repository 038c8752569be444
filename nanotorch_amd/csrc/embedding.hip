// Rows of a table looked up by token, and the table's gradient:
//
//   y[i, :]  = scale * W[t_i, :]
//   dW[v, :] = scale * sum over the i with t_i = v, in rising i, of g[i, :]
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

// ---------------------------------------------------------------- lookup

template <class T>
__global__ __launch_bounds__(EMB_THREADS) void embedding_kernel(
    const T *__restrict__ table, int64_t rs, int64_t cs, int64_t V, Tokens tok,
    int64_t padding, T scale, T *__restrict__ out, int64_t N, int64_t D,
    int *err) {
  const int64_t total = N * D, stride = int64_t(gridDim.x) * EMB_THREADS;
  for (int64_t e = int64_t(blockIdx.x) * EMB_THREADS + threadIdx.x; e < total;
       e += stride) {
    const int64_t i = e / D, c = e - i * D, t = tok[i];
    T v = T(0);
    if (t >= 0 && t < V) {
      if (t != padding)
        v = table[t * rs + c * cs] * scale;
    } else {
      *err = NT_ERR_INDEX; // the deferred-error word (host memory)
    }
    out[e] = v;
  }
}

// -------------------------------------------------------------- gradient

constexpr int EMB_SCAN = 2048;          // tokens that one scan holds
constexpr int EMB_SEG = EMB_SCAN / 4;   // of them per wave
constexpr int EMB_FLIGHT = 8;           // rows of g in flight per wave

// Tokens i0 .. i0 + n - 1, n <= EMB_SCAN.  A workgroup owns R rows of dW and
// 64 vectors of columns.  Each wave lists the tokens of its quarter that name
// one of the rows, in order; then each wave sums and writes the rows
// wave, wave + 4, ...
template <class T, bool ACC>
__global__ __launch_bounds__(EMB_THREADS) void embedding_scan_kernel(
    const T *__restrict__ g, Tokens tok, int64_t i0, int n, int64_t padding,
    T scale, T *__restrict__ dw, int64_t rs, int64_t V, int64_t D, int R,
    int chunks, int *err) {
  using RV = RowVec<T>;
  __shared__ uint32_t list[4][EMB_SEG]; // row in the tile << 11 | token
  __shared__ int count[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t v0 = int64_t(blockIdx.x / chunks) * R;
  const int64_t col = (int64_t(blockIdx.x % chunks) * 64 + lane) * RV::N;
  {
    const int per = ((n + 3) / 4 + 63) / 64 * 64;
    const int beg = wave * per, end = min(n, beg + per);
    int have = 0;
    for (int b = beg; b < end; b += 64) {
      const int i = b + lane;
      int64_t t = -1;
      if (i < end) {
        t = tok[i0 + i];
        if ((t < 0 || t >= V) && blockIdx.x == 0)
          *err = NT_ERR_INDEX;
      }
      const bool mine = i < end && t >= v0 && t < v0 + R && t < V && t != padding;
      const uint64_t m = __ballot(mine);
      if (mine)
        list[wave][have + __popcll(m & ((uint64_t(1) << lane) - 1))] =
            uint32_t(t - v0) << 11 | uint32_t(i);
      have += __popcll(m);
    }
    if (lane == 0)
      count[wave] = have;
  }
  __syncthreads();
  for (int r = wave; r < R && v0 + r < V; r += 4) {
    T acc[RV::N] = {};
    bool any = false;
    for (int s = 0; s < 4; ++s) {
      const int have = count[s];
      for (int b = 0; b < have; b += 64) {
        const uint32_t e = b + lane < have ? list[s][b + lane] : ~0u;
        uint64_t m = __ballot(e != ~0u && int(e >> 11) == r);
        any |= m != 0;
        while (m) {
          const int i = int(__builtin_amdgcn_readlane(e, __ffsll((unsigned long long)m) - 1)) & 2047;
          m &= m - 1;
          const T *row = g + (i0 + i) * D;
          for (int j = 0; j < RV::N; ++j)
            if (col + j < D)
              acc[j] += row[col + j];
        }
      }
    }
    T *to = dw + (v0 + r) * rs;
    if (ACC && !any)
      continue;
    for (int j = 0; j < RV::N; ++j)
      if (col + j < D)
        to[col + j] = ACC ? to[col + j] + acc[j] * scale : acc[j] * scale;
  }
}

namespace {

template <class T>
void run_embedding(const nt_view *table, const Tokens &tok, int64_t N,
                   int64_t padding, double scale, const nt_view *out) {
  const int64_t V = table->shape[0], D = table->shape[1];
  if (N == 0 || D == 0)
    return;
  const int64_t blocks = std::min<int64_t>((N * D + EMB_THREADS - 1) / EMB_THREADS,
                                           int64_t(1) << 22);
  embedding_kernel<T><<<dim3(unsigned(blocks)), EMB_THREADS, 0, stream()>>>(
      typed_ptr<const T>(table), table->strides[0], table->strides[1], V, tok,
      padding, T(scale), typed_ptr<T>(out), N, D, deferred_error_word());
  NT_LAUNCH_CHECK();
}

template <class T>
void run_embedding_bwd(const nt_view *g, const Tokens &tok, int64_t padding,
                       double scale, const nt_view *dw, bool accumulate) {
  const int64_t N = g->shape[0], D = g->shape[1], V = dw->shape[0];
  if (V == 0 || D == 0)
    return;
  const int chunks = int((D + 64 * RowVec<T>::N - 1) / (64 * RowVec<T>::N));
  const int R = 64;
  const int64_t tiles = (V + R - 1) / R;
  if (tiles * chunks >= (int64_t(1) << 24))
    fail(NT_ERR_VALUE, "embedding_bwd: table too large");
  int64_t i0 = 0;
  do {
    const int n = int(std::min<int64_t>(EMB_SCAN, N - i0));
    const auto args = [&](auto kernel) {
      kernel<<<dim3(unsigned(tiles * chunks)), EMB_THREADS, 0, stream()>>>(
          typed_ptr<const T>(g), tok, i0, n, padding, T(scale), typed_ptr<T>(dw),
          dw->strides[0], V, D, R, chunks, deferred_error_word());
      NT_LAUNCH_CHECK();
    };
    if (accumulate || i0 > 0)
      args(embedding_scan_kernel<T, true>);
    else
      args(embedding_scan_kernel<T, false>);
    i0 += n;
  } while (i0 < N);
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
    dispatch_float(table->dtype, [&]<class T>() {
      run_embedding<T>(table, tok, tokens->shape[0], padding, scale, out);
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
    dispatch_float(g->dtype, [&]<class T>() {
      run_embedding_bwd<T>(g, tok, padding, scale, dtable, accumulate != 0);
    });
  });
}

} // extern "C"

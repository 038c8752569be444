// Log probabilities of given tokens from rows of logits, the entropy of each
// row, its top alternatives, and the gradient of the logits.
//
// One pass over a row keeps, per lane, the running maximum m and the sums
//   s = sum exp(z_j - m),   u = sum exp(z_j - m) (z_j - m),
// from which
//   log p_t = (z_t - m) - log s,
//   H       = -sum p log p = log s - u / s.
// Two such states join by moving both to the larger maximum: with d = m - m'
//   s' = exp(d) s,   u' = exp(d) (u + d s).
// The gradient for upstream a (of log p_t) and b (of H) is
//   dz_j = a [j = t] - p_j (a + b (log p_j + H)),   p_j = exp(z_j - m) / s,
// one pass that reads z and writes dz.  There log p_j + H = (z_j - m) - u / s:
// log s drops out, whose rounding would be all of that difference where a row
// is nearly uniform, as a model's are at its start (64 x 32000 float32 of
// deviation 2^-13: off by 3.0e-7 of its norm, by way of H by 2.5e-3).
//
// Bound by memory where rows are many: 8192 x 32000 float32 (a tenth of the
// rows left out) reads 0.94 GB in 156 us (6.0 TB/s), and its gradient moves
// 2.0 GB in 328 us (6.1 TB/s; with half of the rows left out 268, with all
// 183).  2000 x 50001 takes 68 us, with 5 alternatives 74, with 20 79, with 64
// 115.  Few rows are split over several workgroups and joined by a second
// kernel: 8 x 128000 with 8 alternatives 7.5 + 5.5 us, with 50 14 + 5.5;
// 64 x 128000 10 us in all without alternatives, with 50 25.  Joined by each
// row's last workgroup instead, one launch less, 64 x 128000 without
// alternatives takes 50: every part's release to the other XCDs writes back an
// L2.
//
// Logits of -inf are tokens without probability and count for nothing; a row
// that holds nothing else has log probability -inf, entropy 0 and no
// gradient.  A NaN or +inf makes the row's results NaN.  A row whose token
// is `ignore` is not read: results 0, alternatives -inf and -1, gradient 0.
// One whose token lies outside the row is treated so too and reported at the
// next synchronisation (the library's deferred error).
//
// The alternatives are the k largest logits, ties to the lowest token, NaN
// above every number.  Each wave keeps its own k best, the i-th in lane i;
// a chunk's elements are looked at one by one only where some lane's maximum
// (which the pass computes anyway) exceeds the k-th best so far, and the first
// chunk's only where they reach the k-th largest of the maxima of all lanes
// that share the row: in n elements of random order about k (1 + ln(n / c))
// of them, c being a chunk.  The lists of waves and workgroups are merged by a
// bitonic network over the lanes (K. Batcher, "Sorting networks and their
// applications", AFIPS 1968), about a hundred instructions a list; entry by
// entry, 8 x 128000 with 50 alternatives took 18 + 28 us.
#include "tokens.h"

#include <algorithm>
#include <limits>

namespace nt {

constexpr int LP_THREADS = 256;
constexpr int LP_WAVES = LP_THREADS / WAVE;
constexpr int LP_UNROLL = 4;  // vectors in flight per lane
constexpr int LP_TOP_MAX = WAVE;

// exp of d <= 0.  exp2's argument d log2 e is taken in two parts, the rounded
// product h and its error l, so that the rounding (2^-24 of |d| log2 e) is not
// multiplied up by large |d|: log2 e as a sum of two constants (W. Cody,
// W. Waite, "Software manual for the elementary functions", 1980), the
// product's own error by a fused multiply-add.
__device__ __forceinline__ float exp_of(float d) {
  constexpr float L = 1.44269504f;          // log2 e, rounded
  constexpr float L_LOW = 1.92596303e-8f;   // log2 e - L
  constexpr float LN2 = 0.693147181f;
  const float h = d * L;
  const float l = __builtin_fmaf(d, L_LOW, __builtin_fmaf(d, L, -h));
  const float e = __builtin_amdgcn_exp2f(h);
  return __builtin_fmaf(e, l * LN2, e);
}
// 2^k exp(r) with |r| <= ln 2 / 2, k ln 2 subtracted in two parts as there,
// where exp(r) is 1 + r + r^2 q(r); q
// interpolates at the Chebyshev nodes of that interval (error 0.15 2^-53).
// 8192 x 16000 takes 207 us and 383 for its gradient, with the general exp()
// 236 and 389.
__device__ __forceinline__ double exp_of(double d) {
  const double k = __builtin_rint(d * 1.4426950408889634);
  const double r = __builtin_fma(k, -2.3190468138462996e-17,
                                 __builtin_fma(k, -0.6931471805599453, d));
  double q = 2.510038549551032e-08;
  q = __builtin_fma(q, r, 2.7620088445409746e-07);
  q = __builtin_fma(q, r, 2.7557268459997064e-06);
  q = __builtin_fma(q, r, 2.4801521295954376e-05);
  q = __builtin_fma(q, r, 0.00019841269863053618);
  q = __builtin_fma(q, r, 0.0013888888917213717);
  q = __builtin_fma(q, r, 0.008333333333330062);
  q = __builtin_fma(q, r, 0.04166666666662413);
  q = __builtin_fma(q, r, 0.16666666666666669);
  q = __builtin_fma(q, r, 0.5000000000000001);
  q = __builtin_fma(q * r, r, r);
  return __builtin_amdgcn_ldexp(1.0 + q, int(k));
}

// Past this distance from the maximum exp() is 0 in T.
template <class T> constexpr T LP_CUT = sizeof(T) == 4 ? T(-200) : T(-800);

template <class T> __device__ __forceinline__ T not_below_cut(T d) {
  if constexpr (sizeof(T) == 4)
    return __builtin_elementwise_maximum(d, LP_CUT<T>); // NaN stays
  else // float64 has no such instruction
    return d < LP_CUT<T> ? LP_CUT<T> : d;
}

// The larger one; NaN if either is.
template <class T> __device__ __forceinline__ T max_nan(T a, T b) {
  return __builtin_elementwise_maximum(a, b);
}

// A lane's value from the lane that the data-parallel control CTRL names;
// `none` where there is no such lane or ROWS leaves the lane's row out.
template <int CTRL, int ROWS, class T> __device__ __forceinline__ T from_lane(T v, T none) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(
        T, __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, none),
                                       __builtin_bit_cast(int, v), CTRL, ROWS, 0xf, false));
  } else {
    const uint64_t a = __builtin_bit_cast(uint64_t, none), b = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(int(a), int(b), CTRL, ROWS, 0xf, false);
    const uint32_t hi =
        __builtin_amdgcn_update_dpp(int(a >> 32), int(b >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(T, uint64_t(hi) << 32 | lo);
  }
}
constexpr int DPP_ROW_SHR = 0x110, DPP_WAVE_SHR1 = 0x138, DPP_BCAST15 = 0x142,
              DPP_BCAST31 = 0x143;

__device__ __forceinline__ uint32_t read_lane(uint32_t v, int l) {
  return __builtin_amdgcn_readlane(v, l);
}
__device__ __forceinline__ uint64_t read_lane(uint64_t v, int l) {
  return uint64_t(uint32_t(__builtin_amdgcn_readlane(uint32_t(v >> 32), l))) << 32 |
         uint32_t(__builtin_amdgcn_readlane(uint32_t(v), l));
}

// f over the wave's values, in every lane; `none` is f's neutral value.
template <class T, class F> __device__ __forceinline__ T over_wave(T v, T none, F f) {
  v = f(v, from_lane<DPP_ROW_SHR + 1, 0xf>(v, none));
  v = f(v, from_lane<DPP_ROW_SHR + 2, 0xf>(v, none));
  v = f(v, from_lane<DPP_ROW_SHR + 4, 0xf>(v, none));
  v = f(v, from_lane<DPP_ROW_SHR + 8, 0xf>(v, none));
  v = f(v, from_lane<DPP_BCAST15, 0xa>(v, none));
  v = f(v, from_lane<DPP_BCAST31, 0xc>(v, none));
  using I = std::conditional_t<sizeof(T) == 4, uint32_t, uint64_t>;
  return __builtin_bit_cast(T, read_lane(__builtin_bit_cast(I, v), WAVE - 1));
}

// f over each group of G adjacent lanes (4 or 16), in every lane of it; f is
// commutative.
template <int G, class T, class F> __device__ __forceinline__ T over_lanes(T v, F f) {
  static_assert(G == 4 || G == 16);
  v = f(v, from_lane<0xB1, 0xf>(v, v)); // lane i: i ^ 1
  v = f(v, from_lane<0x4E, 0xf>(v, v)); // i ^ 2
  if constexpr (G == 16) {
    v = f(v, from_lane<0x141, 0xf>(v, v)); // the other end of eight
    v = f(v, from_lane<0x140, 0xf>(v, v)); // of sixteen
  }
  return v;
}

// A word from lane i ^ S.
template <int S> __device__ __forceinline__ uint32_t from_xor(uint32_t v) {
  if constexpr (S == 1)
    return from_lane<0xB1, 0xf>(v, v);
  else if constexpr (S == 2)
    return from_lane<0x4E, 0xf>(v, v);
  else if constexpr (S == 4) { // four lanes up in every other four, down in the rest
    const int up = __builtin_amdgcn_update_dpp(int(v), int(v), 0x104, 0xf, 0x5, false);
    return __builtin_amdgcn_update_dpp(up, int(v), 0x114, 0xf, 0xa, false);
  } else if constexpr (S == 8)
    return from_lane<0x128, 0xf>(v, v);
  else if constexpr (S == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  } else {
    static_assert(S == 32);
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return threadIdx.x & 32 ? r[0] : r[1];
  }
}
template <int S> __device__ __forceinline__ uint64_t from_xor(uint64_t v) {
  return uint64_t(from_xor<S>(uint32_t(v >> 32))) << 32 | from_xor<S>(uint32_t(v));
}

template <class T> struct RowState {
  T m = -std::numeric_limits<T>::infinity(), s = T(0), u = T(0);

  __device__ __forceinline__ void move_to(T to) {
    if (s != T(0) && m != to) {
      const T d = not_below_cut(m - to), c = exp_of(d);
      u = c * (u + d * s);
      s = c * s;
    }
    m = to;
  }
  __device__ __forceinline__ void join(RowState o) {
    const T to = max_nan(m, o.m);
    move_to(to);
    o.move_to(to);
    s += o.s;
    u += o.u;
  }
  // A lane's N values; -inf where there is none.
  template <int N> __device__ __forceinline__ void add(const T (&z)[N], T top) {
    if (!(top <= m))
      move_to(max_nan(m, top));
    const T ref = m == -std::numeric_limits<T>::infinity() ? T(0) : m;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const T d = not_below_cut(z[i] - ref), e = exp_of(d);
      s += e;
      u = __builtin_elementwise_fma(e, d, u);
    }
  }
  // Every lane gets the state of its group of G lanes.
  template <int G = WAVE> __device__ __forceinline__ void join_lanes() {
    const auto larger = [](T a, T b) { return max_nan(a, b); };
    const auto add = [](T a, T b) { return a + b; };
    if constexpr (G == WAVE) {
      move_to(over_wave(m, -std::numeric_limits<T>::infinity(), larger));
      s = over_wave(s, T(0), add);
      u = over_wave(u, T(0), add);
    } else {
      move_to(over_lanes<G>(m, larger));
      s = over_lanes<G>(s, add);
      u = over_lanes<G>(u, add);
    }
  }
};

// ------------------------------------------------------------ alternatives

// Keys order as the logits do, as unsigned integers: 0 is no entry, NaN is
// the largest, -0 equals 0.
template <class T> struct Key;
template <> struct Key<float> {
  using K = uint32_t;
  static __device__ __forceinline__ K of(float v) {
    if (v != v)
      return ~K(0);
    const K b = __builtin_bit_cast(K, v + 0.0f);
    return b >> 31 ? ~b : b | K(1) << 31;
  }
  static __device__ __forceinline__ float value(K k) {
    if (k == ~K(0))
      return std::numeric_limits<float>::quiet_NaN();
    return __builtin_bit_cast(float, k >> 31 ? k ^ K(1) << 31 : ~k);
  }
};
template <> struct Key<double> {
  using K = uint64_t;
  static __device__ __forceinline__ K of(double v) {
    if (v != v)
      return ~K(0);
    const K b = __builtin_bit_cast(K, v + 0.0);
    return b >> 63 ? ~b : b | K(1) << 63;
  }
  static __device__ __forceinline__ double value(K k) {
    if (k == ~K(0))
      return std::numeric_limits<double>::quiet_NaN();
    return __builtin_bit_cast(double, k >> 63 ? k ^ K(1) << 63 : ~k);
  }
};

constexpr int RAISE_BITS = 20; // sign, exponent and 11 (of a double, 8) bits more

constexpr int TOP_ALONE = WAVE / 2;

// A wave's best entries in falling order, the i-th in lane i.
template <class T> struct TopList {
  using K = typename Key<T>::K;
  K key = 0;
  int32_t token = -1;
  K least = 0; // what an entry has to exceed to be among the k best

  __device__ __forceinline__ void insert(K v, int32_t t, int k) {
    // Lanes of smaller keys move on by one: each key becomes the middle one
    // of itself, its neighbour's (no smaller) and v.
    const K up = from_lane<DPP_WAVE_SHR1, 0xf>(key, ~K(0));
    const int32_t up_t = from_lane<DPP_WAVE_SHR1, 0xf>(token, 0);
    const bool stays = key >= v, here = up >= v;
    token = stays ? token : here ? t : up_t;
    key = stays ? key : here ? v : up;
    least = max(least, read_lane(key, k - 1));
  }
  // Lists of up to 16 entries are joined within 16 lanes.
  static __device__ __forceinline__ int width(int k) { return k <= 16 ? 16 : WAVE; }
  // The entry that a lane brings to merge(); its list has it if it is below k.
  static __device__ __forceinline__ uint32_t brings(int lane, int k) {
    return uint32_t(width(k) - 1 - lane);
  }
  // Another list, from its end.  The better one of each lane's two entries is
  // among the best of both lists, and these rise and then fall along the
  // lanes: exchanges at halving distances sort them.
  __device__ __forceinline__ void merge(K v, int32_t t, int k) {
    if (read_lane(v, width(k) - 1) < least)
      return;
    const bool take = v > key || (v == key && t < token);
    key = take ? v : key;
    token = take ? t : token;
    if (k > 16) {
      exchange<32>();
      exchange<16>();
    }
    exchange<8>();
    exchange<4>();
    exchange<2>();
    exchange<1>();
    least = max(least, read_lane(key, k - 1));
  }
  template <int S> __device__ __forceinline__ void exchange() {
    const K v = from_xor<S>(key);
    const int32_t t = int32_t(from_xor<S>(uint32_t(token)));
    const bool better = v > key || (v == key && t < token);
    const bool take = better == ((threadIdx.x & S) == 0);
    key = take ? v : key;
    token = take ? t : token;
  }
  // Of the lanes' keys x, N each, the k-th largest is found bit by bit, its
  // leading RAISE_BITS; nothing below it is among the k best of anything that
  // holds those keys.
  template <int N> __device__ __forceinline__ void raise(const K (&x)[N], int k) {
    K at = 0;
#pragma unroll
    for (int b = 0; b < RAISE_BITS; ++b) {
      const K up = at | K(1) << (8 * sizeof(K) - 1 - b);
      int n = 0;
#pragma unroll
      for (int j = 0; j < N; ++j)
        n += __popcll(__ballot(x[j] >= up));
      at = n >= k ? up : at;
    }
    // just below it; no logit has the key below 0's (that of -0)
    if (at)
      least = max(least, at - (at == Key<T>::of(T(0)) ? 2 : 1));
  }
  // From a wave's first chunk alone.  Beyond TOP_ALONE alternatives the 64
  // maxima bound little: then a lane gives the maximum of each of its vectors
  // (8192 x 1000, k = 50 and 64, us: 33 and 39, by 64 maxima 46 and 100).
  template <int N> __device__ __forceinline__ void raise_alone(const T (&v)[N], T most, int k) {
    if (k <= TOP_ALONE) {
      const K one[1] = {Key<T>::of(most)};
      return raise(one, k);
    }
    constexpr int PER = N / LP_UNROLL;
    K each[LP_UNROLL];
#pragma unroll
    for (int c = 0; c < LP_UNROLL; ++c) {
      T x = v[c * PER];
#pragma unroll
      for (int j = 1; j < PER; ++j)
        x = max_nan(x, v[c * PER + j]);
      each[c] = Key<T>::of(x);
    }
    raise(each, k);
  }
};

// ---------------------------------------------------------------- forward

template <class T> struct LpForward {
  const T *z;
  int64_t row_stride;
  int64_t rows;
  int32_t V;
  Tokens tok; // p null: no given tokens
  int64_t ignore;
  T *logprob, *entropy, *stats, *top_value; // null: not wanted
  int64_t *top_token;
  int k;
  int splits;    // workgroups per row
  int32_t part;  // elements per wave
  // partial states of split rows: [rows][splits] each
  T *pm, *ps, *pu;
  typename Key<T>::K *pkey; // [rows][splits][k]
  int32_t *ptoken;
  int *err;
};

template <class T, int G = WAVE>
__device__ __forceinline__ void write_left_out(const LpForward<T> &a, int64_t row) {
  const int lane = threadIdx.x % G;
  if (lane == 0) {
    if (a.logprob)
      a.logprob[row] = T(0);
    if (a.entropy)
      a.entropy[row] = T(0);
    if (a.stats) {
      a.stats[row] = T(0);
      a.stats[a.rows + row] = T(0);
      a.stats[2 * a.rows + row] = T(0);
    }
  }
  if (lane < a.k) {
    a.top_value[row * a.k + lane] = -std::numeric_limits<T>::infinity();
    a.top_token[row * a.k + lane] = -1;
  }
}

template <class T, int G = WAVE>
__device__ __forceinline__ void write_row(const LpForward<T> &a, int64_t row, int64_t t,
                                          const RowState<T> &r, const TopList<T> &top) {
  const int lane = threadIdx.x % G;
  const bool none = r.s == T(0);
  const T log_s = log(r.s), low = -std::numeric_limits<T>::infinity();
  if (lane == 0) {
    if (a.logprob)
      a.logprob[row] = none ? low : (a.z[row * a.row_stride + t] - r.m) - log_s;
    if (a.entropy)
      a.entropy[row] = none ? T(0) : log_s - r.u / r.s;
    if (a.stats) {
      a.stats[row] = r.m;
      a.stats[a.rows + row] = r.s;
      a.stats[2 * a.rows + row] = r.u;
    }
  }
  if (lane < a.k) {
    a.top_value[row * a.k + lane] =
        none ? low : (Key<T>::value(top.key) - r.m) - log_s;
    a.top_token[row * a.k + lane] = top.token;
  }
}

// The row's token, and whether the row is left out.
template <class T>
__device__ __forceinline__ bool row_left_out(const LpForward<T> &a, int64_t row,
                                             int64_t &t) {
  t = 0;
  if (a.tok.p == nullptr)
    return false;
  t = a.tok[row];
  if (t == a.ignore)
    return true;
  if (t < 0 || t >= a.V) {
    *a.err = NT_ERR_INDEX;
    return true;
  }
  return false;
}

// Elements beg .. end - 1 of a row into the wave's state and list; `first`
// gets each lane's values of the first chunk and their maximum.
template <class T, bool TOP, bool STREAM, class F>
__device__ __forceinline__ void walk(const T *z, int32_t beg, int32_t end, int k,
                                     RowState<T> &r, TopList<T> &top, F &&first) {
  using RV = RowVec<T>;
  constexpr int N = RV::N, CHUNK = WAVE * N * LP_UNROLL;
  const int lane = threadIdx.x & 63;
  const T none = -std::numeric_limits<T>::infinity();
  for (int64_t b = beg; b < end; b += CHUNK) {
    T v[LP_UNROLL * N];
#pragma unroll
    for (int c = 0; c < LP_UNROLL; ++c) {
      const int64_t i = b + (c * WAVE + lane) * N;
      if (i + N <= end) {
        const typename RV::V w = RV::template load<STREAM>(z + i);
#pragma unroll
        for (int j = 0; j < N; ++j)
          v[c * N + j] = w[j];
      } else {
#pragma unroll
        for (int j = 0; j < N; ++j)
          v[c * N + j] = i + j < end ? z[i + j] : none;
      }
    }
    T most = v[0];
#pragma unroll
    for (int j = 1; j < LP_UNROLL * N; ++j)
      most = max_nan(most, v[j]);
    if constexpr (TOP) {
      if (b == beg)
        first(v, most);
      // NaN, which nothing is below, while there is no such bound
      const T least = Key<T>::value(top.least);
      if (__ballot(!(most <= least))) {
#pragma unroll
        for (int c = 0; c < LP_UNROLL; ++c) {
          const int64_t i = b + (c * WAVE + lane) * N;
          uint32_t hits = 0; // a bit per element
#pragma unroll
          for (int j = 0; j < N; ++j)
            hits |= uint32_t(!(v[c * N + j] <= least) && i + j < end) << j;
          uint64_t m = __ballot(hits != 0);
          while (m) { // lane by lane, element by element: in rising order
            const int l = __ffsll((unsigned long long)m) - 1;
            m &= m - 1;
            const uint32_t h = read_lane(hits, l);
#pragma unroll
            for (int j = 0; j < N; ++j)
              if (h >> j & 1) {
                using K = typename Key<T>::K;
                const K x = Key<T>::of(__builtin_bit_cast(
                    T, read_lane(__builtin_bit_cast(K, v[c * N + j]), l)));
                if (x > top.least)
                  top.insert(x, int32_t(b) + (c * WAVE + l) * N + j, k);
              }
          }
        }
      }
    }
    r.add(v, most);
  }
}

// G lanes per row, for short rows without alternatives: 1000000 x 10 float32
// takes 21 us and 22 for its gradient, 100000 x 100 12 and 16 (with a wave per
// row 660 and 71 for both).
template <class T, int G>
__global__ __launch_bounds__(LP_THREADS) void logprob_lanes_kernel(LpForward<T> a,
                                                                   int64_t row0) {
  using RV = RowVec<T>;
  constexpr int N = RV::N;
  const int64_t row = row0 + (int64_t(blockIdx.x) * LP_THREADS + threadIdx.x) / G;
  if (row >= a.rows)
    return;
  int64_t t;
  if (row_left_out(a, row, t))
    return write_left_out<T, G>(a, row);
  const T *z = a.z + row * a.row_stride;
  RowState<T> r;
#pragma unroll
  for (int c = 0; c < LP_UNROLL; ++c) {
    const int i = (c * G + int(threadIdx.x % G)) * N;
    if (c * G * N >= a.V)
      break;
    T v[N];
    if (i + N <= a.V) {
      const typename RV::V w = RV::load(z + i);
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[j] = w[j];
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j)
        v[j] = i + j < a.V ? z[i + j] : -std::numeric_limits<T>::infinity();
    }
    T most = v[0];
#pragma unroll
    for (int j = 1; j < N; ++j)
      most = max_nan(most, v[j]);
    r.add(v, most);
  }
  r.template join_lanes<G>();
  write_row<T, G>(a, row, t, r, TopList<T>());
}

// A wave per row.
template <class T, bool TOP>
__global__ __launch_bounds__(LP_THREADS) void logprob_wave_kernel(LpForward<T> a,
                                                                  int64_t row0) {
  const int64_t row = row0 + int64_t(blockIdx.x) * LP_WAVES + (threadIdx.x >> 6);
  if (row >= a.rows)
    return;
  int64_t t;
  if (row_left_out(a, row, t))
    return write_left_out(a, row);
  RowState<T> r;
  TopList<T> top;
  walk<T, TOP, false>(a.z + row * a.row_stride, 0, a.V, a.k, r, top,
                      [&](const auto &v, T most) { top.raise_alone(v, most, a.k); });
  r.join_lanes();
  write_row(a, row, t, r, top);
}

// `splits` workgroups per row, each wave a part of `part` elements.  Eight
// waves per SIMD (at most 64 registers) hold 2000 rows at once.
template <class T, bool TOP, bool STREAM>
__global__ __launch_bounds__(LP_THREADS, sizeof(T) == 4 ? 8 : 4) void logprob_group_kernel(
    LpForward<T> a, int64_t row0) {
  __shared__ T sm[3][LP_WAVES];
  __shared__ typename Key<T>::K skey[LP_WAVES][LP_TOP_MAX];
  __shared__ int32_t stoken[LP_WAVES][LP_TOP_MAX];
  const int64_t row = row0 + blockIdx.x / a.splits;
  const int split = blockIdx.x % a.splits;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t t;
  if (row_left_out(a, row, t)) {
    if (wave == 0 && a.splits == 1)
      write_left_out(a, row);
    return;
  }
  RowState<T> r;
  TopList<T> top;
  const int64_t row_part = int64_t(split) * LP_WAVES * a.part; // of the workgroup
  const int64_t beg = row_part + wave * int64_t(a.part);
  // the bound by all waves together, unless most of them have nothing
  const bool alone = a.k > TOP_ALONE && row_part + a.part >= a.V;
  const auto share = [&](typename Key<T>::K x) {
    __shared__ typename Key<T>::K most[LP_WAVES][WAVE];
    most[wave][lane] = x;
    __syncthreads();
    typename Key<T>::K all[LP_WAVES];
#pragma unroll
    for (int w = 0; w < LP_WAVES; ++w)
      all[w] = most[w][lane];
    top.raise(all, a.k);
  };
  if (beg < a.V)
    walk<T, TOP, STREAM>(a.z + row * a.row_stride, int32_t(beg),
                         int32_t(std::min<int64_t>(a.V, beg + a.part)), a.k, r, top,
                         [&](const auto &v, T most) {
                           if (alone)
                             top.raise_alone(v, most, a.k);
                           else
                             share(Key<T>::of(most));
                         });
  else if (TOP && !alone)
    share(0);
  r.join_lanes();
  if (lane == 0) {
    sm[0][wave] = r.m;
    sm[1][wave] = r.s;
    sm[2][wave] = r.u;
  }
  if (TOP && lane < a.k) {
    skey[wave][lane] = top.key;
    stoken[wave][lane] = top.token;
  }
  __syncthreads();
  if (wave != 0)
    return;
  for (int w = 1; w < LP_WAVES; ++w) {
    RowState<T> o;
    o.m = sm[0][w];
    o.s = sm[1][w];
    o.u = sm[2][w];
    r.join(o);
    if constexpr (TOP) {
      const uint32_t e = top.brings(lane, a.k);
      top.merge(e < uint32_t(a.k) ? skey[w][e] : 0, e < uint32_t(a.k) ? stoken[w][e] : -1, a.k);
    }
  }
  if (a.splits == 1)
    return write_row(a, row, t, r, top);
  const int64_t at = row * a.splits + split;
  if (lane == 0) {
    a.pm[at] = r.m;
    a.ps[at] = r.s;
    a.pu[at] = r.u;
  }
  if (TOP && lane < a.k) {
    a.pkey[at * a.k + lane] = top.key;
    a.ptoken[at * a.k + lane] = top.token;
  }
}

// Joins the splits of a row: a wave the states, four waves the alternatives.
template <class T, bool TOP>
__global__ __launch_bounds__(TOP ? LP_THREADS : WAVE) void logprob_join_kernel(LpForward<T> a,
                                                                               int64_t row0) {
  using K = typename Key<T>::K;
  const int64_t row = row0 + blockIdx.x;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  int64_t t;
  if (row_left_out(a, row, t)) {
    if (wave == 0)
      write_left_out(a, row);
    return;
  }
  RowState<T> r;
  TopList<T> top;
  if (wave == 0) {
    for (int b = lane; b < a.splits; b += WAVE) {
      RowState<T> o;
      o.m = a.pm[row * a.splits + b];
      o.s = a.ps[row * a.splits + b];
      o.u = a.pu[row * a.splits + b];
      r.join(o);
    }
    r.join_lanes();
  }
  if constexpr (TOP) {
    __shared__ K skey[LP_WAVES][WAVE];
    __shared__ int32_t stoken[LP_WAVES][WAVE];
    constexpr int AHEAD = 8; // lists on their way
    const uint32_t e = top.brings(lane, a.k);
    for (int b = wave; b < a.splits; b += LP_WAVES * AHEAD) {
      K key[AHEAD];
      int32_t token[AHEAD];
#pragma unroll
      for (int j = 0; j < AHEAD; ++j) {
        const int at = b + j * LP_WAVES;
        const bool in = at < a.splits && e < uint32_t(a.k);
        key[j] = in ? a.pkey[(row * a.splits + at) * a.k + e] : 0;
        token[j] = in ? a.ptoken[(row * a.splits + at) * a.k + e] : -1;
      }
#pragma unroll
      for (int j = 0; j < AHEAD; ++j)
        if (b + j * LP_WAVES < a.splits)
          top.merge(key[j], token[j], a.k);
    }
    if (lane < a.k) {
      skey[wave][lane] = top.key;
      stoken[wave][lane] = top.token;
    }
    __syncthreads();
    if (wave != 0)
      return;
    for (int w = 1; w < LP_WAVES; ++w) {
      const bool in = e < uint32_t(a.k);
      top.merge(in ? skey[w][e] : 0, in ? stoken[w][e] : -1, a.k);
    }
  }
  write_row(a, row, t, r, top);
}

// --------------------------------------------------------------- backward

template <class T> struct LpBackward {
  const T *z;
  int64_t row_stride;
  int64_t rows;
  int32_t V;
  Tokens tok;
  int64_t ignore;
  const T *stats;
  const T *ga, *gb; // null: zero
  int64_t sa, sb;   // their strides
  T *dz;
  int64_t dz_stride;
  int last_first; // the last rows first
};

// G lanes per row, each UNROLL vectors; a whole workgroup (G = LP_THREADS)
// takes one of the row's `chunks`.
template <class T, int G, int UNROLL, bool ACC>
__global__ __launch_bounds__(LP_THREADS) void logprob_bwd_kernel(LpBackward<T> a,
                                                                 int64_t row0, int chunks) {
  using RV = RowVec<T>;
  constexpr int N = RV::N, STEP = G * N;
  int64_t row;
  int32_t first = (threadIdx.x % G) * N;
  if constexpr (G < LP_THREADS) {
    row = row0 + (int64_t(blockIdx.x) * LP_THREADS + threadIdx.x) / G;
    if (row >= a.rows)
      return;
  } else {
    row = row0 + blockIdx.x / chunks;
    first += (blockIdx.x % chunks) * (STEP * UNROLL);
  }
  if (G != WAVE && a.last_first)
    row = a.rows - 1 - row;
  const int64_t t = a.tok.p ? a.tok[row] : 0;
  const T m = a.stats[row], s = a.stats[a.rows + row], u = a.stats[2 * a.rows + row];
  const bool none = s == T(0) || (a.tok.p && (t == a.ignore || t < 0 || t >= a.V));
  T *dz = a.dz + row * a.dz_stride;
  if (none) {
    if (!ACC) {
#pragma unroll
      for (int c = 0; c < UNROLL; ++c) {
        const int64_t i = int64_t(first) + c * STEP;
        if (i + N <= a.V)
          RV::store(dz + i, typename RV::V{});
        else
          for (int64_t j = i; j < a.V; ++j)
            dz[j] = T(0);
      }
    }
    return;
  }
  const T inv = T(1) / s;
  const T ga = a.ga ? a.ga[row * a.sa] : T(0), gb = a.gb ? a.gb[row * a.sb] : T(0);
  // dz = p (c0 + c1 d), d = z - m, + ga at the token
  const T c0 = __builtin_elementwise_fma(gb, u / s, -ga), c1 = -gb;
  const T *z = a.z + row * a.row_stride;
#pragma unroll
  for (int c = 0; c < UNROLL; ++c) {
    const int64_t i = int64_t(first) + c * STEP;
    if (i >= a.V)
      break;
    const bool whole = i + N <= a.V;
    typename RV::V w, old = {};
    if (whole) {
      w = RV::load(z + i);
      if (ACC)
        old = RV::load(dz + i);
    } else {
      for (int j = 0; j < N; ++j) {
        w[j] = i + j < a.V ? z[i + j] : T(0);
        if (ACC)
          old[j] = i + j < a.V ? dz[i + j] : T(0);
      }
    }
    typename RV::V o;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const T d = not_below_cut(w[j] - m);
      T v = exp_of(d) * inv * __builtin_elementwise_fma(c1, d, c0);
      if (a.ga && i + j == t)
        v += ga;
      o[j] = ACC ? old[j] + v : v;
    }
    if (whole) {
      RV::store(dz + i, o);
    } else {
      for (int j = 0; j < N; ++j)
        if (i + j < a.V)
          dz[i + j] = o[j];
    }
  }
}

namespace {

// Rows of a [rows, V] view as (pointer, row stride): rows in place, elements
// of a row next to each other.
template <class T> T *row_view(const nt_view *v, int64_t &stride, const char *fname) {
  if (v->ndim != 2 || (v->shape[1] > 1 && v->strides[1] != 1))
    fail(NT_ERR_RUNTIME, std::string(fname) + ": expected rows of adjacent elements");
  stride = v->strides[0];
  return typed_ptr<T>(v);
}

template <class T>
T *out_vector(const nt_view *v, int64_t n, int dtype, const char *what) {
  if (v == nullptr)
    return nullptr;
  check_view(v, "token_logprobs");
  if (v->dtype != dtype || numel(v) != n || !is_contiguous(v))
    fail(NT_ERR_RUNTIME, std::string("token_logprobs: bad ") + what);
  return typed_ptr<T>(v);
}

// Whether logits are larger than the 256 MB of the Infinity Cache.
template <class T> bool outgrow_cache(int64_t rows, int64_t V) {
  return rows * V * int64_t(sizeof(T)) > int64_t(256) << 20;
}

template <class T> void run_forward(LpForward<T> a) {
  constexpr int CHUNK = WAVE * RowVec<T>::N * LP_UNROLL;
  const auto launch = [&](auto kernel, int threads, int64_t rows_per_block,
                          int64_t blocks_per_row) {
    const int64_t most = std::max<int64_t>(1, (int64_t(1) << 22) / blocks_per_row);
    for (int64_t r = 0; r < a.rows; r += most * rows_per_block) {
      const int64_t rows = std::min(a.rows - r, most * rows_per_block);
      const int64_t blocks = (rows + rows_per_block - 1) / rows_per_block * blocks_per_row;
      kernel<<<dim3(unsigned(blocks)), threads, 0, stream()>>>(a, r);
      NT_LAUNCH_CHECK();
    }
  };
  constexpr int SPAN = RowVec<T>::N * LP_UNROLL; // of a lane
  if (a.k == 0 && a.V <= 4 * SPAN)
    return launch(logprob_lanes_kernel<T, 4>, LP_THREADS, LP_THREADS / 4, 1);
  if (a.k == 0 && a.V <= 16 * SPAN)
    return launch(logprob_lanes_kernel<T, 16>, LP_THREADS, LP_THREADS / 16, 1);
  // A wave per row where that gives every SIMD four of them (float32, us for a
  // wave and a workgroup per row: 16384 x 3001 34 and 37, with 5 alternatives
  // 43 and 60; 8192 x 8000 43 and 41.5, 51.5 and 51), else up to two chunks.
  if (a.V <= (a.rows >= 16 * device_cu_count() ? 4 : 2) * CHUNK) {
    if (a.k)
      launch(logprob_wave_kernel<T, true>, LP_THREADS, LP_WAVES, 1);
    else
      launch(logprob_wave_kernel<T, false>, LP_THREADS, LP_WAVES, 1);
    return;
  }
  const int64_t chunks = (a.V + CHUNK - 1) / CHUNK;
  const int64_t want = std::max<int64_t>(1, 4 * device_cu_count() / a.rows);
  a.splits = int(std::min<int64_t>(want, (chunks + LP_WAVES - 1) / LP_WAVES));
  const int64_t parts = int64_t(a.splits) * LP_WAVES;
  a.part = int32_t((chunks + parts - 1) / parts * CHUNK);
  const int64_t n = a.splits > 1 ? a.rows * a.splits : 0;
  using K = typename Key<T>::K;
  DeviceScratch parts_of(size_t(n) * (3 * sizeof(T) + a.k * (sizeof(K) + sizeof(int32_t))));
  a.pm = parts_of.get<T>();
  a.ps = a.pm + n;
  a.pu = a.ps + n;
  a.pkey = reinterpret_cast<K *>(a.pu + n);
  a.ptoken = reinterpret_cast<int32_t *>(a.pkey + n * a.k);
  // Logits that outgrow the Infinity Cache are streamed past it (8192 x 32000
  // float32: 214 us without, 160 with); smaller ones stay there for the
  // backward pass (8192 x 1000: both passes 24 us, streamed 26).
  const bool stream_in = outgrow_cache<T>(a.rows, a.V);
  const auto group = [&](auto top, auto streams) {
    launch(logprob_group_kernel<T, top.value, streams.value>, LP_THREADS, 1, a.splits);
  };
  using Yes = std::true_type;
  using No = std::false_type;
  if (a.k)
    stream_in ? group(Yes{}, Yes{}) : group(Yes{}, No{});
  else
    stream_in ? group(No{}, Yes{}) : group(No{}, No{});
  if (a.splits == 1)
    return;
  if (a.k)
    launch(logprob_join_kernel<T, true>, LP_THREADS, 1, 1);
  else
    launch(logprob_join_kernel<T, false>, WAVE, 1, 1);
}

template <class T, bool ACC, int G, int UNROLL> void launch_backward(const LpBackward<T> &a) {
  constexpr int SPAN = G * RowVec<T>::N * UNROLL, PER = LP_THREADS / G; // rows at once
  const int64_t chunks = PER > 1 ? 1 : (a.V + SPAN - 1) / SPAN;
  const int64_t most = std::max<int64_t>(1, (int64_t(1) << 22) / chunks) * PER;
  for (int64_t r = 0; r < a.rows; r += most) {
    const int64_t rows = std::min(a.rows - r, most);
    logprob_bwd_kernel<T, G, UNROLL, ACC>
        <<<dim3(unsigned((rows + PER - 1) / PER * chunks)), LP_THREADS, 0, stream()>>>(
            a, r, int(chunks));
    NT_LAUNCH_CHECK();
  }
}

template <class T, bool ACC> void run_backward(LpBackward<T> a) {
  // Of logits that outgrow the Infinity Cache, what the forward pass read last
  // is still there: the backward pass begins with it, unless a wave takes a
  // row (both passes, us, rows in order and last rows first: 8192 x 32000
  // float32 with the entropy 509 and 492, 1000000 x 100 265 and 252, but 200000 x
  // 1000 476 and 487).  Smaller ones lie in the L2 of the XCD that takes the
  // same row again (8192 x 1000 18.9 and 20.4).
  a.last_first = outgrow_cache<T>(a.rows, a.V);
  constexpr int SPAN = RowVec<T>::N * LP_UNROLL; // of a lane
  if (a.V <= 4 * SPAN)
    launch_backward<T, ACC, 4, LP_UNROLL>(a);
  else if (a.V <= 16 * SPAN)
    launch_backward<T, ACC, 16, LP_UNROLL>(a);
  else if (a.V <= WAVE * SPAN)
    launch_backward<T, ACC, WAVE, LP_UNROLL>(a);
  else // 8192 x 32000 float32 takes 328 us, with one vector per lane 361, with four 347
    launch_backward<T, ACC, LP_THREADS, 2>(a);
}

void check_logits(const nt_view *z, const nt_view *tokens, const char *fname) {
  check_view(z, fname);
  if (z->ndim != 2)
    fail(NT_ERR_RUNTIME, std::string(fname) + ": logits must be [rows, V]");
  if (z->shape[1] < 1 || z->shape[1] > std::numeric_limits<int32_t>::max() - (1 << 20))
    fail(NT_ERR_VALUE, std::string(fname) + ": a row must hold 1 to 2^31 - 2^20 logits");
  if (tokens && tokens->ndim == 1 && tokens->shape[0] != z->shape[0])
    fail(NT_ERR_RUNTIME, std::string(fname) + ": one token per row");
}

} // namespace
} // namespace nt

using namespace nt;

extern "C" {

int nt_token_logprobs(const nt_view *logits, const nt_view *tokens, int64_t ignore,
                      const nt_view *logprob, const nt_view *entropy,
                      const nt_view *stats, const nt_view *top_logprobs,
                      const nt_view *top_tokens) {
  return guard([&] {
    check_logits(logits, tokens, "token_logprobs");
    const int64_t rows = logits->shape[0];
    int64_t k = 0;
    if (top_logprobs || top_tokens) {
      check_view(top_logprobs, "token_logprobs");
      check_view(top_tokens, "token_logprobs");
      if (top_logprobs->ndim != 2 || top_tokens->ndim != 2 ||
          top_logprobs->shape[1] != top_tokens->shape[1])
        fail(NT_ERR_RUNTIME, "token_logprobs: alternatives must be [rows, k]");
      k = top_logprobs->shape[1];
      if (k < 1 || k > LP_TOP_MAX || k > logits->shape[1])
        fail(NT_ERR_VALUE, "token_logprobs: 1 to 64 alternatives, at most V");
    }
    if (logprob && !tokens)
      fail(NT_ERR_RUNTIME, "token_logprobs: a log probability needs given tokens");
    dispatch_float(logits->dtype, [&]<class T>() {
      LpForward<T> a{};
      a.z = row_view<const T>(logits, a.row_stride, "token_logprobs");
      a.rows = rows;
      a.V = int32_t(logits->shape[1]);
      if (tokens)
        a.tok = token_view(tokens, "token_logprobs");
      a.ignore = ignore;
      const int dt = logits->dtype;
      a.logprob = out_vector<T>(logprob, rows, dt, "logprob");
      a.entropy = out_vector<T>(entropy, rows, dt, "entropy");
      a.stats = out_vector<T>(stats, 3 * rows, dt, "stats");
      a.top_value = out_vector<T>(k ? top_logprobs : nullptr, rows * k, dt, "top_logprobs");
      a.top_token =
          out_vector<int64_t>(k ? top_tokens : nullptr, rows * k, NT_INT64, "top_tokens");
      a.k = int(k);
      a.splits = 1;
      a.err = deferred_error_word();
      if (rows)
        run_forward(a);
    });
  });
}

int nt_token_logprobs_bwd(const nt_view *logits, const nt_view *tokens, int64_t ignore,
                          const nt_view *stats, const nt_view *g_logprob,
                          const nt_view *g_entropy, const nt_view *dlogits,
                          int32_t accumulate) {
  return guard([&] {
    check_logits(logits, tokens, "token_logprobs_bwd");
    check_view(dlogits, "token_logprobs_bwd");
    require_same_shape(logits, dlogits, "token_logprobs_bwd");
    require_same_dtype(logits, dlogits, "token_logprobs_bwd");
    const int64_t rows = logits->shape[0];
    for (const nt_view *g : {g_logprob, g_entropy}) {
      if (g == nullptr)
        continue;
      check_view(g, "token_logprobs_bwd");
      require_same_dtype(g, logits, "token_logprobs_bwd");
      if (g->ndim != 1 || g->shape[0] != rows)
        fail(NT_ERR_RUNTIME, "token_logprobs_bwd: one gradient per row");
    }
    if (g_logprob && !tokens)
      fail(NT_ERR_RUNTIME, "token_logprobs_bwd: a log probability needs given tokens");
    dispatch_float(logits->dtype, [&]<class T>() {
      LpBackward<T> a{};
      a.z = row_view<const T>(logits, a.row_stride, "token_logprobs_bwd");
      a.dz = row_view<T>(dlogits, a.dz_stride, "token_logprobs_bwd");
      a.rows = rows;
      a.V = int32_t(logits->shape[1]);
      if (tokens)
        a.tok = token_view(tokens, "token_logprobs_bwd");
      a.ignore = ignore;
      a.stats = out_vector<const T>(stats, 3 * rows, logits->dtype, "stats");
      if (a.stats == nullptr)
        fail(NT_ERR_RUNTIME, "token_logprobs_bwd: stats missing");
      if (g_logprob) {
        a.ga = typed_ptr<const T>(g_logprob);
        a.sa = g_logprob->strides[0];
      }
      if (g_entropy) {
        a.gb = typed_ptr<const T>(g_entropy);
        a.sb = g_entropy->strides[0];
      }
      if (rows == 0)
        return;
      if (accumulate)
        run_backward<T, true>(a);
      else
        run_backward<T, false>(a);
    });
  });
}

} // extern "C"

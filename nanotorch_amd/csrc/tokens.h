// What the kernels over token numbers share: reading them in either integer
// type, and vectors of 16 bytes whose address is aligned to one element only.
#pragma once

#include "nt_internal.h"

namespace nt {

// A 1-D view of int32 or int64 token numbers.
struct Tokens {
  const void *p;
  int64_t stride;
  int wide; // int64

  __device__ __forceinline__ int64_t operator[](int64_t i) const {
    return wide ? static_cast<const int64_t *>(p)[i * stride]
                : int64_t(static_cast<const int32_t *>(p)[i * stride]);
  }
};

inline Tokens token_view(const nt_view *v, const char *fname) {
  check_view(v, fname);
  if (v->dtype != NT_INT32 && v->dtype != NT_INT64)
    fail(NT_ERR_VALUE, std::string(fname) + ": tokens must be int32 or int64");
  if (v->ndim != 1)
    fail(NT_ERR_RUNTIME, std::string(fname) + ": tokens must be 1-D");
  Tokens t;
  t.wide = v->dtype == NT_INT64;
  t.stride = v->strides[0];
  t.p = static_cast<const char *>(v->data) + v->offset * (t.wide ? 8 : 4);
  return t;
}

// 16 bytes of elements.  Rows of odd length start at any element, so loads
// and stores state element alignment; gfx950 takes such a 16-byte access in
// one instruction.
template <class T> struct RowVec {
  static constexpr int N = int(16 / sizeof(T));
  typedef T V __attribute__((ext_vector_type(16 / sizeof(T))));
  typedef V U __attribute__((aligned(alignof(T))));

  template <bool STREAM = false>
  static __device__ __forceinline__ V load(const T *p) {
    if constexpr (STREAM)
      return __builtin_nontemporal_load(reinterpret_cast<const U *>(p));
    else
      return *reinterpret_cast<const U *>(p);
  }
  template <bool STREAM = false>
  static __device__ __forceinline__ void store(T *p, V v) {
    if constexpr (STREAM)
      __builtin_nontemporal_store(v, reinterpret_cast<U *>(p));
    else
      *reinterpret_cast<U *>(p) = v;
  }
};

constexpr int WAVE = 64;

} // namespace nt

// Rows of fp32 / bf16 / fp16 values as the row-wise kernels read and write them: 8 (or 1) values at a time, from an address
// that need only be aligned to the value (rows of 513 bins start anywhere; gfx950 loads 16 bytes from any address, and the
// cache lines touched are the same), arithmetic in fp32, one rounding on the way out.
#pragma once
#include "common.h"

namespace advoc {

typedef float f32x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

template <typename T>
__device__ __forceinline__ f32x8 load8(const T* p) {
  typename vec8<T>::type v;
  __builtin_memcpy(&v, p, sizeof(v));
  return __builtin_convertvector(v, f32x8);
}

// nearest, ties to even (v_cvt_pk_bf16_f32 and v_cvt_f16_f32 in the default mode)
template <typename T>
__device__ __forceinline__ void store8(T* p, f32x8 f) {
  const typename vec8<T>::type v = __builtin_convertvector(f, typename vec8<T>::type);
  __builtin_memcpy(p, &v, sizeof(v));
}

static inline int dtype_bytes(int dtype) { return dtype == ADVOC_F32 ? 4 : 2; }
static inline bool dtype_ok(int dtype) { return dtype == ADVOC_F32 || dtype == ADVOC_BF16 || dtype == ADVOC_F16; }

}  // namespace advoc

// Rows of fp32 / bf16 / fp16 values as the row-wise kernels read and write them: 8 (or 1) values at a time, from an address
// that need only be aligned to the value (rows of 513 bins start anywhere; gfx950 loads 16 bytes from any address, and the
// cache lines touched are the same), arithmetic in fp32, one rounding on the way out.
#pragma once
#include "common.h"

namespace advoc {

// N fp32 values in N registers of their own (a 256-bit vector type would tie them together)
template <int N>
struct Vals {
  float v[N];
  Vals() = default;
  __device__ __forceinline__ explicit Vals(float x) {
#pragma unroll
    for (int k = 0; k < N; ++k) v[k] = x;
  }
  __device__ __forceinline__ float& operator[](int k) { return v[k]; }
  __device__ __forceinline__ float operator[](int k) const { return v[k]; }
};
#define ADVOC_VALS_OP(OP)                                                                  \
  template <int N>                                                                         \
  __device__ __forceinline__ Vals<N> operator OP(Vals<N> a, const Vals<N>& b) {            \
    _Pragma("unroll") for (int k = 0; k < N; ++k) a.v[k] = a.v[k] OP b.v[k];               \
    return a;                                                                              \
  }                                                                                        \
  template <int N>                                                                         \
  __device__ __forceinline__ Vals<N> operator OP(Vals<N> a, float b) {                     \
    _Pragma("unroll") for (int k = 0; k < N; ++k) a.v[k] = a.v[k] OP b;                    \
    return a;                                                                              \
  }                                                                                        \
  template <int N>                                                                         \
  __device__ __forceinline__ Vals<N>& operator OP##=(Vals<N>& a, const Vals<N>& b) {       \
    _Pragma("unroll") for (int k = 0; k < N; ++k) a.v[k] = a.v[k] OP b.v[k];               \
    return a;                                                                              \
  }                                                                                        \
  template <int N>                                                                         \
  __device__ __forceinline__ Vals<N>& operator OP##=(Vals<N>& a, float b) {                \
    _Pragma("unroll") for (int k = 0; k < N; ++k) a.v[k] = a.v[k] OP b;                    \
    return a;                                                                              \
  }
ADVOC_VALS_OP(+)
ADVOC_VALS_OP(-)
ADVOC_VALS_OP(*)
#undef ADVOC_VALS_OP
typedef Vals<8> f32x8;

template <typename T>
struct vec8 {
  typedef T type __attribute__((ext_vector_type(8)));
};

// nearest, ties to even (v_cvt_pk_bf16_f32 and v_cvt_f16_f32 in the default mode)
template <typename T>
__device__ __forceinline__ void store8(T* p, const f32x8& f) {
  typename vec8<T>::type v;
#pragma unroll
  for (int k = 0; k < 8; ++k) v[k] = (T)f.v[k];
  __builtin_memcpy(p, &v, sizeof(v));
}

static inline int dtype_bytes(int dtype) { return dtype == ADVOC_F32 ? 4 : 2; }
static inline bool dtype_ok(int dtype) { return dtype == ADVOC_F32 || dtype == ADVOC_BF16 || dtype == ADVOC_F16; }

}  // namespace advoc

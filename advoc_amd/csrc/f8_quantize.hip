// 8-bit operands with a power of two per block of 128 (gfx950): rounding, and the transposed form that gradients contract over.
//
// HBM-bound: x is read once, a byte per element (and one per block) is written.  A power of two as the scale costs at most one bit
// of a block's range -- none of its precision, the formats being floating -- and makes the scaling exact, so what is rounded is x
// itself, once; the matrix instruction of gfx950 takes such scales as they are.
#include "rows.h"

namespace {

constexpr int kBlock = 128;

__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) { return a > b ? a : b; }
constexpr uint32_t kInfinity = 0x7f800000u;

// Largest finite magnitude of N values, as its bits (which order like the values); get(i) gives a value.  Infinities and NaN order
// above everything finite: only where the largest is one of them are the values looked at again.
template <int N, typename F>
__device__ __forceinline__ uint32_t largest_finite(F&& get) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < N; ++i) m = larger(m, magnitude(get(i)));
  if (m >= kInfinity) {
    m = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t b = magnitude(get(i));
      if (b < kInfinity) m = larger(m, b);
    }
  }
  return m;
}

// Largest over 16 consecutive lanes, within rows of 16 by lane moves that come with the comparison
template <int CTRL>
__device__ __forceinline__ uint32_t larger_moved(uint32_t m) {
  return larger(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ uint32_t largest16(uint32_t m) {
  m = larger_moved<0xB1>(m);               // quad_perm 1 0 3 2
  m = larger_moved<0x4E>(m);               // quad_perm 2 3 0 1
  m = larger_moved<0x141>(m);              // row_half_mirror
  return larger_moved<0x140>(m);           // row_mirror
}
// Largest over the four lanes of a wave that have their place in a row of 16
__device__ __forceinline__ uint32_t largest_rows(uint32_t m) {
  const auto a = __builtin_amdgcn_permlane16_swap(m, m, false, false);
  m = larger(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(m, m, false, false);
  return larger(b[0], b[1]);
}

// exponent byte of a block: the format's largest value is 1.75 * 2^8 (E4M3) or 1.75 * 2^15 (E5M2), and 1.75 is 0x600000 of
// mantissa; 1 (2^-126) is the smallest that is used
template <int FMT>
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 23) - (FMT == ADVOC_E4M3 ? 8 : 15) + ((amax & 0x7fffffu) > 0x600000u);
  return e < 1 ? 1 : e;
}
__device__ __forceinline__ float scale_value(int byte) { return __uint_as_float((uint32_t)byte << 23); }

// four values over a power of two to four bytes
typedef short short2v __attribute__((ext_vector_type(2)));
template <int FMT>
__device__ __forceinline__ int pack4(float a, float b, float c, float d, float scale) {
  short2v w = {0, 0};
  if constexpr (FMT == ADVOC_E4M3) {
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, a, b, scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, c, d, scale, true);
  } else {
    w = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(w, a, b, scale, false);
    w = __builtin_amdgcn_cvt_scalef32_pk_bf8_f32(w, c, d, scale, true);
  }
  return __builtin_bit_cast(int, w);
}

// eight values as they lie in memory, zeros behind the row's end
template <typename T>
struct Eight {
  typename advoc::vec8<T>::type v;
  __device__ __forceinline__ void load(const T* row, int64_t col, int64_t cols) {
    if (col + 8 <= cols) {
      __builtin_memcpy(&v, row + col, sizeof(v));
      return;
    }
    for (int k = 0; k < 8; ++k) v[k] = col + k < cols ? row[col + k] : (T)0.f;
  }
  __device__ __forceinline__ float operator[](int k) const { return (float)v[k]; }
  // (the compiler would keep 16-bit values converted from one use to the next, in twice the registers)
  __device__ __forceinline__ void forget_converted() {
    if constexpr (sizeof(T) == 2) {
      int w[4];
      __builtin_memcpy(w, &v, sizeof(w));
#pragma unroll
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(w[i]));
      __builtin_memcpy(&v, w, sizeof(w));
    }
  }
};

struct Args {
  const void* x;
  int64_t pitch, rows, cols;
  uint8_t *q, *scale, *qt, *scale_t;
  int64_t kp, sp, mp, sp_t;      // row pitches of the outputs
};

// Blocks of rows: 16 lanes x 8 values are a block.  16384 x 4096 bf16 (202 MB): 44 us, 4.6 TB/s; adding 1 to as much takes 36.
template <typename T, int FMT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(Args a) {
  const int sub = threadIdx.x & 15;
  const uint32_t per_row = (uint32_t)(a.kp / kBlock), total = (uint32_t)a.rows * per_row;
  for (uint32_t b = blockIdx.x * 16u + (threadIdx.x >> 4); b < total; b += gridDim.x * 16u) {
    const uint32_t row = b / per_row, kb = b - row * per_row;
    const int64_t col = (int64_t)kb * kBlock + sub * 8;
    Eight<T> v;
    v.load((const T*)a.x + row * a.pitch, col, a.cols);
    const int byte = scale_byte<FMT>(largest16(largest_finite<8>([&](int k) { return v[k]; })));
    const float s = scale_value(byte);
    *reinterpret_cast<int2*>(a.q + row * a.kp + col) =
        make_int2(pack4<FMT>(v[0], v[1], v[2], v[3], s), pack4<FMT>(v[4], v[5], v[6], v[7], s));
    if (sub == 0) {
      uint8_t* out = a.scale + row * a.sp;
      out[kb] = (uint8_t)byte;
      if (kb + 1 == per_row)
        for (int64_t k = per_row; k < a.sp; ++k) out[k] = 0;
    }
  }
}

// A tile of 128 rows x 128 columns per workgroup: thread (rg, cg) holds rows 8 rg .. + 7, columns 8 cg .. + 7.  A column's largest
// magnitude meets over 4 lanes and, in LDS, over the 4 waves; the bytes of a column are turned around through LDS and leave as whole
// 128-byte lines.  ROWS: the row blocks of the same tile as well, from the same registers.
// Bound by HBM and by the load, arithmetic and store of one round of workgroups not overlapping: 16384 x 1024 bf16, both forms, in
// 17 us (67 MB, 3.9 TB/s; adding 1 to as much takes 11, or 14 where no cache holds it).  What it took from 24: the largest magnitude
// as an integer maximum that looks at infinities only where there are any, lanes met by moves instead of LDS, the division by the
// scale inside the conversion, the turned bytes without bank conflicts, 65 registers instead of 167 (four workgroups to a CU).
template <typename T, int FMT, bool ROWS>
__global__ __launch_bounds__(256, 4) void quantize_tile_kernel(Args a) {
  __shared__ __align__(16) uint32_t cm[4][kBlock];
  __shared__ __align__(16) uint8_t turn[kBlock * kBlock];            // a column's 16-byte pieces at piece ^ (column / 8 % 8)
  const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4, wave = tid >> 6;
  const int64_t r0 = (int64_t)blockIdx.x * kBlock, c0 = (int64_t)blockIdx.y * kBlock;
  Eight<T> v[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int64_t row = r0 + rg * 8 + t;
    if (row < a.rows) {
      v[t].load((const T*)a.x + row * a.pitch, c0 + cg * 8, a.cols);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[t].v[k] = (T)0.f;
    }
  }
  if constexpr (ROWS) {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int byte = scale_byte<FMT>(largest16(largest_finite<8>([&](int k) { return v[t][k]; })));
      const int64_t row = r0 + rg * 8 + t;
      if (row >= a.rows) continue;
      const float s = scale_value(byte);
      *reinterpret_cast<int2*>(a.q + row * a.kp + c0 + cg * 8) =
          make_int2(pack4<FMT>(v[t][0], v[t][1], v[t][2], v[t][3], s), pack4<FMT>(v[t][4], v[t][5], v[t][6], v[t][7], s));
      if (cg == 0) {
        uint8_t* out = a.scale + row * a.sp;
        out[blockIdx.y] = (uint8_t)byte;
        if (blockIdx.y + 1 == gridDim.y)
          for (int64_t k = gridDim.y; k < a.sp; ++k) out[k] = 0;
      }
    }
  }
#pragma unroll
  for (int t = 0; t < 8; ++t) v[t].forget_converted();
  uint32_t m[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) m[k] = largest_rows(largest_finite<8>([&](int t) { return v[t][k]; }));
  if ((tid & 63) < 16) {
    *reinterpret_cast<uint4*>(&cm[wave][cg * 8]) = make_uint4(m[0], m[1], m[2], m[3]);
    *reinterpret_cast<uint4*>(&cm[wave][cg * 8 + 4]) = make_uint4(m[4], m[5], m[6], m[7]);
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int c = cg * 8 + k;
    const int byte = scale_byte<FMT>(larger(larger(cm[0][c], cm[1][c]), larger(cm[2][c], cm[3][c])));
    const float s = scale_value(byte);
    *reinterpret_cast<int2*>(turn + c * kBlock + (((rg >> 1) ^ (cg & 7)) << 4) + (rg & 1) * 8) =
        make_int2(pack4<FMT>(v[0][k], v[1][k], v[2][k], v[3][k], s), pack4<FMT>(v[4][k], v[5][k], v[6][k], v[7][k], s));
    if (rg == 0 && c0 + c < a.cols) {
      uint8_t* out = a.scale_t + (c0 + c) * a.sp_t;
      out[blockIdx.x] = (uint8_t)byte;
      if (blockIdx.x + 1 == gridDim.x)
        for (int64_t i = gridDim.x; i < a.sp_t; ++i) out[i] = 0;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kBlock * kBlock / 16 / 256; ++i) {
    const int idx = i * 256 + tid, c = idx >> 3, p = (idx & 7) * 16;
    if (c0 + c < a.cols)
      *reinterpret_cast<int4*>(a.qt + (c0 + c) * a.mp + r0 + p) = *reinterpret_cast<const int4*>(turn + c * kBlock + (p ^ ((c >> 3 & 7) << 4)));
  }
}

template <typename T, int FMT>
void launch(const Args& a, hipStream_t stream) {
  if (!a.qt) {
    int64_t blocks = advoc::ceil_div(a.rows * (a.kp / kBlock), 16);
    if (blocks > 256 * 16) blocks = 256 * 16;
    hipLaunchKernelGGL((quantize_rows_kernel<T, FMT>), dim3((unsigned)blocks), dim3(256), 0, stream, a);
    return;
  }
  const dim3 grid((unsigned)(a.mp / kBlock), (unsigned)(a.kp / kBlock));
  if (a.q)
    hipLaunchKernelGGL((quantize_tile_kernel<T, FMT, true>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((quantize_tile_kernel<T, FMT, false>), grid, dim3(256), 0, stream, a);
}

template <typename T>
void launch_format(const Args& a, int format, hipStream_t stream) {
  if (format == ADVOC_E4M3) launch<T, ADVOC_E4M3>(a, stream);
  else launch<T, ADVOC_E5M2>(a, stream);
}

int64_t up(int64_t v, int64_t to) { return advoc::ceil_div(v, to) * to; }

}  // namespace

extern "C" int advoc_f8_quantize(const void* x, int64_t x_pitch, int64_t rows, int64_t cols, int32_t dtype, int32_t format,
                                 uint8_t* q, uint8_t* scale, uint8_t* qt, uint8_t* scale_t, advoc_stream_t stream) {
  if (rows < 0 || cols < 0) return ADVOC_ERR_BAD_SHAPE;
  if (rows == 0 || cols == 0) return ADVOC_OK;
  if (!x || (!q && !qt) || (q && !scale) || (qt && !scale_t)) return ADVOC_ERR_NULL;
  if (rows > 1 && x_pitch < cols) return ADVOC_ERR_BAD_SHAPE;
  if (!advoc::dtype_ok(dtype) || (format != ADVOC_E4M3 && format != ADVOC_E5M2)) return ADVOC_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(qt)) & 15) return ADVOC_ERR_UNSUPPORTED;
  // 31-bit block numbers, and 2^16 column blocks in a grid's second dimension
  if (rows > (1LL << 37) / cols || rows > 0x7fffff00LL || cols > 128LL * 65535) return ADVOC_ERR_UNSUPPORTED;
  if (rows * advoc::ceil_div(cols, kBlock) > 0x7fffffffLL) return ADVOC_ERR_UNSUPPORTED;
  const int64_t kp = up(cols, kBlock), mp = up(rows, kBlock);
  const Args a = {x, x_pitch, rows, cols, q, scale, qt, scale_t, kp, up(kp / kBlock, 4), mp, up(mp / kBlock, 4)};
  ADVOC_CLEAR_LAUNCH_ERROR();
  if (dtype == ADVOC_F32)
    launch_format<float>(a, format, advoc::as_stream(stream));
  else if (dtype == ADVOC_BF16)
    launch_format<__bf16>(a, format, advoc::as_stream(stream));
  else
    launch_format<_Float16>(a, format, advoc::as_stream(stream));
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

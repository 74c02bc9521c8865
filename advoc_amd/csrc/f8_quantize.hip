// 8-bit operands with a power of two per block of 128 (gfx950): rounding, and the transposed form that gradients contract over.
//
// HBM-bound: x is read once, a byte per element (and one per block) is written.  A power of two as the scale costs at most one bit
// of a block's range -- none of its precision, the formats being floating -- and makes the scaling exact, so what is rounded is x
// itself, once; the matrix instruction of gfx950 takes such scales as they are.
#include "rows.h"

namespace {

using advoc::f32x8;

constexpr int kBlock = 128;

// largest finite magnitude so far, as its bits (which order like the values)
__device__ __forceinline__ uint32_t amax_bits(uint32_t m, float v) {
  const uint32_t b = __float_as_uint(v) & 0x7fffffffu;
  return b < 0x7f800000u && b > m ? b : m;
}

// exponent byte of a block: the format's largest value is 1.75 * 2^8 (E4M3) or 1.75 * 2^15 (E5M2), and 1.75 is 0x600000 of
// mantissa; 1 (2^-126) is the smallest that is used
template <int FMT>
__device__ __forceinline__ int scale_byte(uint32_t amax) {
  const int e = (int)(amax >> 23) - (FMT == ADVOC_E4M3 ? 8 : 15) + ((amax & 0x7fffffu) > 0x600000u);
  return e < 1 ? 1 : e;
}
__device__ __forceinline__ float inverse_scale(int byte) { return __uint_as_float((uint32_t)(254 - byte) << 23); }

// four values to four bytes
template <int FMT>
__device__ __forceinline__ int pack4(float a, float b, float c, float d) {
  int w = 0;
  if constexpr (FMT == ADVOC_E4M3) {
    w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
  } else {
    w = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, w, false);
    w = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, w, true);
  }
  return w;
}

template <typename T>
__device__ __forceinline__ f32x8 load_cols(const T* row, int64_t col, int64_t cols) {
  if (col + 8 <= cols) return advoc::load8(row + col);
  f32x8 v = (f32x8)(0.f);
  for (int k = 0; k < 8; ++k)
    if (col + k < cols) v[k] = (float)row[col + k];
  return v;
}

struct Args {
  const void* x;
  int64_t pitch, rows, cols;
  uint8_t *q, *scale, *qt, *scale_t;
  int64_t kp, sp, mp, sp_t;      // row pitches of the outputs
};

// Blocks of rows: 16 lanes x 8 values are a block
template <typename T, int FMT>
__global__ __launch_bounds__(256) void quantize_rows_kernel(Args a) {
  const int sub = threadIdx.x & 15;
  const uint32_t per_row = (uint32_t)(a.kp / kBlock), total = (uint32_t)a.rows * per_row;
  for (uint32_t b = blockIdx.x * 16u + (threadIdx.x >> 4); b < total; b += gridDim.x * 16u) {
    const uint32_t row = b / per_row, kb = b - row * per_row;
    const int64_t col = (int64_t)kb * kBlock + sub * 8;
    const f32x8 v = load_cols((const T*)a.x + row * a.pitch, col, a.cols);
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) m = amax_bits(m, v[k]);
#pragma unroll
    for (int off = 8; off > 0; off >>= 1) {
      const uint32_t o = __shfl_xor(m, off, 64);
      m = o > m ? o : m;
    }
    const int byte = scale_byte<FMT>(m);
    const f32x8 s = v * inverse_scale(byte);
    *reinterpret_cast<int2*>(a.q + row * a.kp + col) =
        make_int2(pack4<FMT>(s[0], s[1], s[2], s[3]), pack4<FMT>(s[4], s[5], s[6], s[7]));
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
template <typename T, int FMT, bool ROWS>
__global__ __launch_bounds__(256) void quantize_tile_kernel(Args a) {
  constexpr int kPitch = kBlock + 16;
  __shared__ uint32_t cm[4][kBlock];
  __shared__ __align__(16) uint8_t turn[kBlock * kPitch];
  const int tid = threadIdx.x, cg = tid & 15, rg = tid >> 4, wave = tid >> 6;
  const int64_t r0 = (int64_t)blockIdx.x * kBlock, c0 = (int64_t)blockIdx.y * kBlock;
  f32x8 v[8];
#pragma unroll
  for (int t = 0; t < 8; ++t) {
    const int64_t row = r0 + rg * 8 + t;
    v[t] = (f32x8)(0.f);
    if (row < a.rows) v[t] = load_cols((const T*)a.x + row * a.pitch, c0 + cg * 8, a.cols);
  }
  uint32_t m[8] = {};
#pragma unroll
  for (int t = 0; t < 8; ++t)
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = amax_bits(m[k], v[t][k]);
#pragma unroll
  for (int k = 0; k < 8; ++k) {
#pragma unroll
    for (int off = 16; off < 64; off <<= 1) {
      const uint32_t o = __shfl_xor(m[k], off, 64);
      m[k] = o > m[k] ? o : m[k];
    }
    if ((tid & 63) < 16) cm[wave][cg * 8 + k] = m[k];
  }
  if constexpr (ROWS) {
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      uint32_t rm = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) rm = amax_bits(rm, v[t][k]);
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) {
        const uint32_t o = __shfl_xor(rm, off, 64);
        rm = o > rm ? o : rm;
      }
      const int64_t row = r0 + rg * 8 + t;
      if (row >= a.rows) continue;
      const int byte = scale_byte<FMT>(rm);
      const f32x8 s = v[t] * inverse_scale(byte);
      *reinterpret_cast<int2*>(a.q + row * a.kp + c0 + cg * 8) =
          make_int2(pack4<FMT>(s[0], s[1], s[2], s[3]), pack4<FMT>(s[4], s[5], s[6], s[7]));
      if (cg == 0) {
        uint8_t* out = a.scale + row * a.sp;
        out[blockIdx.y] = (uint8_t)byte;
        if (blockIdx.y + 1 == gridDim.y)
          for (int64_t k = gridDim.y; k < a.sp; ++k) out[k] = 0;
      }
    }
  }
  __syncthreads();
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    const int c = cg * 8 + k;
    uint32_t top = cm[0][c];
#pragma unroll
    for (int w = 1; w < 4; ++w) top = cm[w][c] > top ? cm[w][c] : top;
    const int byte = scale_byte<FMT>(top);
    const float s = inverse_scale(byte);
    *reinterpret_cast<int2*>(turn + c * kPitch + rg * 8) =
        make_int2(pack4<FMT>(v[0][k] * s, v[1][k] * s, v[2][k] * s, v[3][k] * s),
                  pack4<FMT>(v[4][k] * s, v[5][k] * s, v[6][k] * s, v[7][k] * s));
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
      *reinterpret_cast<int4*>(a.qt + (c0 + c) * a.mp + r0 + p) = *reinterpret_cast<const int4*>(turn + c * kPitch + p);
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

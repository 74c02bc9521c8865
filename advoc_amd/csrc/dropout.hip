// Dropout whose mask is never stored (gfx950): y_i = x_i / keep where word i of the Philox stream (philox.h) is kept, exactly 0
// elsewhere whatever x_i holds; the gradient is the same call on dy.  Reads and writes each element once: no byte of mask in
// HBM, and the backward pass draws the same words again.  HBM-bound: 65536 x 1024 bf16 (268 MB) in 43 us, 6.2 TB/s (adding 1
// to as much: 46 to 48 us; 45 with the loads behind the drawing); 8192 x 513 fp16 in padded rows 8.4, one round of workgroups; one frame takes the 6.6 us of a
// call.
#include "philox.h"
#include "rows.h"

namespace {

using advoc::DropKey;
using advoc::f32x8;

constexpr int kThreads = 256, kPer = 8;              // a thread's chunk: 8 consecutive elements = two Philox blocks

struct Args {
  const void* x;
  void* y;
  int64_t n, x_pitch, y_pitch;
  uint32_t cols;
  DropKey key;
};

// PITCHED: rows of `cols` elements with a distance of their own; otherwise the n elements are one run.  The index that is
// drawn for is the logical one (row * cols + column), so a tensor and its padded copy drop the same elements.
template <typename T, bool PITCHED>
__global__ __launch_bounds__(kThreads) void dropout_kernel(Args a) {
  const uint2 key = advoc::drop_key_words(a.key);
  const uint32_t thresh = a.key.thresh;
  const float scale = a.key.scale;
  const int64_t base = (int64_t)blockIdx.x * (kThreads * kPer);      // a multiple of 4, as the offset is
  const int64_t i = base + threadIdx.x * kPer;
  if (i >= a.n) return;
  const T* x = (const T*)a.x;
  T* y = (T*)a.y;
  uint32_t col = 0;
  if constexpr (PITCHED) {
    const uint64_t row0 = (uint64_t)base / a.cols;                   // uniform: one 64-bit division per workgroup
    const uint32_t off = (uint32_t)((uint64_t)base - row0 * a.cols) + threadIdx.x * kPer;
    const uint32_t r = off / a.cols;
    col = off - r * a.cols;
    x += (int64_t)(row0 + r) * a.x_pitch + col;
    y += (int64_t)(row0 + r) * a.y_pitch + col;
  } else {
    x += i;
    y += i;
  }
  // A chunk in which a row or the tensor ends (one in a wave for rows of 513) goes by elements.  Loads first, all of them in flight
  // while the words are drawn.
  const bool whole = i + kPer <= a.n && (!PITCHED || col + kPer <= a.cols);
  typename advoc::vec8<T>::type v;
  T* to[kPer];
  if (whole) {
    __builtin_memcpy(&v, x, sizeof(v));
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      to[k] = y;
      v[k] = *x;
      if (i + k + 1 >= a.n) continue;           // (behind the last element: that one again, not stored)
      ++x, ++y;
      if (PITCHED && ++col == a.cols) {
        col = 0;
        x += a.x_pitch - a.cols;
        y += a.y_pitch - a.cols;
      }
    }
  }
  uint32_t words[kPer] = {};
  if (thresh) advoc::drop_words<kPer>(words, a.key.offset + (uint64_t)i, true, key);
  f32x8 o;
#pragma unroll
  for (int k = 0; k < kPer; ++k) o[k] = words[k] >= thresh ? (float)v[k] * scale : 0.f;
  if (whole) {
    advoc::store8(y, o);
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k)
      if (i + k < a.n) *to[k] = (T)o[k];
  }
}

template <typename T>
void launch(const Args& a, bool pitched, hipStream_t stream) {
  const dim3 grid((unsigned)advoc::ceil_div(a.n, kThreads * kPer));
  if (pitched)
    hipLaunchKernelGGL((dropout_kernel<T, true>), grid, dim3(kThreads), 0, stream, a);
  else
    hipLaunchKernelGGL((dropout_kernel<T, false>), grid, dim3(kThreads), 0, stream, a);
}

}  // namespace

extern "C" int advoc_dropout(const void* x, int64_t x_pitch, void* y, int64_t y_pitch, int64_t rows, int64_t cols, int32_t dtype,
                             float keep_prob, uint64_t seed, uint64_t offset, const uint64_t* seed_dev, advoc_stream_t stream) {
  if (rows < 0 || cols < 0 || !(keep_prob > 0.f && keep_prob <= 1.f)) return ADVOC_ERR_BAD_SHAPE;
  if (rows == 0 || cols == 0) return ADVOC_OK;
  if (!x || !y) return ADVOC_ERR_NULL;
  if (rows > 1 && (x_pitch < cols || y_pitch < cols)) return ADVOC_ERR_BAD_SHAPE;
  if (!advoc::dtype_ok(dtype) || (offset & 3)) return ADVOC_ERR_UNSUPPORTED;
  if (cols > 0x7fffffffLL - 2 * kThreads * kPer && rows > 1 && (x_pitch != cols || y_pitch != cols)) return ADVOC_ERR_UNSUPPORTED;
  // a launch ends at 2^32 - 1 work-items of 8 elements
  if (rows > ((1LL << 35) - kThreads * kPer) / cols) return ADVOC_ERR_UNSUPPORTED;
  const bool pitched = rows > 1 && (x_pitch != cols || y_pitch != cols);
  Args a = {x, y, rows * cols, x_pitch, y_pitch, pitched ? (uint32_t)cols : 0u,
            advoc::make_drop_key(keep_prob, seed, offset, seed_dev)};
  ADVOC_CLEAR_LAUNCH_ERROR();
  if (dtype == ADVOC_F32)
    launch<float>(a, pitched, advoc::as_stream(stream));
  else if (dtype == ADVOC_BF16)
    launch<__bf16>(a, pitched, advoc::as_stream(stream));
  else
    launch<_Float16>(a, pitched, advoc::as_stream(stream));
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

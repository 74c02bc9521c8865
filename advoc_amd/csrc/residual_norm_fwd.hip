// Forward pass of the residual norm (gfx950): the norm behind a block, its gate, residual scale and dropout, the residual sum and
// the norm before the next block in one pass over the rows (residual_norm.h).  HBM-bound: h, x and the gate are read once, r and
// z written once; the mask is drawn, not read.
//
// The variance of a LAYER norm is the mean of (a - mean)^2, taken from the registers in a second sum: sum a^2 - n mean^2 would
// lose what matters for rows whose mean is large against their spread.  r is rounded when it is stored; z and the statistics are
// those of the unrounded r.
#include "residual_norm.h"

namespace {

using advoc::f32x8;
using advoc::NormArgs;
using advoc::Team;

// mean and 1 / sqrt(var + eps) of a row
template <int V, int L, int NV, int WG>
__device__ __forceinline__ void row_stats(const f32x8 (&a)[NV], const int (&dup)[NV], bool ragged, int kind, float inv_cols, float eps,
                                          float* red, int& turn, float& mean, float& rstd) {
  mean = 0.f;
  float none = 0.f;
  if (kind == ADVOC_NORM_LAYER) {
    mean = advoc::own_sum<V>(dup, ragged, [&](int j, int k) { return a[j][k]; });
    Team<L, WG>::sum2(mean, none, red, turn);
    mean *= inv_cols;
  }
  float sq = advoc::own_sum<V>(dup, ragged, [&](int j, int k) {
    const float d = a[j][k] - mean;
    return d * d;
  });
  Team<L, WG>::sum2(sq, none, red, turn);
  rstd = 1.f / sqrtf(sq * inv_cols + eps);
}

template <typename T, typename R, int V, int L, int NV, int WG>
__global__ __launch_bounds__(WG) void norm_forward_kernel(NormArgs a) {
  using Row = Team<L, WG>;
  __shared__ float red[L > 64 ? 4 * (L / 64) : 1];
  int turn = 0;
  const int lane = Row::lane();
  const uint2 key = advoc::drop_key_words(a.key);
  const bool aligned = (a.cols & 3) == 0, ragged = a.cols % V != 0;
  int col[NV], dup[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) advoc::chunk_place<V, L>(j, lane, a.cols, col[j], dup[j]);
  // a workgroup-wide row must take every lane through the same number of rows (the sums meet at barriers)
  for (int64_t row = (int64_t)blockIdx.x * Row::kRows + (L > 64 ? 0 : Row::slot()); row < a.rows;
       row += (int64_t)gridDim.x * Row::kRows) {
    f32x8 r[NV], u[NV], g[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
        r[j] = advoc::load_chunk<V>((const R*)a.x + row * a.x_pitch + col[j]);
        if (a.h) u[j] = advoc::load_chunk<V>((const T*)a.h + row * a.h_pitch + col[j]);
        if (a.gate) g[j] = advoc::load_chunk<V>((const T*)a.gate + (int64_t)((uint32_t)row / (uint32_t)a.gate_group) * a.gate_pitch + col[j]);
      }
    if constexpr (L > 64) __syncthreads();      // outputs may be the inputs' own buffers, and a column may have two holders
    float mean0 = 0.f, rstd0 = 0.f, mean1 = 0.f, rstd1 = 0.f;
    if (a.h) {
      if (a.post != ADVOC_NORM_NONE) row_stats<V, L, NV, WG>(u, dup, ragged, a.post, a.inv_cols, a.eps, red, turn, mean0, rstd0);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (a.post != ADVOC_NORM_NONE) {
          const f32x8 w = advoc::cols_chunk<V>(a.w_post, col[j], 1.f), b = advoc::cols_chunk<V>(a.b_post, col[j], 0.f);
          u[j] = (u[j] - mean0) * rstd0 * w + b;
        }
        const uint32_t keep = advoc::keep_chunk<V>(a.key.offset + (uint64_t)(row * a.cols + col[j]), aligned, key, a.key.thresh);
        f32x8 s = advoc::cols_chunk<V>(a.scale, col[j], 1.f) * a.alpha;
        if (a.gate) {
          advoc::activate<V>(g[j], a.act);
          s *= g[j];
        }
#pragma unroll
        for (int k = 0; k < V; ++k) r[j][k] += s[k] * ((keep >> k & 1) ? u[j][k] * a.key.scale : 0.f);
        advoc::store_chunk<V>((R*)a.r + row * a.r_pitch + col[j], r[j]);
      }
    }
    if (a.pre != ADVOC_NORM_NONE) {
      row_stats<V, L, NV, WG>(r, dup, ragged, a.pre, a.inv_cols, a.eps, red, turn, mean1, rstd1);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const f32x8 w = advoc::cols_chunk<V>(a.w_pre, col[j], 1.f), b = advoc::cols_chunk<V>(a.b_pre, col[j], 0.f);
        advoc::store_chunk<V>((T*)a.z + row * a.z_pitch + col[j], (r[j] - mean1) * rstd1 * w + b);
      }
    }
    if (a.stats && lane == 0) a.stats[row] = make_float4(mean0, rstd0, mean1, rstd1);
  }
}

template <typename T, typename R>
struct Launch {
  const NormArgs& a;
  hipStream_t stream;
  template <int V, int L, int NV, int WG>
  void run() const {
    int64_t blocks = advoc::ceil_div(a.rows, Team<L, WG>::kRows);
    const int64_t most = 256 * (2048 / WG);      // every resident workgroup of the chip, then rows in turn
    if (blocks > most) blocks = most;
    hipLaunchKernelGGL((norm_forward_kernel<T, R, V, L, NV, WG>), dim3((unsigned)blocks), dim3(WG), 0, stream, a);
  }
};

}  // namespace

namespace advoc {

bool launch_norm_forward(const NormArgs& a, int dtype, int res_dtype, hipStream_t stream) {
  if (dtype == ADVOC_F32) return norm_dispatch(a.cols, Launch<float, float>{a, stream});
  if (dtype == ADVOC_BF16)
    return res_dtype == ADVOC_F32 ? norm_dispatch(a.cols, Launch<__bf16, float>{a, stream})
                                  : norm_dispatch(a.cols, Launch<__bf16, __bf16>{a, stream});
  return res_dtype == ADVOC_F32 ? norm_dispatch(a.cols, Launch<_Float16, float>{a, stream})
                                : norm_dispatch(a.cols, Launch<_Float16, _Float16>{a, stream});
}

}  // namespace advoc

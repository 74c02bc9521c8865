// Forward pass of the residual norm (gfx950): the norm behind a block, its gate, residual scale and dropout, the residual sum and
// the norm before the next block in one pass over the rows (residual_norm.h).  HBM-bound: h, x and the gate are read once, r and
// z written once; the mask is drawn, not read.
//
// The variance of a LAYER norm is the mean of (a - mean)^2, taken from the registers in a second sum: sum a^2 - n mean^2 would
// lose what matters for rows whose mean is large against their spread.  r is rounded when it is stored; z and the statistics are
// those of the unrounded r.
#include "residual_norm.h"

namespace {

using advoc::NormArgs;
using advoc::Team;
using advoc::Vals;

// mean and 1 / sqrt(var + eps) of a row
template <int V, int L, int NV, int WG>
__device__ __forceinline__ void row_stats(const Vals<V> (&a)[NV], const int (&dup)[NV], bool ragged, int kind, float inv_cols, float eps,
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

// Vectors in LDS: five, and four where a row is a workgroup's: five of 2048 or 4096 columns and the sums' place are more than a CU's
// 160 KB over the workgroups that its waves allow, and one of those then waits for a round of its own (8192 x 2048 bf16: 50 us, four
// vectors 45; 4096 x 4096 fp16: 39, 33; with five vectors and the launch cut to what fits 44 and 35).  There a lane
// holds its part of b_pre in registers; with 16 columns a lane it reads it for each row.
template <int L>
constexpr int kVectors = L > 64 ? 4 : 5;

constexpr int kWavesPerSimd = 4, kCuLds = 160 * 1024;
// LDS that a workgroup takes, in the 1280 bytes that a CU gives out
template <int V, int L>
constexpr int lds_taken(int cols) {
  const int bytes = 4 * kVectors<L> * ((cols + V - 1) / V * V + 3) + 4 * (L > 64 ? 4 * (L / 64) : 1);
  return (bytes + 1279) / 1280 * 1280;
}

// H: there is a block output; PRE: there is a pre norm.  Nothing else that may be absent is a branch around memory: an absent gate is
// read from where h lies and replaced by ones.
// Four waves to a SIMD, 128 registers to a lane.  With 8 columns a lane the next row's loads are in flight while a row is computed
// (measured with five vectors: 8192 x 2048 50 us, without 55; 4096 x 4096 50, without 62); with 16 they would spill (16384 x 1024: 38
// us, with them 65).  A wave waits for its loads and stores in the order of their issue, so that the number of stores behind the loads
// is to be known where the loads are waited for: hence the templates.
// 16384 x 1024, bf16 with fp32 residuals, a gate per clip, dropout (202 MB): 36.6 us, 5.5 TB/s (adding 1 to as much: 36.4).  Rows of a
// whole workgroup meet four times on their way: 4096 x 4096 in the same types 50 us, 4.0 TB/s, 8192 x 2048 48.  16384 x 513: 25 us, 4.0
// TB/s, bound by arithmetic (rows at odd offsets, three Philox blocks for nine words).  One row: 3 us, latency.
template <typename T, typename R, int V, int L, int NV, int WG, bool H, bool PRE>
__global__ __launch_bounds__(WG, kWavesPerSimd) void norm_forward_kernel(NormArgs a) {
  using Row = Team<L, WG>;
  extern __shared__ __align__(16) float vec[];  // scale, w_post, b_post, w_pre and, where kFive, b_pre
  constexpr bool kAhead = NV == 1;
  constexpr bool kFive = kVectors<L> == 5, kHeld = !kFive && NV == 1;
  __shared__ float red[L > 64 ? 4 * (L / 64) : 1];
  int turn = 0;
  const int lane = Row::lane(), cols = a.cols;
  const uint2 key = advoc::drop_key_words(a.key);
  const bool aligned = (cols & 3) == 0, ragged = cols % V != 0, has_gate = a.gate, post = a.post != ADVOC_NORM_NONE;
  const void* gate_base = has_gate ? a.gate : a.h;
  const int64_t gate_pitch = has_gate ? a.gate_pitch : a.h_pitch;
  const uint32_t gate_group = has_gate ? (uint32_t)a.gate_group : 1u;
  int chunk[NV], col[NV], dup[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) advoc::chunk_place<V, L>(j, lane, cols, chunk[j], col[j], dup[j]);

  const advoc::Chunks<V> chunks(cols);
  const int floats = chunks.floats();
  advoc::Raw<T, V, NV> h, gate;
  advoc::Raw<R, V, NV> x;
  auto load = [&](int64_t row) {
    if (row >= a.rows) row = a.rows - 1;        // (the lanes of a wave leave the loop together)
    x.load(a.x, row * a.x_pitch, col);
    if constexpr (H) {
      h.load(a.h, row * a.h_pitch, col);
      gate.load(gate_base, (int64_t)((uint32_t)row / gate_group) * gate_pitch, col);
    }
  };
  const int64_t step = (int64_t)gridDim.x * Row::kRows;
  const float kept = a.alpha * a.key.scale;
  int64_t row = (int64_t)blockIdx.x * Row::kRows + Row::slot();
  if constexpr (kAhead) load(row);
  if constexpr (kFive)
    advoc::stage_vectors<WG, V, 5>(vec, {a.scale, a.w_post, a.b_post, a.w_pre, a.b_pre}, {1.f, 1.f, 0.f, 1.f, 0.f}, cols);
  else
    advoc::stage_vectors<WG, V, 4>(vec, {a.scale, a.w_post, a.b_post, a.w_pre}, {1.f, 1.f, 0.f, 1.f}, cols);
  Row::meet();
  Vals<V> b_pre(0.f);
  if constexpr (kHeld && PRE)
    if (a.b_pre) b_pre = advoc::floats_at<V>(a.b_pre + col[0]);
  for (; row < a.rows; row += step) {
    advoc::forget_lds();
    if constexpr (!kAhead) load(row);
    if constexpr (L > 64) {                     // outputs may be the inputs' own buffers, and a column may have two holders
      x.arrived();
      if constexpr (H) h.arrived(), gate.arrived();
      Row::meet();
    }
    Vals<V> r[NV], u[NV], g[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      r[j] = x[j];
      if constexpr (H) {
        u[j] = h[j];
        g[j] = gate[j];
      }
    }
    if constexpr (kAhead) load(row + step);
    float mean0 = 0.f, rstd0 = 0.f, mean1 = 0.f, rstd1 = 0.f;
    if constexpr (H) {
      if (post) row_stats<V, L, NV, WG>(u, dup, ragged, a.post, a.inv_cols, a.eps, red, turn, mean0, rstd0);
      const float by = post ? rstd0 : 1.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        u[j] = (u[j] - mean0) * by * chunks.get(vec + floats, chunk[j]) + chunks.get(vec + 2 * floats, chunk[j]);
        uint32_t words[V];
        advoc::draw_chunk<V>(words, a.key.offset + (uint64_t)(row * cols + col[j]), aligned, key, a.key.thresh);
        Vals<V> s = chunks.get(vec, chunk[j]) * kept;
        advoc::activate<V>(g[j], a.act);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          s[k] *= has_gate ? g[j][k] : 1.f;
          r[j][k] += s[k] * (words[k] >= a.key.thresh ? u[j][k] : 0.f);
        }
        advoc::store_chunk<V>(advoc::row_at<R>(a.r, row * a.r_pitch, col[j]), r[j]);
      }
    }
    if constexpr (PRE) {
      row_stats<V, L, NV, WG>(r, dup, ragged, a.pre, a.inv_cols, a.eps, red, turn, mean1, rstd1);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Vals<V> z = (r[j] - mean1) * rstd1 * chunks.get(vec + 3 * floats, chunk[j]);
        if constexpr (kFive) z += chunks.get(vec + 4 * floats, chunk[j]);
        else if constexpr (kHeld) z += b_pre;
        else if (a.b_pre) z += advoc::floats_at<V>(a.b_pre + col[j]);
        advoc::store_chunk<V>(advoc::row_at<T>(a.z, row * a.z_pitch, col[j]), z);
      }
    }
    if (a.stats && lane == 0) a.stats[row] = make_float4(mean0, rstd0, mean1, rstd1);
  }
}

template <typename T, typename R>
struct Launch {
  const NormArgs& a;
  hipStream_t stream;
  template <int V, int L, int NV>
  void run() const {
    constexpr int WG = L > 64 ? L : 256;
    int64_t blocks = advoc::ceil_div(a.rows, Team<L, WG>::kRows);
    // the workgroups that are resident together, by waves and by LDS, then rows in turn
    constexpr int kByWaves = 4 * 64 * kWavesPerSimd / WG;
    static_assert(NV > 1 || kByWaves * lds_taken<V, L>(V * L * NV) <= kCuLds, "rows of this instance's width leave no wave without LDS");
    const int by_lds = kCuLds / lds_taken<V, L>(a.cols);
    const int64_t most = 256 * (by_lds < kByWaves ? by_lds : kByWaves);
    if (blocks > most) blocks = most;
    const dim3 grid((unsigned)blocks), block(WG);
    const unsigned lds = 4u * kVectors<L> * advoc::Chunks<V>(a.cols).floats();
    if (!a.h) hipLaunchKernelGGL((norm_forward_kernel<T, R, V, L, NV, WG, false, true>), grid, block, lds, stream, a);
    else if (a.pre == ADVOC_NORM_NONE) hipLaunchKernelGGL((norm_forward_kernel<T, R, V, L, NV, WG, true, false>), grid, block, lds, stream, a);
    else hipLaunchKernelGGL((norm_forward_kernel<T, R, V, L, NV, WG, true, true>), grid, block, lds, stream, a);
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

// Backward pass of the residual norm (gfx950), with the statistics the forward pass left:
//
//   rhat = (r - mean1) rstd1;  t = dz w_pre;     g  = dr + rstd1 (t - [mean t] - rhat mean(t rhat))        ([..]: LAYER only)
//   hhat = (h - mean0) rstd0;  v = drop(hhat w_post + b_post);   k = alpha scale act(gate)
//   dx = g;   dscale = sum alpha act(gate) v g;   dgate = sum alpha scale v g act'(gate);   du = drop(k g)
//   t = du w_post;             dh = rstd0 (t - [mean t] - hhat mean(t hhat))
//   dw_post = sum du hhat, db_post = sum du;      dw_pre = sum dz rhat, db_pre = sum dz
//
// One pass: the five inputs of a row are read once and the three outputs written once; u and v are computed again instead of being
// stored by the forward pass.  The column sums live in registers while a worker (the lanes of one row) walks over its rows, meet in
// LDS per workgroup and in HBM once per workgroup; a second small launch adds those up in a fixed order (no atomics: two runs give
// the same bits).  A gate row shared by the frames of a clip is summed the same way, a worker's rows never crossing a clip.
#include "residual_norm.h"

namespace {

using advoc::f32x8;
using advoc::NormArgs;
using advoc::Team;

enum { kDwPost, kDbPost, kDscale, kDwPre, kDbPre, kSums };

struct Sums {
  int slot[kSums];              // place in NormArgs.part, -1: not wanted
};

// g <- the gradient of a row given that of its normed values (times the weight): rstd (t - [mean t] - hat mean(t hat))
template <int V, int L, int NV, int WG>
__device__ __forceinline__ void norm_back(f32x8 (&t)[NV], const f32x8 (&hat)[NV], const int (&dup)[NV], int kind, float inv_cols,
                                          float rstd, float* red, int& turn) {
  float s0 = 0.f, s1 = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int k = 0; k < V; ++k) {
      s0 += k >= dup[j] ? t[j][k] : 0.f;
      s1 += k >= dup[j] ? t[j][k] * hat[j][k] : 0.f;
    }
  Team<L, WG>::sum2(s0, s1, red, turn);
  s0 = kind == ADVOC_NORM_LAYER ? s0 * inv_cols : 0.f;
  s1 *= inv_cols;
#pragma unroll
  for (int j = 0; j < NV; ++j) t[j] = (t[j] - s0 - hat[j] * s1) * rstd;
}

template <typename T, typename R, int V, int L, int NV, int WG>
__global__ __launch_bounds__(WG) void norm_backward_kernel(NormArgs a, Sums sums) {
  using Row = Team<L, WG>;
  __shared__ float red[L > 64 ? 4 * (L / 64) : 1];
  __shared__ float fold[L <= 64 ? Row::kRows * L * NV * V : 1];
  int turn = 0;
  const int lane = Row::lane();
  const uint2 key = advoc::drop_key_words(a.key);
  const bool aligned = (a.cols & 3) == 0;
  const int64_t group_rows = a.gate && a.gate_group > 1 ? a.gate_group : a.rows;
  const bool shared_gate = a.gate && a.gate_group > 1;
  int col[NV], dup[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) advoc::chunk_place<V, L>(j, lane, a.cols, col[j], dup[j]);

  f32x8 acc[kSums][NV];
#pragma unroll
  for (int s = 0; s < kSums; ++s)
#pragma unroll
    for (int j = 0; j < NV; ++j) acc[s][j] = (f32x8)(0.f);

  const int64_t workers = (int64_t)gridDim.x * Row::kRows;
  for (int64_t seg = (int64_t)blockIdx.x * Row::kRows + (L > 64 ? 0 : Row::slot()); seg < a.segments; seg += workers) {
    const int64_t group = seg / a.splits, first = (seg - group * a.splits) * a.chunk;
    const int64_t last = first + a.chunk < group_rows ? first + a.chunk : group_rows;
    f32x8 gacc[NV], gate[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      gacc[j] = (f32x8)(0.f);
      gate[j] = (f32x8)(1.f);
      if (shared_gate && dup[j] < V) gate[j] = advoc::load_chunk<V>((const T*)a.gate + group * a.gate_pitch + col[j]);
    }
    for (int64_t row = group * group_rows + first; row < group * group_rows + last; ++row) {
      f32x8 hat[NV], t[NV], g[NV], u[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        hat[j] = t[j] = g[j] = u[j] = (f32x8)(0.f);
        if (dup[j] >= V) continue;
        if (a.pre != ADVOC_NORM_NONE) {
          t[j] = advoc::load_chunk<V>((const T*)a.dz + row * a.dz_pitch + col[j]);
          hat[j] = advoc::load_chunk<V>((const R*)a.x + row * a.x_pitch + col[j]);
        }
        if (a.dr) g[j] = advoc::load_chunk<V>((const R*)a.dr + row * a.dr_pitch + col[j]);
        if (a.h) u[j] = advoc::load_chunk<V>((const T*)a.h + row * a.h_pitch + col[j]);
        if (a.gate && !shared_gate) gate[j] = advoc::load_chunk<V>((const T*)a.gate + row * a.gate_pitch + col[j]);
      }
      if constexpr (L > 64) __syncthreads();    // outputs may be the inputs' own buffers, and a column may have two holders
      const float4 st = a.stats ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
      if (a.pre != ADVOC_NORM_NONE) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (dup[j] >= V) continue;
          hat[j] = (hat[j] - st.z) * st.w;
          acc[kDwPre][j] += t[j] * hat[j];
          acc[kDbPre][j] += t[j];
          t[j] *= advoc::cols_chunk<V>(a.w_pre, col[j], 1.f);
        }
        norm_back<V, L, NV, WG>(t, hat, dup, a.pre, a.inv_cols, st.w, red, turn);
#pragma unroll
        for (int j = 0; j < NV; ++j) g[j] += t[j];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (dup[j] < V && a.dx) advoc::store_chunk<V>((R*)a.dx + row * a.dx_pitch + col[j], g[j]);
      if (!a.h) continue;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (dup[j] >= V) continue;
        hat[j] = u[j];
        if (a.post != ADVOC_NORM_NONE) {
          hat[j] = (u[j] - st.x) * st.y;
          u[j] = hat[j] * advoc::cols_chunk<V>(a.w_post, col[j], 1.f) + advoc::cols_chunk<V>(a.b_post, col[j], 0.f);
        }
        const uint32_t keep = advoc::keep_chunk<V>(a.key.offset + (uint64_t)(row * a.cols + col[j]), aligned, key, a.key.thresh);
        const f32x8 s = advoc::cols_chunk<V>(a.scale, col[j], 1.f);
        f32x8 dg;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float gt = a.gate ? advoc::gate_act(gate[j][k], a.act) : 1.f;
          const float v = (keep >> k & 1) ? u[j][k] * a.key.scale : 0.f, ag = a.alpha * g[j][k];
          acc[kDscale][j][k] += ag * gt * v;
          dg[k] = ag * s[k] * v;
          if (!shared_gate && a.act == ADVOC_GATE_SIGMOID) dg[k] *= gt * (1.f - gt);
          t[j][k] = (keep >> k & 1) ? ag * s[k] * gt * a.key.scale : 0.f;
        }
        if (shared_gate) gacc[j] += dg;
        else if (a.gate && a.dgate) advoc::store_chunk<V>((T*)a.dgate + row * a.dgate_pitch + col[j], dg);
        if (a.post != ADVOC_NORM_NONE) {
          acc[kDwPost][j] += t[j] * hat[j];
          acc[kDbPost][j] += t[j];
          t[j] *= advoc::cols_chunk<V>(a.w_post, col[j], 1.f);
        }
      }
      if (a.post != ADVOC_NORM_NONE) norm_back<V, L, NV, WG>(t, hat, dup, a.post, a.inv_cols, st.y, red, turn);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (dup[j] < V && a.dh) advoc::store_chunk<V>((T*)a.dh + row * a.dh_pitch + col[j], t[j]);
    }
    if (shared_gate && a.dgate) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (dup[j] >= V) continue;
        if (a.act == ADVOC_GATE_SIGMOID)
#pragma unroll
          for (int k = 0; k < V; ++k) {
            const float gt = advoc::gate_act(gate[j][k], a.act);
            gacc[j][k] *= gt * (1.f - gt);
          }
        if (a.gate_part) advoc::store_chunk<V>(a.gate_part + seg * a.cols + col[j], gacc[j]);
        else advoc::store_chunk<V>((T*)a.dgate + group * a.dgate_pitch + col[j], gacc[j]);
      }
    }
  }

  // the workgroup's column sums: values of a column with two holders are equal, so either may store them
#pragma unroll
  for (int s = 0; s < kSums; ++s) {
    if (sums.slot[s] < 0) continue;
    float* out = a.part + ((int64_t)sums.slot[s] * gridDim.x + blockIdx.x) * a.cols;
    if constexpr (L > 64) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (dup[j] < V) advoc::store_chunk<V>(out + col[j], acc[s][j]);
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (dup[j] < V) advoc::store_chunk<V>(fold + Row::slot() * a.cols + col[j], acc[s][j]);
      __syncthreads();
      for (int c = threadIdx.x; c < a.cols; c += WG) {
        float v = 0.f;
        for (int w = 0; w < Row::kRows; ++w) v += fold[w * a.cols + c];
        out[c] = v;
      }
    }
  }
}

// Adds up what the workgroups (column sums) and segments (shared gate rows) left, 64 columns to a block of four waves: wave w
// takes entries w, w + 4, ...
struct FoldArgs {
  const float *part, *gate_part;
  float* out[kSums];            // in the order of the slots
  void* dgate;
  int64_t dgate_pitch;
  int cols, col_blocks, sums, entries, splits, accumulate;
};

template <typename T>
__global__ __launch_bounds__(256) void norm_fold_kernel(FoldArgs a) {
  __shared__ float red[4][64];
  const int item = blockIdx.x / a.col_blocks, c = (blockIdx.x - item * a.col_blocks) * 64 + (threadIdx.x & 63);
  const int wave = threadIdx.x >> 6;
  const bool is_gate = item >= a.sums;
  const int n = is_gate ? a.splits : a.entries;
  const float* p = is_gate ? a.gate_part + (int64_t)(item - a.sums) * n * a.cols : a.part + (int64_t)item * n * a.cols;
  float v = 0.f;
  if (c < a.cols)
    for (int e = wave; e < n; e += 4) v += p[(int64_t)e * a.cols + c];
  red[wave][threadIdx.x & 63] = v;
  __syncthreads();
  if (wave == 0 && c < a.cols) {
    v = red[0][threadIdx.x] + red[1][threadIdx.x] + red[2][threadIdx.x] + red[3][threadIdx.x];
    if (is_gate) ((T*)a.dgate)[(int64_t)(item - a.sums) * a.dgate_pitch + c] = (T)v;
    else a.out[item][c] = a.accumulate ? a.out[item][c] + v : v;
  }
}

// How the rows are cut: workgroups, and for a shared gate how many workers share a gate row.
struct Plan {
  int64_t blocks = 0, chunk = 0, segments = 0;
  int splits = 0, sums = 0;
  bool gate_fold = false;
  int64_t part_floats = 0, gate_floats = 0;
};

struct MakePlan {
  const NormArgs& a;
  const Sums& sums;
  Plan& p;
  template <int V, int L, int NV, int WG>
  void run() const {
    constexpr int kRows = Team<L, WG>::kRows;
    const int64_t most = 512 * 256 / WG;
    const bool shared_gate = a.gate && a.gate_group > 1;
    const int64_t rows = shared_gate ? a.gate_group : a.rows, groups = a.rows / rows;
    int64_t splits = most * kRows / groups;
    if (splits > rows) splits = rows;
    if (splits < 1) splits = 1;
    p.chunk = advoc::ceil_div(rows, splits);
    p.splits = (int)advoc::ceil_div(rows, p.chunk);
    p.segments = groups * p.splits;
    p.blocks = advoc::ceil_div(p.segments, kRows);
    if (p.blocks > most) p.blocks = most;
    for (int s = 0; s < kSums; ++s) p.sums += sums.slot[s] >= 0;
    p.gate_fold = shared_gate && a.dgate && p.splits > 1;
    p.part_floats = p.sums * p.blocks * a.cols;
    p.gate_floats = p.gate_fold ? p.segments * a.cols : 0;
  }
};

template <typename T, typename R>
struct Launch {
  const NormArgs& a;
  const Sums& sums;
  int64_t blocks;
  hipStream_t stream;
  template <int V, int L, int NV, int WG>
  void run() const {
    hipLaunchKernelGGL((norm_backward_kernel<T, R, V, L, NV, WG>), dim3((unsigned)blocks), dim3(WG), 0, stream, a, sums);
  }
};

Sums wanted_sums(float* const (&out)[kSums], float* (&packed)[kSums]) {
  Sums s;
  int n = 0;
  for (int i = 0; i < kSums; ++i) {
    s.slot[i] = out[i] ? n : -1;
    if (out[i]) packed[n++] = out[i];
  }
  for (; n < kSums; ++n) packed[n] = nullptr;
  return s;
}

}  // namespace

namespace advoc {

int64_t norm_backward_workspace(const NormArgs& a, float* const (&out)[5]) {
  float* packed[kSums];
  const Sums sums = wanted_sums(out, packed);
  Plan p;
  if (!norm_dispatch(a.cols, MakePlan{a, sums, p})) return 0;
  return 4 * (p.part_floats + p.gate_floats);
}

int launch_norm_backward(NormArgs a, int dtype, int res_dtype, float* const (&out)[5], int accumulate, void* workspace,
                         int64_t workspace_bytes, hipStream_t stream) {
  FoldArgs f = {};
  const Sums sums = wanted_sums(out, f.out);
  Plan p;
  if (!norm_dispatch(a.cols, MakePlan{a, sums, p})) return ADVOC_ERR_UNSUPPORTED;
  if (4 * (p.part_floats + p.gate_floats) > workspace_bytes) return ADVOC_ERR_NULL;
  a.part = (float*)workspace;
  a.gate_part = p.gate_fold ? (float*)workspace + p.part_floats : nullptr;
  a.chunk = p.chunk;
  a.segments = p.segments;
  a.splits = p.splits;
  ADVOC_CLEAR_LAUNCH_ERROR();
  if (dtype == ADVOC_F32)
    norm_dispatch(a.cols, Launch<float, float>{a, sums, p.blocks, stream});
  else if (dtype == ADVOC_BF16 && res_dtype == ADVOC_F32)
    norm_dispatch(a.cols, Launch<__bf16, float>{a, sums, p.blocks, stream});
  else if (dtype == ADVOC_BF16)
    norm_dispatch(a.cols, Launch<__bf16, __bf16>{a, sums, p.blocks, stream});
  else if (res_dtype == ADVOC_F32)
    norm_dispatch(a.cols, Launch<_Float16, float>{a, sums, p.blocks, stream});
  else
    norm_dispatch(a.cols, Launch<_Float16, _Float16>{a, sums, p.blocks, stream});
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  if (p.sums == 0 && !p.gate_fold) return ADVOC_OK;
  f.part = a.part;
  f.gate_part = a.gate_part;
  f.dgate = a.dgate;
  f.dgate_pitch = a.dgate_pitch;
  f.cols = a.cols;
  f.col_blocks = (int)ceil_div(a.cols, 64);
  f.sums = p.sums;
  f.entries = (int)p.blocks;
  f.splits = p.splits;
  f.accumulate = accumulate;
  const int64_t items = p.sums + (p.gate_fold ? a.rows / a.gate_group : 0);
  const dim3 grid((unsigned)(items * f.col_blocks));
  ADVOC_CLEAR_LAUNCH_ERROR();
  if (dtype == ADVOC_F32) hipLaunchKernelGGL(norm_fold_kernel<float>, grid, dim3(256), 0, stream, f);
  else if (dtype == ADVOC_BF16) hipLaunchKernelGGL(norm_fold_kernel<__bf16>, grid, dim3(256), 0, stream, f);
  else hipLaunchKernelGGL(norm_fold_kernel<_Float16>, grid, dim3(256), 0, stream, f);
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

}  // namespace advoc

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

// t <- the gradient of a row given that of its normed values (times the weight): rstd (t - [mean t] - hat mean(t hat))
template <int V, int L, int NV, int WG>
__device__ __forceinline__ void norm_back(f32x8 (&t)[NV], const f32x8 (&hat)[NV], const int (&dup)[NV], bool ragged, int kind,
                                          float inv_cols, float rstd, float* red, int& turn) {
  float s0 = advoc::own_sum<V>(dup, ragged, [&](int j, int k) { return t[j][k]; });
  float s1 = advoc::own_sum<V>(dup, ragged, [&](int j, int k) { return t[j][k] * hat[j][k]; });
  Team<L, WG>::sum2(s0, s1, red, turn);
  s0 = kind == ADVOC_NORM_LAYER ? s0 * inv_cols : 0.f;
  s1 *= inv_cols;
#pragma unroll
  for (int j = 0; j < NV; ++j) t[j] = (t[j] - s0 - hat[j] * s1) * rstd;
}

// Two workgroups of 256 on a CU (256 registers a lane): the column vectors are read again for every row, from the caches -- held in
// registers they left one wave to a SIMD.
template <typename T, typename R, int V, int L, int NV, int WG>
__global__ __launch_bounds__(WG, 2) void norm_backward_kernel(NormArgs a, Sums sums) {
  using Row = Team<L, WG>;
  __shared__ float red[L > 64 ? 4 * (L / 64) : 1];
  __shared__ float fold[L <= 64 ? Row::kRows * L * NV * V : 1];
  int turn = 0;
  const int lane = Row::lane();
  const uint2 key = advoc::drop_key_words(a.key);
  const bool aligned = (a.cols & 3) == 0, ragged = a.cols % V != 0;
  const bool shared_gate = a.gate && a.gate_group > 1;
  const int group_rows = (int)(shared_gate ? a.gate_group : a.rows);
  int col[NV], dup[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) advoc::chunk_place<V, L>(j, lane, a.cols, col[j], dup[j]);

  f32x8 acc[kSums][NV];
#pragma unroll
  for (int s = 0; s < kSums; ++s)
#pragma unroll
    for (int j = 0; j < NV; ++j) acc[s][j] = (f32x8)(0.f);

  const int workers = (int)gridDim.x * Row::kRows;
  for (int seg = (int)blockIdx.x * Row::kRows + (L > 64 ? 0 : Row::slot()); seg < a.segments; seg += workers) {
    const int group = seg / a.splits, first = (seg - group * a.splits) * (int)a.chunk;
    const int last = first + (int)a.chunk < group_rows ? first + (int)a.chunk : group_rows;
    f32x8 gacc[NV], gate[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      gacc[j] = (f32x8)(0.f);
      gate[j] = (f32x8)(1.f);
      if (shared_gate) {
        gate[j] = advoc::load_chunk<V>((const T*)a.gate + group * a.gate_pitch + col[j]);
        advoc::activate<V>(gate[j], a.act);
      }
    }
    for (int64_t row = (int64_t)group * group_rows + first; row < (int64_t)group * group_rows + last; ++row) {
      asm volatile("" ::: "memory");            // (keeps the column vectors out of registers between rows)
      f32x8 hat[NV], t[NV], g[NV], u[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        hat[j] = t[j] = g[j] = u[j] = (f32x8)(0.f);
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
            hat[j] = (hat[j] - st.z) * st.w;
          acc[kDwPre][j] += t[j] * hat[j];
          acc[kDbPre][j] += t[j];
          t[j] *= advoc::cols_chunk<V>(a.w_pre, col[j], 1.f);
        }
        norm_back<V, L, NV, WG>(t, hat, dup, ragged, a.pre, a.inv_cols, st.w, red, turn);
#pragma unroll
        for (int j = 0; j < NV; ++j) g[j] += t[j];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (a.dx) advoc::store_chunk<V>((R*)a.dx + row * a.dx_pitch + col[j], g[j]);
      if (!a.h) continue;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        hat[j] = u[j];
        if (a.post != ADVOC_NORM_NONE) {
          hat[j] = (u[j] - st.x) * st.y;
          u[j] = hat[j] * advoc::cols_chunk<V>(a.w_post, col[j], 1.f) + advoc::cols_chunk<V>(a.b_post, col[j], 0.f);
        }
        const uint32_t keep = advoc::keep_chunk<V>(a.key.offset + (uint64_t)(row * a.cols + col[j]), aligned, key, a.key.thresh);
        if (a.gate && !shared_gate) advoc::activate<V>(gate[j], a.act);
        const f32x8 ks = advoc::cols_chunk<V>(a.scale, col[j], 1.f) * a.alpha;
        f32x8 dg;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const float f = (keep >> k & 1) ? a.key.scale : 0.f;
          const float v = (keep >> k & 1) ? u[j][k] * a.key.scale : 0.f, gv = g[j][k] * v;
          acc[kDscale][j][k] += gv * gate[j][k];         // alpha is applied once, at the end
          dg[k] = gv * ks[k];
          t[j][k] = f * (ks[k] * gate[j][k] * g[j][k]);
          if (!(keep >> k & 1)) t[j][k] = 0.f;
        }
        if (shared_gate) {
          gacc[j] += dg;
        } else if (a.gate && a.dgate) {
          if (a.act == ADVOC_GATE_SIGMOID) dg *= gate[j] * (f32x8(1.f) - gate[j]);
          advoc::store_chunk<V>((T*)a.dgate + row * a.dgate_pitch + col[j], dg);
        }
        if (a.post != ADVOC_NORM_NONE) {
          acc[kDwPost][j] += t[j] * hat[j];
          acc[kDbPost][j] += t[j];
          t[j] *= advoc::cols_chunk<V>(a.w_post, col[j], 1.f);
        }
      }
      if (a.post != ADVOC_NORM_NONE) norm_back<V, L, NV, WG>(t, hat, dup, ragged, a.post, a.inv_cols, st.y, red, turn);
#pragma unroll
      for (int j = 0; j < NV; ++j)
        if (a.dh) advoc::store_chunk<V>((T*)a.dh + row * a.dh_pitch + col[j], t[j]);
    }
    if (shared_gate && a.dgate) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (a.act == ADVOC_GATE_SIGMOID) gacc[j] *= gate[j] * (f32x8(1.f) - gate[j]);
        if (a.gate_part) advoc::store_chunk<V>(a.gate_part + (int64_t)seg * a.cols + col[j], gacc[j]);
        else advoc::store_chunk<V>((T*)a.dgate + group * a.dgate_pitch + col[j], gacc[j]);
      }
    }
  }

  // the workgroup's column sums: values of a column with two holders are equal, so either may store them
#pragma unroll
  for (int j = 0; j < NV; ++j) acc[kDscale][j] *= a.alpha;
#pragma unroll
  for (int s = 0; s < kSums; ++s) {
    if (sums.slot[s] < 0) continue;
    float* out = a.part + ((int64_t)sums.slot[s] * gridDim.x + blockIdx.x) * a.cols;
    if constexpr (L > 64) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
        advoc::store_chunk<V>(out + col[j], acc[s][j]);
    } else {
      __syncthreads();
#pragma unroll
      for (int j = 0; j < NV; ++j)
        advoc::store_chunk<V>(fold + Row::slot() * a.cols + col[j], acc[s][j]);
      __syncthreads();
      for (int c = threadIdx.x; c < a.cols; c += WG) {
        float v = 0.f;
        for (int w = 0; w < Row::kRows; ++w) v += fold[w * a.cols + c];
        out[c] = v;
      }
    }
  }
}

// Adds up what the workgroups (column sums) and segments (shared gate rows) left, 64 columns to a block of 16 waves: wave w takes
// entries w, w + 16, ..., eight of them in flight.
struct FoldArgs {
  const float *part, *gate_part;
  float* out[kSums];            // in the order of the slots
  void* dgate;
  int64_t dgate_pitch;
  int cols, col_blocks, sums, entries, splits, accumulate;
};

template <typename T>
__global__ __launch_bounds__(1024) void norm_fold_kernel(FoldArgs a) {
  constexpr int kWaves = 16, kDeep = 8;
  __shared__ float red[kWaves][64];
  const int item = blockIdx.x / a.col_blocks, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int c = (blockIdx.x - item * a.col_blocks) * 64 + lane;
  const bool is_gate = item >= a.sums;
  const int n = is_gate ? a.splits : a.entries;
  const float* p = is_gate ? a.gate_part + (int64_t)(item - a.sums) * n * a.cols : a.part + (int64_t)item * n * a.cols;
  float v = 0.f;
  if (c < a.cols) {
    int e = wave;
    for (; e + (kDeep - 1) * kWaves < n; e += kDeep * kWaves) {
      float x[kDeep];
#pragma unroll
      for (int i = 0; i < kDeep; ++i) x[i] = p[(int64_t)(e + i * kWaves) * a.cols + c];
#pragma unroll
      for (int i = 0; i < kDeep; ++i) v += x[i];
    }
    for (; e < n; e += kWaves) v += p[(int64_t)e * a.cols + c];
  }
  red[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && c < a.cols) {
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v += red[w][lane];
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
  if (dtype == ADVOC_F32) hipLaunchKernelGGL(norm_fold_kernel<float>, grid, dim3(1024), 0, stream, f);
  else if (dtype == ADVOC_BF16) hipLaunchKernelGGL(norm_fold_kernel<__bf16>, grid, dim3(1024), 0, stream, f);
  else hipLaunchKernelGGL(norm_fold_kernel<_Float16>, grid, dim3(1024), 0, stream, f);
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

}  // namespace advoc

// Backward pass of the residual norm (gfx950), with the statistics the forward pass left:
//
//   rhat = (r - mean1) rstd1;  t = dz w_pre;     g  = dr + rstd1 (t - [mean t] - rhat mean(t rhat))        ([..]: LAYER only)
//   hhat = (h - mean0) rstd0;  e = drop(alpha g);   E0 = sum e act(gate),  E1 = sum e act(gate) hhat
//   dx = g;   du = e scale act(gate);   t = du w_post;   dh = rstd0 (t - [mean t] - hhat mean(t hhat))
//   dgate = sum e scale (hhat w_post + b_post) act'(gate)
//   dw_post = scale E1,  db_post = scale E0,  dscale = w_post E1 + b_post E0;      dw_pre = sum dz rhat, db_pre = sum dz
//
// Four column sums in registers give the five parameter gradients: what is constant in a column stays outside its sums, and is
// multiplied in when a workgroup's sums leave it (five of them, those that are wanted).  One pass: the five
// inputs of a row are read once and the three outputs written once; the mask is drawn again.  The sums live in registers while a
// worker (the lanes of one row) walks over its rows, meet in LDS per workgroup and in HBM once per workgroup; a second small launch
// adds those up in a fixed order (no atomics: two runs give the same bits).  A gate row shared by the frames of a clip is summed the
// same way, a worker's rows never crossing a clip: G0 = sum e, G1 = sum e hhat over them give dgate = scale (w_post G1 + b_post G0)
// act' and their part of E0, E1.
//
// Measured (kernel + the second launch): 16384 x 1024, bf16 with fp32 residuals, a gate per clip, dropout (302 MB): 68 + 5 us, 4.4
// TB/s; each further row comes at 5.0 TB/s (adding 1 to as much: 5.8), and 12 us are the way of the first row (arguments and vectors 4,
// loads 2, arithmetic 4, the workgroup's column sums 3).  (A gate's gradient that left every worker instead of every workgroup: 69 + 6.)
// 4096 x 4096 fp16 (201 MB, and 21 MB of column sums written and read again): 52 + 5.  3999 x 513 fp32 (66 MB): 21 + 4, two rows a
// worker: the same start and end, and the arithmetic.
#include "residual_norm.h"

namespace {

using advoc::NormArgs;
using advoc::Team;
using advoc::Vals;

enum { kDwPost, kDbPost, kDscale, kDwPre, kDbPre, kSums };

struct Sums {
  int slot[kSums];              // place in NormArgs.part, -1: not wanted
};

// Two waves to a SIMD, 256 registers to a lane: rows of 16 columns a lane need them all, a third for the sums, and have 512 lanes to a
// workgroup (half the partial column sums of 256); rows of 8 columns a lane use the rest to fetch a row ahead, which is worth more
// than a third wave (16384 x 256: 24 -> 20 us, 8192 x 2048: 80 -> 74, 4096 x 4096 fp16: 60 -> 52).
constexpr int kWavesPerSimd = 2;
template <int L, int NV>
constexpr int kLanes = L > 64 ? L : NV > 1 ? 512 : 256;

// Sums that go through LDS together at the end of a workgroup: up to 55 KB with two workgroups to a CU, 128 KB with one.
template <int NV>
constexpr int kSumsTogether = NV > 1 ? 4 : 6;

// t <- the gradient of a row given that of its normed values (times the weight): rstd (t - [mean t] - hat mean(t hat))
template <int V, int L, int NV, int WG>
__device__ __forceinline__ void norm_back(Vals<V> (&t)[NV], const Vals<V> (&hat)[NV], const int (&dup)[NV], bool ragged, int kind,
                                          float inv_cols, float rstd, float* red, int& turn) {
  float s0 = advoc::own_sum<V>(dup, ragged, [&](int j, int k) { return t[j][k]; });
  float s1 = advoc::own_sum<V>(dup, ragged, [&](int j, int k) { return t[j][k] * hat[j][k]; });
  Team<L, WG>::sum2(s0, s1, red, turn);
  s0 = kind == ADVOC_NORM_LAYER ? s0 * inv_cols : 0.f;
  s1 *= inv_cols;
#pragma unroll
  for (int j = 0; j < NV; ++j) t[j] = (t[j] - s0 - hat[j] * s1) * rstd;
}

// H: there is a block output (otherwise only the pre norm is differentiated); PRE: there is a pre norm.  Everything else that may be
// absent is not a branch (register allocation around those cost more than the work they save): an absent dr or gate is read from
// where r or h lies and replaced by its neutral value, absent vectors are staged as theirs.
template <typename T, typename R, int V, int L, int NV, int WG, bool H, bool PRE>
__global__ __launch_bounds__(WG, kWavesPerSimd) void norm_backward_kernel(NormArgs a, Sums sums) {
  using Row = Team<L, WG>;
  // a row's loads go out as soon as those of the row before have been used, ahead of that one's second half (with 16 columns a lane
  // that spills: 16384 x 1024 69 -> 116 us)
  constexpr bool kAhead = NV == 1;
  __shared__ float red[L > 64 ? 4 * (L / 64) : 1];
  extern __shared__ __align__(16) float vec[];                // w_pre, w_post, b_post, scale; afterwards the column sums of the workgroup's rows
  int turn = 0;
  const int lane = Row::lane(), cols = a.cols;
  const uint2 key = advoc::drop_key_words(a.key);
  const bool aligned = (cols & 3) == 0, ragged = cols % V != 0;
  const bool has_dr = a.dr, has_gate = a.gate, shared_gate = has_gate && a.gate_group > 1, row_gate = has_gate && !shared_gate;
  const bool post = a.post != ADVOC_NORM_NONE;
  const int group_rows = (int)(shared_gate ? a.gate_group : a.rows);
  const void* dr = has_dr ? a.dr : a.x;
  const void* gate_base = has_gate ? a.gate : a.h;
  const int64_t dr_pitch = has_dr ? a.dr_pitch : a.x_pitch, gate_pitch = has_gate ? a.gate_pitch : a.h_pitch;
  int chunk[NV], col[NV], dup[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) advoc::chunk_place<V, L>(j, lane, cols, chunk[j], col[j], dup[j]);

  const advoc::Chunks<V> chunks(cols);
  const int floats = chunks.floats();
  auto w_pre = [&](int j) { return chunks.get(vec, chunk[j]); };
  auto w_post = [&](int j) { return chunks.get(vec + floats, chunk[j]); };
  auto b_post = [&](int j) { return chunks.get(vec + 2 * floats, chunk[j]); };
  auto scale = [&](int j) { return chunks.get(vec + 3 * floats, chunk[j]); };

  advoc::stage_vectors<WG, V, 4>(vec, {a.w_pre, a.w_post, a.b_post, a.scale}, {1.f, 1.f, 0.f, 1.f}, cols);
  Row::meet();

  // sums over rows.  g0, g1 are E0, E1 but for the gate where rows share one
  Vals<V> dw_pre[NV], db_pre[NV], g0[NV], g1[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) dw_pre[j] = db_pre[j] = g0[j] = g1[j] = Vals<V>(0.f);
  // a worker with several clips carries E0, E1 of those before in memory of its own
  constexpr int kOwn = NV * L * V;
  float* const carry = a.carry ? a.carry + ((int64_t)blockIdx.x * Row::kRows + Row::slot()) * 2 * kOwn + lane * V : nullptr;

  const int workers = (int)gridDim.x * Row::kRows;
  const float kept = a.alpha * a.key.scale;
  bool again = false;
  for (int seg = (int)blockIdx.x * Row::kRows + Row::slot(); seg < a.segments; seg += workers) {
    // part p of a group takes rows p, p + splits, ...: what runs together lies together
    const int group = seg / a.splits, first = seg - group * a.splits;
    const int64_t end = (int64_t)(group + 1) * group_rows;
    if (H && carry)
#pragma unroll
      for (int j = 0; j < NV; ++j) g0[j] = g1[j] = Vals<V>(0.f);
    advoc::Raw<T, V, NV> raw_gate, raw_dz, raw_h;
    advoc::Raw<R, V, NV> raw_r, raw_dr;
    auto load = [&](int64_t row) {
      if constexpr (PRE) {
        raw_dz.load(a.dz, row * a.dz_pitch, col);
        raw_r.load(a.x, row * a.x_pitch, col);
      }
      raw_dr.load(dr, row * dr_pitch, col);
      if constexpr (H) {
        raw_h.load(a.h, row * a.h_pitch, col);
        raw_gate.load(gate_base, (shared_gate ? group : row) * gate_pitch, col);
      }
    };
    if constexpr (kAhead) load(end - group_rows + first);
    for (int64_t row = end - group_rows + first; row < end; row += a.splits) {
      advoc::forget_lds();
      if constexpr (!kAhead) load(row);
      Vals<V> hat[NV], t[NV], g[NV], gate[NV];
      const float4 st = PRE || post ? a.stats[row] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        g[j] = raw_dr[j];
#pragma unroll
        for (int k = 0; k < V; ++k) g[j][k] = has_dr ? g[j][k] : 0.f;
        if constexpr (PRE) {
          t[j] = raw_dz[j];
          hat[j] = (raw_r[j] - st.z) * st.w;
          dw_pre[j] += t[j] * hat[j];
          db_pre[j] += t[j];
          t[j] *= w_pre(j);
        }
      }
      if constexpr (PRE) {
        norm_back<V, L, NV, WG>(t, hat, dup, ragged, a.pre, a.inv_cols, st.w, red, turn);
#pragma unroll
        for (int j = 0; j < NV; ++j) g[j] += t[j];
      }
      if constexpr (H) {
        const float mean = post ? st.x : 0.f, rstd = post ? st.y : 1.f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          hat[j] = (raw_h[j] - mean) * rstd;
          gate[j] = raw_gate[j];
        }
      }
      if constexpr (L > 64) {                   // outputs may be the inputs' own buffers, and a column may have two holders
        raw_dr.arrived();
        if constexpr (H) raw_h.arrived(), raw_gate.arrived();
        Row::meet();
      }
      if constexpr (kAhead) load(row + a.splits < end ? row + a.splits : row);
      if (a.dx)
#pragma unroll
        for (int j = 0; j < NV; ++j) advoc::store_chunk<V>(advoc::row_at<R>(a.dx, row * a.dx_pitch, col[j]), g[j]);
      if constexpr (!H) continue;
      advoc::forget_lds();
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        uint32_t words[V];
        advoc::draw_chunk<V>(words, a.key.offset + (uint64_t)(row * cols + col[j]), aligned, key, a.key.thresh);
        advoc::activate<V>(gate[j], a.act);
        const Vals<V> s = scale(j);
        // What is dropped has no gradient and is no part of a sum, whatever its h and gate hold: 0 times an infinity or a NaN would be
        // one, so both are replaced (norm_back below takes hat as it is: there a NaN is its row's).
        Vals<V> hat_kept;
#pragma unroll
        for (int k = 0; k < V; ++k) {
          const bool stays = words[k] >= a.key.thresh;
          gate[j][k] = has_gate && stays ? gate[j][k] : 1.f;
          hat_kept[k] = stays ? hat[j][k] : 0.f;
          t[j][k] = stays ? g[j][k] * kept : 0.f;
        }
        if (row_gate && a.dgate) {
          Vals<V> dg = t[j] * s * (hat_kept * w_post(j) + b_post(j));
          if (a.act == ADVOC_GATE_SIGMOID) dg *= gate[j] * (Vals<V>(1.f) - gate[j]);
          advoc::store_chunk<V>(advoc::row_at<T>(a.dgate, row * a.dgate_pitch, col[j]), dg);
        }
        const Vals<V> e = t[j] * gate[j];
        Vals<V> sum = shared_gate ? t[j] : e;
        g0[j] += sum;
        g1[j] += sum * hat_kept;
        t[j] = e * s * w_post(j);               // (w_post is staged as ones without a post norm)
      }
      if (post) norm_back<V, L, NV, WG>(t, hat, dup, ragged, a.post, a.inv_cols, st.y, red, turn);
      if (a.dh)
#pragma unroll
        for (int j = 0; j < NV; ++j) advoc::store_chunk<V>(advoc::row_at<T>(a.dh, row * a.dh_pitch, col[j]), t[j]);
    }
    if (H && shared_gate && !a.gate_blocks) {
      raw_gate.load(gate_base, group * gate_pitch, col);
      if constexpr (L > 64) {
        raw_gate.arrived();
        Row::meet();
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Vals<V> gate = raw_gate[j];
        advoc::activate<V>(gate, a.act);
        if (a.dgate) {
          Vals<V> dg = scale(j) * (w_post(j) * g1[j] + b_post(j) * g0[j]);
          if (a.act == ADVOC_GATE_SIGMOID) dg *= gate * (Vals<V>(1.f) - gate);
          if (a.gate_part) advoc::store_chunk<V>(a.gate_part + (int64_t)seg * cols + col[j], dg);
          else advoc::store_chunk<V>(advoc::row_at<T>(a.dgate, group * a.dgate_pitch, col[j]), dg);
        }
        g0[j] *= gate;
        g1[j] *= gate;
        if (carry) {
          float *c0 = carry + j * L * V, *c1 = c0 + kOwn;
          if (again) {
            g0[j] += advoc::floats_at<V>(c0);
            g1[j] += advoc::floats_at<V>(c1);
          }
          advoc::store_chunk<V>(c0, g0[j]);
          advoc::store_chunk<V>(c1, g1[j]);
        }
      }
      again = true;
    }
  }

  // the workgroup's column sums: values of a column with two holders are equal, so either may store them
  constexpr int kGate = kSums, kAll = H && L <= 64 ? kSums + 1 : kSums;
  Vals<V> out[kAll][NV];
  if constexpr (kAll > kSums) {
    if (a.gate_blocks) {
      const int group = ((int)blockIdx.x * Row::kRows + Row::slot()) / a.splits;
      advoc::Raw<T, V, NV> raw_gate;
      raw_gate.load(gate_base, group * gate_pitch, col);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        Vals<V> gate = raw_gate[j];
        advoc::activate<V>(gate, a.act);
        out[kGate][j] = scale(j) * (w_post(j) * g1[j] + b_post(j) * g0[j]);
        if (a.act == ADVOC_GATE_SIGMOID) out[kGate][j] *= gate * (Vals<V>(1.f) - gate);
        g0[j] *= gate;
        g1[j] *= gate;
      }
    }
  }
  auto wanted = [&](int s) { return s < kSums ? sums.slot[s] >= 0 : a.gate_blocks != 0; };
  auto entry = [&](int s) {
    return (s < kSums ? a.part + (int64_t)sums.slot[s] * gridDim.x * cols : a.gate_part) + (int64_t)blockIdx.x * cols;
  };
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    out[kDwPost][j] = scale(j) * g1[j];
    out[kDbPost][j] = scale(j) * g0[j];
    out[kDscale][j] = w_post(j) * g1[j] + b_post(j) * g0[j];
    out[kDwPre][j] = dw_pre[j];
    out[kDbPre][j] = db_pre[j];
  }
  if constexpr (L > 64) {
#pragma unroll
    for (int s = 0; s < kSums; ++s)
      if (wanted(s))
#pragma unroll
        for (int j = 0; j < NV; ++j) advoc::store_chunk<V>(entry(s) + col[j], out[s][j]);
  } else {
    // kTogether sums at a time: [sum][row of the workgroup] in LDS
    constexpr int kTogether = kSumsTogether<NV>;
#pragma unroll
    for (int first = 0; first < kAll; first += kTogether) {
      __syncthreads();
#pragma unroll
      for (int s = first; s < kAll && s < first + kTogether; ++s)
        if (wanted(s))
#pragma unroll
          for (int j = 0; j < NV; ++j) chunks.put(vec + ((s - first) * Row::kRows + Row::slot()) * floats, chunk[j], out[s][j]);
      __syncthreads();
      chunks.template walk<WG>([&](int at, int c, auto n) {
        constexpr int kPiece = decltype(n)::value;
#pragma unroll
        for (int s = first; s < kAll && s < first + kTogether; ++s) {
          if (!wanted(s)) continue;
          const float* from = vec + (s - first) * Row::kRows * floats + at;
          float v[kPiece];
#pragma unroll
          for (int k = 0; k < kPiece; ++k) v[k] = 0.f;
          for (int w = 0; w < Row::kRows; ++w) {
            float x[kPiece];
            __builtin_memcpy(x, __builtin_assume_aligned(from + w * floats, 4 * kPiece), sizeof(x));
#pragma unroll
            for (int k = 0; k < kPiece; ++k) v[k] += x[k];
          }
          __builtin_memcpy(entry(s) + c, v, sizeof(v));
        }
      });
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
  int64_t blocks = 0, segments = 0;
  int splits = 0, sums = 0, gate_entries = 0;
  bool gate_fold = false, gate_blocks = false;
  int64_t part_floats = 0, gate_floats = 0, carry_floats = 0;
};

struct MakePlan {
  const NormArgs& a;
  const Sums& sums;
  Plan& p;
  template <int V, int L, int NV>
  void run() const {
    constexpr int kRows = Team<L, kLanes<L, NV>>::kRows;
    const int64_t most = 256 * 4 * 64 * kWavesPerSimd / kLanes<L, NV>;      // what is resident together
    const bool shared_gate = a.gate && a.gate_group > 1;
    const int64_t rows = shared_gate ? a.gate_group : a.rows, groups = a.rows / rows;
    int64_t splits = most * kRows / groups;
    if (splits > rows) splits = rows;
    if (splits < 1) splits = 1;
    // whole workgroups to a gate row, where that makes no worker's share longer: its gradient then meets in LDS first
    const int64_t whole = L <= 64 ? splits - splits % kRows : 0;
    if (shared_gate && whole > 0 && advoc::ceil_div(rows, whole) == advoc::ceil_div(rows, splits)) splits = whole;
    p.splits = (int)splits;
    p.segments = groups * p.splits;
    p.blocks = advoc::ceil_div(p.segments, kRows);
    if (p.blocks > most) p.blocks = most;
    for (int s = 0; s < kSums; ++s) p.sums += sums.slot[s] >= 0;
    p.gate_fold = shared_gate && a.dgate && p.splits > 1;
    p.part_floats = p.sums * p.blocks * a.cols;
    p.gate_blocks = p.gate_fold && L <= 64 && p.splits % kRows == 0;
    p.gate_entries = p.gate_blocks ? p.splits / kRows : p.splits;
    p.gate_floats = p.gate_fold ? groups * p.gate_entries * a.cols : 0;
    if (shared_gate && p.segments > p.blocks * kRows) p.carry_floats = p.blocks * kRows * 2 * NV * L * V;
  }
};

template <typename T, typename R>
struct Launch {
  const NormArgs& a;
  const Sums& sums;
  int64_t blocks;
  hipStream_t stream;
  template <int V, int L, int NV>
  void run() const {
    constexpr int WG = kLanes<L, NV>, kRows = Team<L, WG>::kRows;
    const dim3 grid((unsigned)blocks), block(WG);
    const unsigned lds = 4u * advoc::Chunks<V>(a.cols).floats() * (L > 64 ? 4 : kRows * kSumsTogether<NV>);
    if (!a.h) hipLaunchKernelGGL((norm_backward_kernel<T, R, V, L, NV, WG, false, true>), grid, block, lds, stream, a, sums);
    else if (a.pre == ADVOC_NORM_NONE) hipLaunchKernelGGL((norm_backward_kernel<T, R, V, L, NV, WG, true, false>), grid, block, lds, stream, a, sums);
    else hipLaunchKernelGGL((norm_backward_kernel<T, R, V, L, NV, WG, true, true>), grid, block, lds, stream, a, sums);
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
  return 4 * (p.part_floats + p.gate_floats + p.carry_floats);
}

// what a call without rows overwrites: the sums of no entries
int clear_norm_sums(int cols, float* const (&out)[5], hipStream_t stream) {
  FoldArgs f = {};
  const Sums sums = wanted_sums(out, f.out);
  for (int s = 0; s < kSums; ++s) f.sums += sums.slot[s] >= 0;
  if (f.sums == 0) return ADVOC_OK;
  f.cols = cols;
  f.col_blocks = (int)ceil_div(cols, 64);
  ADVOC_CLEAR_LAUNCH_ERROR();
  hipLaunchKernelGGL(norm_fold_kernel<float>, dim3((unsigned)(f.sums * f.col_blocks)), dim3(1024), 0, stream, f);
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

int launch_norm_backward(NormArgs a, int dtype, int res_dtype, float* const (&out)[5], int accumulate, void* workspace,
                         int64_t workspace_bytes, hipStream_t stream) {
  FoldArgs f = {};
  const Sums sums = wanted_sums(out, f.out);
  Plan p;
  if (!norm_dispatch(a.cols, MakePlan{a, sums, p})) return ADVOC_ERR_UNSUPPORTED;
  if (4 * (p.part_floats + p.gate_floats + p.carry_floats) > workspace_bytes) return ADVOC_ERR_NULL;
  a.part = (float*)workspace;
  a.gate_part = p.gate_fold ? (float*)workspace + p.part_floats : nullptr;
  a.carry = p.carry_floats ? (float*)workspace + p.part_floats + p.gate_floats : nullptr;
  a.gate_blocks = p.gate_blocks;
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
  f.splits = p.gate_entries;
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

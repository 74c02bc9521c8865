// What the forward and the backward pass of the residual norm share: how a row lies on lanes, and row sums.
//
//   u = N_post(h) w_post + b_post;   v = drop(u);   r = x + k v,  k = alpha scale act(gate);   z = N_pre(r) w_pre + b_pre
//
// A row of `cols` values is held by L lanes, V consecutive values at a time, NV times: value k of chunk j of lane l is column
// (j L + l) V + k.  Up to 64 lanes a row is part of a wave and its sums are lane exchanges; wider rows are a workgroup's, whose
// waves meet in LDS.  Everything a row needs is read once and stays in registers for both norms.
// A chunk that would reach past the last column is moved back to end there: it holds columns its neighbour holds too (`dup` of them;
// all V where the whole chunk lies behind the row), computes the same values for them, stores the same values, and leaves them out
// of sums.  So no lane ever branches on where the row ends.
#pragma once
#include "philox.h"
#include "rows.h"

namespace advoc {

struct NormArgs {
  int64_t rows;
  int cols;
  int post, pre, act;           // ADVOC_NORM_*, ADVOC_GATE_*
  int64_t gate_group;           // rows that share a gate row
  const float *w_post, *b_post, *scale, *w_pre, *b_pre;
  float alpha, eps, inv_cols;
  DropKey key;
  const void *h, *x, *gate;     // backward: x holds r
  int64_t h_pitch, x_pitch, gate_pitch;
  void *r, *z;
  int64_t r_pitch, z_pitch;
  float4* stats;                // per row: mean, 1 / sqrt(var + eps) of the post norm, the same of the pre norm
  // backward
  const void *dz, *dr;
  int64_t dz_pitch, dr_pitch;
  void *dh, *dx, *dgate;
  int64_t dh_pitch, dx_pitch, dgate_pitch;
  float* part;                  // [sum][workgroup][cols]
  float* gate_part;             // [gate row][splits][cols], NULL: a gate row's sum is complete in one worker
  int64_t chunk;                // rows of a segment
  int64_t segments;
  int splits;                   // segments of a gate row
};

// 8 values of a column vector, or 8 times `otherwise`
__device__ __forceinline__ f32x8 cols8(const float* p, int col, float otherwise) {
  if (!p) return (f32x8)(otherwise);
  return load8(p + col);
}

// The lanes of one row.  WG lanes per workgroup, L per row.
template <int L, int WG>
struct Team {
  static constexpr int kRows = WG / L;
  static __device__ __forceinline__ int lane() { return threadIdx.x % L; }
  static __device__ __forceinline__ int slot() { return threadIdx.x / L; }

  // sums over the row's lanes, in an order that depends on L alone; `red` is LDS for L > 64 (2 floats a wave, twice: a second
  // call may write while a slow wave still reads what the first left)
  static __device__ __forceinline__ void sum2(float& a, float& b, float* red, int& turn) {
#pragma unroll
    for (int off = (L < 64 ? L : 64) / 2; off > 0; off >>= 1) {
      a += __shfl_xor(a, off, 64);
      b += __shfl_xor(b, off, 64);
    }
    if constexpr (L > 64) {
      constexpr int kWaves = L / 64;
      float* buf = red + turn * 2 * kWaves;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) {
        buf[2 * (threadIdx.x >> 6)] = a;
        buf[2 * (threadIdx.x >> 6) + 1] = b;
      }
      __syncthreads();
      a = b = 0.f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        a += buf[2 * w];
        b += buf[2 * w + 1];
      }
    }
  }
};

// The instance for a number of columns: L lanes, NV chunks of V.  Rows of up to 512 columns have one chunk of 8 a lane.
// (V = 1 only below 8 columns, where a chunk of 8 does not fit.)
template <typename F>
static inline bool norm_dispatch(int cols, F&& f) {
  if (cols < 8) f.template run<1, 8, 1, 256>();
  else if (cols <= 128) f.template run<8, 16, 1, 256>();
  else if (cols <= 256) f.template run<8, 32, 1, 256>();
  else if (cols <= 512) f.template run<8, 64, 1, 256>();
  else if (cols <= 1024) f.template run<8, 64, 2, 256>();
  else if (cols <= 2048) f.template run<8, 256, 1, 256>();
  else if (cols <= 4096) f.template run<8, 256, 2, 256>();
  else if (cols <= 8192) f.template run<8, 512, 2, 512>();
  else return false;
  return true;
}

// One chunk's place: first column, how many leading values a neighbour holds too (V: none are this lane's own).
template <int V, int L>
__device__ __forceinline__ void chunk_place(int j, int lane, int cols, int& col, int& dup) {
  const int at = (j * L + lane) * V;
  col = at <= cols - V ? at : cols - V;
  dup = at < cols ? at - col : V;
}

template <int V, typename T>
__device__ __forceinline__ f32x8 load_chunk(const T* p) {
  if constexpr (V == 8) return load8(p);
  f32x8 v = (f32x8)(0.f);
  v[0] = (float)*p;
  return v;
}
template <int V, typename T>
__device__ __forceinline__ void store_chunk(T* p, f32x8 v) {
  if constexpr (V == 8) store8(p, v);
  else *p = (T)v[0];
}
template <int V>
__device__ __forceinline__ f32x8 cols_chunk(const float* p, int col, float otherwise) {
  if (!p) return (f32x8)(otherwise);
  return load_chunk<V>(p + col);
}

template <int V>
__device__ __forceinline__ uint32_t keep_chunk(uint64_t i, bool aligned, uint2 key, uint32_t thresh) {
  if (!thresh) return 0xffu;
  if constexpr (V == 8) return drop_keep8(i, aligned, key, thresh);
  return drop_keep1(i, key, thresh);
}

// act(gate) in place
template <int V>
__device__ __forceinline__ void activate(f32x8& g, int act) {
  if (act == ADVOC_GATE_SIGMOID)
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] = 1.f / (1.f + expf(-g[k]));
}

// Sums over the columns that this lane owns: f(j, k) gives a term.  `ragged` (uniform) says whether a chunk can be owned in part.
template <int V, int NV, typename F>
__device__ __forceinline__ float own_sum(const int (&dup)[NV], bool ragged, F&& f) {
  float sum = 0.f;
  if (ragged) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int k = 0; k < V; ++k) sum += k >= dup[j] ? f(j, k) : 0.f;
  } else {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      float part = 0.f;
#pragma unroll
      for (int k = 0; k < V; ++k) part += f(j, k);
      sum += dup[j] ? 0.f : part;
    }
  }
  return sum;
}

}  // namespace advoc

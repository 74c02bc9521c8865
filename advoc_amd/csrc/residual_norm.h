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
#include "lanes.h"
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
  float* gate_part;             // [gate row][entries][cols], NULL: a gate row's sum is complete in one worker
  int gate_blocks;              // an entry is a workgroup's: its rows have one segment each, all of one gate row; 0: a segment's
  float* carry;                 // per worker, where workers see several gate rows: see residual_norm_bwd.hip
  int64_t segments;
  int splits;                   // segments of a gate row
};

// The lanes of one row.  WG lanes per workgroup, L per row.
template <int L, int WG>
struct Team {
  static constexpr int kRows = WG / L;
  static __device__ __forceinline__ int lane() { return threadIdx.x % L; }
  // (a wave's rows are said to be uniform: addresses are then a scalar base and a 32-bit offset that all tensors of a type share)
  static __device__ __forceinline__ int slot() {
    if constexpr (L > 64) return 0;
    else if constexpr (L == 64) return __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    else return threadIdx.x / L;
  }

  // A rendezvous of the workgroup that leaves loads in flight; LDS written before it can be read behind it.
  static __device__ __forceinline__ void meet() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

  // sums over the row's lanes, in an order that depends on L alone; `red` is LDS for L > 64 (2 floats a wave, twice: a second
  // call may write while a slow wave still reads what the first left)
  static __device__ __forceinline__ void sum2(float& a, float& b, float* red, int& turn) {
    a = lanes_sum<(L < 64 ? L : 64)>(a);
    b = lanes_sum<(L < 64 ? L : 64)>(b);
    if constexpr (L > 64) {
      constexpr int kWaves = L / 64;
      float* buf = red + turn * 2 * kWaves;
      turn ^= 1;
      if ((threadIdx.x & 63) == 0) {
        buf[2 * (threadIdx.x >> 6)] = a;
        buf[2 * (threadIdx.x >> 6) + 1] = b;
      }
      meet();
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
// V = 1 only below 8 columns, where a chunk of 8 does not fit.
// V = 9 up to an eighth more than a power of two (the 2^n + 1 bins of a transform), where the next instance would leave half of its
// lanes empty or hold two chunks.  Forward | backward in us, 9 columns a lane against 8, bf16 with fp32 residuals and dropout:
//   16384 x 513 fwd 25 | two chunks 32, 3999 x 513 fp32 bwd 21 | 25;   8192 x 2049 fwd 61 | 73, bwd 95 | 124, x 2304 62 | 61, 96 | 110;
//   4096 x 4097 60 | 83, 102 | 140, x 4608 62 | 66, 103 | 113;  1677 rows of fp32: x 2049 23 | 25, 43 | 47, x 4097 43 | 51, 71 | 88.
// Not where a row's share of few rows' time is small or its column sums would come from twice the workgroups, and not by the number
// of rows either (a row's bits depend on its width alone):
//   16384 x 257 17 | 20, 30 | 36, but 256 to 1024 rows 4.7 | 4.1, 11.7 | 10.0, 1677 of fp32 6.3 | 5.8, 15.6 | 15.0;
//   16384 x 1025 (128 lanes) 59 | 72, 90 | 112, but 1024 rows 8.1 | 9.0, 25 | 19, 1677 of fp32 15.5 | 15.3, 31 | 26;
//   16384 x 129 11.5 | 12.9, 24.5 | 22.9.
// Wider rows than 1024 are a workgroup's, 8 columns a lane as far as 512 lanes go: 8192 x 2048 forward 53 us when that was
// chosen, 16 columns a lane 62; 4096 x 4096 51, 78, and backward 88, 97.
template <typename F>
static inline bool norm_dispatch(int cols, F&& f) {
  if (cols < 8) f.template run<1, 8, 1>();
  else if (cols <= 128) f.template run<8, 16, 1>();
  else if (cols <= 256) f.template run<8, 32, 1>();
  else if (cols <= 512) f.template run<8, 64, 1>();
  else if (cols <= 576) f.template run<9, 64, 1>();
  else if (cols <= 1024) f.template run<8, 64, 2>();
  else if (cols <= 2048) f.template run<8, 256, 1>();
  else if (cols <= 2304) f.template run<9, 256, 1>();
  else if (cols <= 4096) f.template run<8, 512, 1>();
  else if (cols <= 4608) f.template run<9, 512, 1>();
  else if (cols <= 8192) f.template run<8, 512, 2>();
  else return false;
  return true;
}

// One chunk's place: which one it is, its first column, how many leading values a neighbour holds too (V: none are this lane's own).
template <int V, int L>
__device__ __forceinline__ void chunk_place(int j, int lane, int cols, int& chunk, int& col, int& dup) {
  const int last = (cols + V - 1) / V - 1, at = (j * L + lane) * V;
  chunk = j * L + lane < last ? j * L + lane : last;
  col = at <= cols - V ? at : cols - V;
  dup = at < cols ? at - col : V;
}

// column `col` of the row that starts at element `at` of `base`
template <typename T>
__device__ __forceinline__ T* row_at(void* base, int64_t at, int col) {
  return reinterpret_cast<T*>(static_cast<char*>(base) + at * (int64_t)sizeof(T) + (uint32_t)col * (uint32_t)sizeof(T));
}
template <typename T>
__device__ __forceinline__ const T* row_at(const void* base, int64_t at, int col) {
  return reinterpret_cast<const T*>(static_cast<const char*>(base) + at * (int64_t)sizeof(T) + (uint32_t)col * (uint32_t)sizeof(T));
}

// NV chunks of a row as they lie in memory: loaded early, converted when they are used
template <typename T, int V, int NV>
struct Raw {
  typename vec8<T>::type v[NV];
  T one[NV];                    // V = 1: the value, V = 9: the last one
  __device__ __forceinline__ void load(const void* base, int64_t at, const int (&col)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const T* p = row_at<T>(base, at, col[j]);
      if constexpr (V >= 8) __builtin_memcpy(&v[j], p, sizeof(v[j]));
      if constexpr (V % 8 == 1) one[j] = p[V - 1];
    }
  }
  __device__ __forceinline__ Vals<V> operator[](int j) const {
    Vals<V> f;
#pragma unroll
    for (int k = 0; k < V; ++k) f[k] = V % 8 == 1 && k == V - 1 ? (float)one[j] : (float)v[j][k & 7];
    return f;
  }
  // The loads have returned behind this.  (A wave may use what it has loaded behind a rendezvous; without this the wait for it would
  // lie there too, and another wave could store to the place first.)
  __device__ __forceinline__ void arrived() {
    static_assert(V >= 8, "wide rows");
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      int w[sizeof(v[j]) / 4];
      __builtin_memcpy(w, &v[j], sizeof(w));
#pragma unroll
      for (int i = 0; i < (int)(sizeof(w) / 4); ++i) asm volatile("" : "+v"(w[i]));
      __builtin_memcpy(&v[j], w, sizeof(w));
      if constexpr (V == 9) {
        int last = 0;
        __builtin_memcpy(&last, &one[j], sizeof(T));
        asm volatile("" : "+v"(last));
        __builtin_memcpy(&one[j], &last, sizeof(T));
      }
    }
  }
};
template <int V, typename T>
__device__ __forceinline__ void store_chunk(T* p, const Vals<V>& v) {
  if constexpr (V >= 8) {
    f32x8 eight;
#pragma unroll
    for (int k = 0; k < 8; ++k) eight[k] = v[k];
    store8(p, eight);
  }
  if constexpr (V % 8 == 1) p[V - 1] = (T)v[V - 1];
}

// Column vectors in LDS: the lanes' chunks side by side, so that 64 lanes read or write theirs without a bank twice.  The first four
// values of every chunk lie together, then the next four, then the ninth (V = 9) or only (V = 1).  The moved-back chunk at the row's
// end is the last one.  A lane reads its columns of the call's vectors for every row (kept in registers they cost the waves that hide
// the loads' latency; from the caches, a round trip per vector and row); an absent vector is staged as its neutral value.
template <int V>
struct Chunks {
  static constexpr int kFours = V / 4, kOnes = V % 4;
  int cols, count;
  __host__ __device__ __forceinline__ explicit Chunks(int cols_) : cols(cols_), count((cols_ + V - 1) / V) {}
  __host__ __device__ __forceinline__ int floats() const { return (count * V + 3) / 4 * 4; }
  __device__ __forceinline__ Vals<V> get(const float* vec, int chunk) const {
    Vals<V> f;
#pragma unroll
    for (int h = 0; h < kFours; ++h) {
      const float4 a = reinterpret_cast<const float4*>(vec)[h * count + chunk];
      f[4 * h] = a.x, f[4 * h + 1] = a.y, f[4 * h + 2] = a.z, f[4 * h + 3] = a.w;
    }
    if constexpr (kOnes) f[V - 1] = vec[4 * kFours * count + chunk];
    return f;
  }
  __device__ __forceinline__ void put(float* vec, int chunk, const Vals<V>& f) const {
#pragma unroll
    for (int h = 0; h < kFours; ++h)
      reinterpret_cast<float4*>(vec)[h * count + chunk] = make_float4(f[4 * h], f[4 * h + 1], f[4 * h + 2], f[4 * h + 3]);
    if constexpr (kOnes) vec[4 * kFours * count + chunk] = f[V - 1];
  }
  // For a workgroup that walks over a vector: f(place in the vector, first column, how many) for this thread's pieces of four values
  // and of one
  template <int WG, typename F>
  __device__ __forceinline__ void walk(F&& f) const {
    for (int q = threadIdx.x; q < kFours * count; q += WG) {
      const int h = kFours > 1 && q >= count;
      f(4 * q, start(q - h * count) + 4 * h, Four());
    }
    if constexpr (kOnes)
      for (int q = threadIdx.x; q < count; q += WG) f(4 * kFours * count + q, start(q) + V - 1, One());
  }
  struct Four { static constexpr int value = 4; };
  struct One { static constexpr int value = 1; };
  __device__ __forceinline__ int start(int chunk) const { return chunk * V <= cols - V ? chunk * V : cols - V; }
};

// (the compiler would carry what it has read of LDS from row to row in registers, and spill)
__device__ __forceinline__ void forget_lds() { asm volatile("" ::: "memory"); }

// Stages N vectors p[i] (where absent: otherwise[i]), a piece of each a lane, all in flight before the first is written.
template <int WG, int V, int N>
__device__ __forceinline__ void stage_vectors(float* lds, const float* const (&p)[N], const float (&otherwise)[N], int cols) {
  const Chunks<V> chunks(cols);
  chunks.template walk<WG>([&](int at, int col, auto n) {
    constexpr int kPiece = decltype(n)::value;
    float v[N][kPiece];
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int k = 0; k < kPiece; ++k) v[i][k] = otherwise[i];
      if (p[i]) __builtin_memcpy(v[i], p[i] + col, sizeof(v[i]));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) __builtin_memcpy(__builtin_assume_aligned(lds + i * chunks.floats() + at, 4 * kPiece), v[i], sizeof(v[i]));
  });
}

// V consecutive floats in global memory
template <int V>
__device__ __forceinline__ Vals<V> floats_at(const float* p) {
  Vals<V> f;
  __builtin_memcpy(f.v, p, sizeof(f.v));
  return f;
}

// what a chunk's elements draw (all kept where nothing is drawn: thresh 0)
template <int V>
__device__ __forceinline__ void draw_chunk(uint32_t (&words)[V], uint64_t i, bool aligned, uint2 key, uint32_t thresh) {
#pragma unroll
  for (int k = 0; k < V; ++k) words[k] = 0;
  if (!thresh) return;
  if constexpr (V >= 8) drop_words<V>(words, i, aligned, key);
  else words[0] = drop_word(i, key);
}

// 1 / (1 + exp(-x)), the exponential as 2^t (1 + the part of -x log2 e that t's rounding dropped, times ln 2): within 6 units in the
// last place wherever the result is a normal number, x >= -87.33 (half the instructions of expf and a division; 16-bit outputs
// round 2^13 units and more away).  Subnormal results become 0.
__device__ __forceinline__ float sigmoid(float x) {
  const float kHigh = 1.44269502f, kLow = 1.92596303e-8f;            // log2 e in two parts
  x = x > 88.f ? 88.f : x;                                           // (1 from 17 on; a NaN stays one)
  const float t = -x * kHigh, rest = fmaf(-x, kLow, fmaf(-x, kHigh, -t));
  const float two_t = __builtin_amdgcn_exp2f(fminf(t, 127.f));
  const float y = __builtin_amdgcn_rcpf(1.f + fmaf(two_t, 0.693147182f * rest, two_t));
  return x < -88.f ? 0.f : y;
}

// act(gate) in place
template <int V>
__device__ __forceinline__ void activate(Vals<V>& g, int act) {
  if (act == ADVOC_GATE_SIGMOID)
#pragma unroll
    for (int k = 0; k < V; ++k) g[k] = sigmoid(g[k]);
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

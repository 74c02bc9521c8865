// Products of 8-bit block-scaled matrices (gfx950): out[m, n] = sum_kb 2^(ea[m, kb] + eb[n, kb]) sum_{k in block kb} a[m, k] b[n, k].
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 values and applies an exponent byte per row and 32 values of k
// to each operand: one instruction per block of 128, the block's byte in all four lane groups, accumulation in its fp32 registers
// across blocks.  Which of the 128 positions of k a lane's 32 bytes are does not matter as long as both operands agree.
// What that instruction adds up is not quite fp32: it aligns the products of eight consecutive k to the largest of them and drops
// what is below 2^-13 of it (measured, also of the unscaled 16x16x32 form).  Against the definition the result is 1.5e-5 off in norm
// -- 1/100 of the rounding of a 16-bit output, so those take it.  An fp32 output is computed EXACTly: the bytes become bf16 with the
// block's power of two applied (v_cvt_scalef32_pk_bf16_fp8) and go through v_mfma_f32_16x16x32_bf16, whose sums are fp32's: 4e-8 off
// in norm, at half the rate.  bf16 holds every 8-bit value with its power of two but at the two ends: below 2^-130 it is rounded to a
// multiple of 2^-133 (blocks whose largest is below 2^-114), and what quantising rounded up to 2^128 (blocks whose largest is above
// 3.1e38) becomes infinite, as it would in fp32.  So a caller's choice of the output's type is one of the sums' too; one or two rows
// (f8_dot_kernel) are summed in fp32 for either, exponents applied to the sums.
// The operand with n rows is the instruction's first: the four accumulators of a lane are then four consecutive n of one output
// row, and for 16-bit outputs the n that two fragments stand for are dealt so that one continues the other: a lane stores 16 bytes,
// four of them 64 consecutive ones, without a turn through LDS.
#include <utility>

#include "lanes.h"
#include "lds_dma.h"
#include "rows.h"

namespace {

using advoc::ceil_div;

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kBlock = 128;

struct Args {
  const uint8_t *a, *a_scale, *b, *b_scale;      // a: m rows, b: n rows
  void* out;
  float* part;                                   // [split][m][n] when the contraction is split
  int64_t m, n;
  int64_t kp, sp;                                // row pitches: kp = 128 blocks, sp = bytes of exponents
  int blocks;                                    // of the contraction
  int per_split;
  int accumulate;
};

__device__ __forceinline__ i32x8 join(int4 lo, int4 hi) {
  return (i32x8){lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
}

// A lane's 32 bytes of one row with their exponent byte, as the matrix instruction takes them
template <int F, bool EXACT>
struct Frag;
template <int F>
struct Frag<F, false> {
  i32x8 q;
  int byte;
  __device__ __forceinline__ Frag(i32x8 v, int b) : q(v), byte(b) {}
};
template <int F>
struct Frag<F, true> {
  bf16x8 v[4];
  __device__ __forceinline__ Frag(i32x8 q, int b) {
    const float scale = __int_as_float(b << 23);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      bf16x2 lo, hi;
      if constexpr (F == ADVOC_E4M3) {
        lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], scale, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(q[i], scale, true);
      } else {
        lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(q[i], scale, false);
        hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(q[i], scale, true);
      }
      v[i / 2][i % 2 * 4] = lo[0];
      v[i / 2][i % 2 * 4 + 1] = lo[1];
      v[i / 2][i % 2 * 4 + 2] = hi[0];
      v[i / 2][i % 2 * 4 + 3] = hi[1];
    }
  }
};

template <int FA, int FB>
__device__ __forceinline__ f32x4 mfma(const Frag<FB, false>& b, const Frag<FA, false>& a, f32x4 c) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b.q, a.q, c, FB, FA, 0, b.byte, 0, a.byte);
}
template <int FA, int FB>
__device__ __forceinline__ f32x4 mfma(const Frag<FB, true>& b, const Frag<FA, true>& a, f32x4 c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[i], a.v[i], c, 0, 0, 0);
  return c;
}

// C consecutive values of one output row, those inside the matrix
template <typename O, int C>
__device__ __forceinline__ void store_part(const Args& g, int64_t row, int64_t col, const float (&v)[C]) {
  if (row >= g.m) return;
  O* p = (O*)g.out + row * g.n + col;
  if (!g.accumulate && col + C <= g.n) {
    O o[C];
#pragma unroll
    for (int k = 0; k < C; ++k) o[k] = (O)v[k];
    __builtin_memcpy(p, o, sizeof(o));
    return;
  }
#pragma unroll
  for (int k = 0; k < C; ++k)
    if (col + k < g.n) p[k] = (O)((g.accumulate ? (float)p[k] : 0.f) + v[k]);
}

// ---- one or two rows: dot products ----
// A wave is one row of b and reads it in pieces of 1024 bytes, 16 a lane, all of up to 8192 in flight together; a lane's products are
// summed in fp32 and take their two exponents once per piece.  Bound by the weights' latency, and with 512 rows of b half of the
// CUs have no workgroup: 1 x 512 x 8192 3.5 us with the weights in a cache, 5.5 to 5.9 from HBM; 1 x 4096 x 4096 3.7 and 6.4.  (Calls
// with the same weights again and again: 3.9 and 4.2, the thin kernel 8.4 and 6.4.)  From three rows on its arithmetic costs more (3 x
// 4096 x 4096: 8.1, thin 6.5).
template <int F>
__device__ __forceinline__ void widen(int word, float (&v)[4]) {
  if constexpr (F == ADVOC_E4M3) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(word, true);
    v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
  } else {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_bf8(word, false), hi = __builtin_amdgcn_cvt_pk_f32_bf8(word, true);
    v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
  }
}

template <typename O, int FA, int FB, int M>
__global__ __launch_bounds__(256) void f8_dot_kernel(Args g) {
  constexpr int kPieces = 8, kPiece = 1024;
  const int lane = threadIdx.x & 63, kp = (int)g.kp;
  const int64_t n = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (n >= g.n) return;
  const uint8_t *b = g.b + n * g.kp, *bs = g.b_scale + n * g.sp;
  float acc[M];
#pragma unroll
  for (int i = 0; i < M; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < kp; k0 += kPieces * kPiece) {
    int4 qb[kPieces];
    int eb[kPieces];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      if (k0 + p * kPiece >= kp) continue;
      const int k = k0 + p * kPiece + lane * 16, at = k < kp ? k : 0;      // (lanes behind the row's end: some piece, times nothing)
      qb[p] = *reinterpret_cast<const int4*>(b + at);
      eb[p] = bs[at / kBlock];
    }
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      if (k0 + p * kPiece >= kp) continue;
      const int k = k0 + p * kPiece + lane * 16, at = k < kp ? k : 0;
      const int words[4] = {qb[p].x, qb[p].y, qb[p].z, qb[p].w};
      float w[16];
#pragma unroll
      for (int i = 0; i < 4; ++i) widen<FB>(words[i], *reinterpret_cast<float(*)[4]>(w + 4 * i));
#pragma unroll
      for (int i = 0; i < M; ++i) {
        const int4 qa = *reinterpret_cast<const int4*>(g.a + i * g.kp + at);
        const int ea = g.a_scale[i * g.sp + at / kBlock], word[4] = {qa.x, qa.y, qa.z, qa.w};
        float dot = 0.f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float v[4];
          widen<FA>(word[q], v);
#pragma unroll
          for (int e = 0; e < 4; ++e) dot = fmaf(v[e], w[4 * q + e], dot);
        }
        const float term = ldexpf(dot, ea + eb[p] - 254);
        acc[i] += k < kp ? term : 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < M; ++i) {
    const float v = advoc::lanes_sum<64>(acc[i]);
    if (lane == 0) {
      O* p = (O*)g.out + i * g.n + n;
      *p = (O)((g.accumulate ? (float)*p : 0.f) + v);
    }
  }
}

// ---- three to 16 rows: the weights are read once, by whoever multiplies them ----
// A workgroup is 16 rows of b; its waves take the blocks of the contraction in turn, straight from memory to registers (lane
// group g the 16-byte pieces g and g + 4 of 16 rows, so that a load covers half lines whole), and meet in LDS in wave order.
// Bound by the weights' latency and, with few columns, by the lines a CU asks for: 4 x 4096 x 4096 6.0 us, 7.2 with the weights from HBM
// (2.3 TB/s), 4 x 512 x 8192 9.4 (32 workgroups).
template <typename O, bool EXACT, int FA, int FB>
__global__ __launch_bounds__(1024) void f8_thin_kernel(Args g) {
  extern __shared__ f32x4 red[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t nrow = n0 + (lane & 15) < g.n ? n0 + (lane & 15) : g.n - 1, mrow = (lane & 15) < g.m ? (lane & 15) : g.m - 1;
  const uint8_t *bp = g.b + nrow * g.kp + (lane >> 4) * 16, *ap = g.a + mrow * g.kp + (lane >> 4) * 16;
  const uint8_t *bs = g.b_scale + nrow * g.sp, *as = g.a_scale + mrow * g.sp;
  f32x4 acc = (f32x4)(0.f);
#pragma unroll 2
  for (int kb = wave; kb < g.blocks; kb += waves) {
    const int4 *p = reinterpret_cast<const int4*>(bp + (int64_t)kb * kBlock), *q = reinterpret_cast<const int4*>(ap + (int64_t)kb * kBlock);
    acc = mfma<FA, FB>(Frag<FB, EXACT>(join(p[0], p[4]), bs[kb]), Frag<FA, EXACT>(join(q[0], q[4]), as[kb]), acc);
  }
  red[wave * 64 + lane] = acc;
  __syncthreads();
  if (wave == 0) {
    f32x4 v = red[lane];
    for (int w = 1; w < waves; ++w) v += red[w * 64 + lane];
    float o[4] = {v[0], v[1], v[2], v[3]};
    store_part<O, 4>(g, lane & 15, n0 + (lane >> 4) * 4, o);
  }
}

// ---- tiles ----
// BM x BN outputs per workgroup, WM x WN per wave.  A block of the contraction of both operands is one of S stages in LDS, fetched by
// LDS-DMA while those before are multiplied.  (Loads that the compiler counts must not follow a DMA in the loop: memory counters
// retire in order, and waiting for such a load waits for the next stage too.  That alone held the first form of this kernel at 0.8
// PFLOP/s.)  The exponents of four blocks are a dword of every row, fetched with the first of them, into one of two places: a row's
// dword is a cache line of its own in a long contraction, as much to ask for as the row's 128 bytes.
// A row's eight 16-byte pieces lie at piece ^ key(row), and lane group g reads pieces g and g + 4: measured without bank conflicts, 4
// cycles for a wave's 16 bytes a lane.  (Pieces 2 g and 2 g + 1 take 8.)
template <typename O, int BM, int BN, int WM, int WN, int S>
struct Tile {
  static constexpr int kWaves = BM / WM * (BN / WN), kFm = WM / 16, kFn = WN / 16;
  static constexpr int kRun = sizeof(O) == 4 ? 1 : 2;            // fragments of b that give a lane 16 consecutive bytes of output
  static constexpr int kRows = BM + BN, kStage = kRows * kBlock, kExp = kRows * 4;
  static constexpr int kLds = S * kStage + 2 * kExp;
  static constexpr int kDma = kRows / 8 / kWaves;                // a DMA instruction fetches 8 rows, or the exponents of 64
  static_assert(kFn % kRun == 0, "whole runs");
  static_assert(kDma * 8 * kWaves == kRows && BM % (8 * kWaves) == 0, "whole DMA instructions per wave and operand");
  static_assert(8 * kWaves % 32 == 0, "the keys of the rows that a lane fetches repeat");
  static_assert(BM % 64 == 0 && BN % 64 == 0 && kWaves >= kRows / 64, "64 rows of one operand per wave's exponent fetch");

  advoc::u32x4s ra, rb, rea, reb;
  const uint8_t* lds;
  unsigned base;
  int lane, wave, wm, wn, spitch;
  int kp, voff_a, voff_b;                // what this lane fetches: its first row of a and of b, the others are 8 kWaves rows on
  int off_a, off_b, piece0, piece1;      // this lane's first rows in a stage, its two pieces of a row

  // which column of a wave's part of the output is row `row` of the matrix instruction's operand for fragment j
  static __device__ __forceinline__ constexpr int place_b(int j, int row) {
    return j / kRun * 16 * kRun + (row >> 2) * 4 * kRun + j % kRun * 4 + (row & 3);
  }
  static __device__ __forceinline__ int key_a(int row) { return (row >> 1) & 7; }
  static __device__ __forceinline__ int key_b(int row) { return kRun == 1 ? key_a(row) : ((row >> 1) & 1) | ((row >> 3) & 3) << 1; }

  __device__ __forceinline__ Tile(const Args& g, const uint8_t* lds_, int64_t m0, int64_t n0) : lds(lds_) {
    lane = threadIdx.x & 63;
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    wm = wave / (BN / WN) * WM;
    wn = wave % (BN / WN) * WN;
    // rows behind the last one read as zeros: their offsets are behind the descriptor's end
    const int64_t mrows = g.m - m0 < BM ? g.m - m0 : BM, nrows = g.n - n0 < BN ? g.n - n0 : BN;
    ra = advoc::dma_rsrc(g.a + m0 * g.kp, (unsigned)(mrows * g.kp));
    rb = advoc::dma_rsrc(g.b + n0 * g.kp, (unsigned)(nrows * g.kp));
    rea = advoc::dma_rsrc(g.a_scale + m0 * g.sp, (unsigned)(mrows * g.sp));
    reb = advoc::dma_rsrc(g.b_scale + n0 * g.sp, (unsigned)(nrows * g.sp));
    base = advoc::lds_address(lds);
    spitch = (int)g.sp;
    kp = (int)g.kp;
    const int first = wave * 8 + (lane >> 3);
    voff_a = first * kp + (((lane & 7) ^ key_a(first)) << 4);
    voff_b = first * kp + (((lane & 7) ^ key_b(first)) << 4);
    // fragment i of a: rows wm + 16 i + lane % 16; fragment j of b: rows wn + place_b(j, lane % 16).  Their keys are lane / 2 % 8 for
    // every fragment
    off_a = wm + (lane & 15);
    off_b = BM + wn + place_b(0, lane & 15);
    piece0 = ((lane >> 4) ^ ((lane >> 1) & 7)) << 4;
    piece1 = piece0 ^ 64;
  }

  // block kb of the contraction, which is part of one that starts at kb0, into stage `slot`
  __device__ __forceinline__ void fetch(int kb, int kb0, int slot) const {
#pragma unroll
    for (int t = 0; t < kDma; ++t) {
      const unsigned to = base + slot * kStage + (t * kWaves + wave) * 1024;
      if (t * 8 * kWaves < BM) advoc::dma16(ra, to, voff_a + t * 8 * kWaves * kp, kb * kBlock);
      else advoc::dma16(rb, to, voff_b + (t * 8 * kWaves - BM) * kp, kb * kBlock);
    }
    if ((kb & 3) && kb != kb0) return;
    const int first = wave % (kRows / 64) * 64;                  // (waves beyond the rows fetch the same dwords again)
    const bool is_a = first < BM;
    advoc::dma4(is_a ? rea : reb, base + S * kStage + (kb >> 2 & 1) * kExp + first * 4, (first + lane - (is_a ? 0 : BM)) * spitch, kb & ~3);
  }

  __device__ __forceinline__ i32x8 bytes(int row) const {      // slot * kRows + row of the stage
    const uint8_t* p = lds + row * kBlock;
    return join(*reinterpret_cast<const int4*>(p + piece0), *reinterpret_cast<const int4*>(p + piece1));
  }
  __device__ __forceinline__ i32x8 bytes_a(int slot, int i) const { return bytes(slot * kRows + off_a + i * 16); }
  __device__ __forceinline__ i32x8 bytes_b(int slot, int j) const { return bytes(slot * kRows + off_b + place_b(j, 0)); }
  __device__ __forceinline__ int exponent_a(int kb, int i) const { return exponent(off_a + i * 16, kb); }
  __device__ __forceinline__ int exponent_b(int kb, int j) const { return exponent(off_b + place_b(j, 0), kb); }
  __device__ __forceinline__ int exponent(int row, int kb) const { return lds[S * kStage + (kb >> 2 & 1) * kExp + row * 4 + (kb & 3)]; }

  // Four lane groups store 64 consecutive bytes of a row together.  Tiles inside the matrix have a loop of their own: next to the
  // element-wise form the compiler cut their 16-byte stores in two (with that, 16384 x 1024 x 1024 took 28 us instead of 22).
  __device__ __forceinline__ void store(const Args& g, int64_t m0, int64_t n0, const f32x4 (&acc)[kFm][kFn]) const {
    constexpr int C = 4 * kRun;
    typedef O run __attribute__((ext_vector_type(C)));
    const bool whole = m0 + BM <= g.m && n0 + BN <= g.n && !g.accumulate;
    if (whole) {
      O* p = (O*)g.out + (m0 + off_a) * g.n + n0 + wn + place_b(0, (lane >> 4) * 4);
#pragma unroll
      for (int i = 0; i < kFm; ++i, p += 16 * g.n)
#pragma unroll
        for (int j = 0; j < kFn; j += kRun) {
          run v;
#pragma unroll
          for (int q = 0; q < C; ++q) v[q] = (O)acc[i][j + q / 4][q % 4];
          __builtin_memcpy(p + place_b(j, 0), &v, sizeof(v));
        }
      return;
    }
#pragma unroll
    for (int i = 0; i < kFm; ++i)
#pragma unroll
      for (int j = 0; j < kFn; j += kRun) {
        float v[C];
#pragma unroll
        for (int q = 0; q < C; ++q) v[q] = acc[i][j + q / 4][q % 4];
        store_part<O, C>(g, m0 + off_a + i * 16, n0 + wn + place_b(j, (lane >> 4) * 4), v);
      }
  }
};

// A workgroup's tile.  Workgroups go to the eight XCDs in turn; each XCD gets a run of the tiles instead, those of one part of a split
// contraction behind one another and within it eight tiles of m for one of n after the other: what runs on an XCD together shares
// its rows in that L2.
struct Place {
  int64_t m0, n0;
  int z;
  __device__ __forceinline__ Place(const Args& g, int bm, int bn) {
    const unsigned total = gridDim.x, q = total / 8, r = total % 8, xcd = blockIdx.x % 8;
    unsigned at = xcd * q + (xcd < r ? xcd : r) + blockIdx.x / 8;
    const unsigned mt = (unsigned)((g.m + bm - 1) / bm), nt = (unsigned)((g.n + bn - 1) / bn);
    z = at / (mt * nt);
    at -= z * mt * nt;
    const unsigned band = at / (8 * nt), first = band * 8, rows = mt - first < 8 ? mt - first : 8;
    at -= band * 8 * nt;
    m0 = (int64_t)(first + at % rows) * bm;
    n0 = (int64_t)(at / rows) * bn;
  }
};

// EXACT, 4096 x 4096 x 4096: 127 us, 1.08 PFLOP/s in tiles of 256 x 128, 142 in tiles of 128 x 128 (a library product of bf16 matrices
// of 8192 reaches 1.41); 1024 x 1024 x 16384: 40 us and 5 for adding up its parts.  A block of 128 x 128 takes a CU 1.1 us: with the
// matrix instructions and conversions left out 0.66 to 1.0 (DMA into LDS and fragments out of it), with only the conversions left out
// 1.0; conversions dealt between the matrix instructions, and wave tiles of 64 x 64 in the same tile, measured the same.
template <typename O, bool EXACT, int FA, int FB, int BM, int BN, int WM, int WN, int S, bool SPLIT>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void f8_tile_kernel(Args g) {
  using T = Tile<O, BM, BN, WM, WN, S>;
  __shared__ __align__(1024) uint8_t lds[T::kLds];
  const Place at(g, BM, BN);
  const int64_t m0 = at.m0, n0 = at.n0;
  const int kb0 = SPLIT ? at.z * g.per_split : 0;
  const int kb1 = SPLIT ? (kb0 + g.per_split < g.blocks ? kb0 + g.per_split : g.blocks) : g.blocks;
  const T t(g, lds, m0, n0);

  f32x4 acc[T::kFm][T::kFn];
#pragma unroll
  for (int i = 0; i < T::kFm; ++i)
#pragma unroll
    for (int j = 0; j < T::kFn; ++j) acc[i][j] = (f32x4)(0.f);

  // Block kb is in registers when its turn comes: the reads of kb + 1 go out in front of the multiplications of kb, and with them the
  // fetch of kb + S into the stage that kb has left.
  i32x8 qa[T::kFm], qb[T::kFn];
  int ea[T::kFm], eb[T::kFn];
  auto read = [&](int slot, int kb) {
#pragma unroll
    for (int j = 0; j < T::kFn; ++j) qb[j] = t.bytes_b(slot, j), eb[j] = t.exponent_b(kb, j);
#pragma unroll
    for (int i = 0; i < T::kFm; ++i) qa[i] = t.bytes_a(slot, i), ea[i] = t.exponent_a(kb, i);
  };
  for (int kb = kb0; kb < kb0 + S && kb < kb1; ++kb) t.fetch(kb, kb0, kb - kb0);
  if (kb0 + S - 1 < kb1) advoc::dma_ring_barrier<(S - 1) * T::kDma>();
  else advoc::dma_ring_barrier<0>();
  read(0, kb0);
  int slot = 0;
#pragma unroll 2
  for (int kb = kb0; kb < kb1; ++kb) {
    // everyone holds block kb, block kb + 1 has landed; S - 2 younger stages may be in flight (but for a fetch of exponents, which is
    // not counted), the last ones are waited for
    if (kb + S - 1 < kb1) advoc::dma_ring_barrier<(S - 2) * T::kDma>();
    else advoc::dma_ring_barrier<0>();
    if (kb + S < kb1) t.fetch(kb + S, kb0, slot);
    slot = slot == S - 1 ? 0 : slot + 1;
    auto multiply = [&](const auto&... b) {
      const Frag<FA, EXACT> fa[] = {{qa[0], ea[0]}, {qa[1], ea[1]}, {qa[T::kFm - 2], ea[T::kFm - 2]}, {qa[T::kFm - 1], ea[T::kFm - 1]}};
      read(slot, kb + 1);      // (behind the last block: what lies there, unused)
#pragma unroll
      for (int i = 0; i < T::kFm; ++i) {
        int j = 0;
        ((acc[i][j] = mfma<FA, FB>(b, fa[i < 2 ? i : i + 4 - T::kFm], acc[i][j]), ++j), ...);
      }
    };
    static_assert(T::kFm == 2 || T::kFm == 4, "two or four fragments of a");
    if constexpr (T::kFn == 2) multiply(Frag<FB, EXACT>(qb[0], eb[0]), Frag<FB, EXACT>(qb[1], eb[1]));
    else multiply(Frag<FB, EXACT>(qb[0], eb[0]), Frag<FB, EXACT>(qb[1], eb[1]), Frag<FB, EXACT>(qb[2], eb[2]), Frag<FB, EXACT>(qb[3], eb[3]));
  }

  Args o = g;
  if constexpr (SPLIT) {
    o.out = g.part + (int64_t)at.z * g.m * g.n;
    o.accumulate = 0;
  }
  t.store(o, m0, n0, acc);
}

// The instruction as assembly, so that it stays between two rendezvous: the compiler sinks the builtin below the second one, out of
// its turn, and moves all accumulators once a block for it (349 against 314 us at 16384 x 4096 x 4096).  It waits the two states that
// a vector instruction's result needs before a matrix instruction reads it.  Whoever reads an accumulator by other means waits for
// the instruction himself and then says settled().
// BYTE_B, BYTE_A: which byte of the exponent registers.
template <int FA, int FB, int BYTE_B, int BYTE_A>
__device__ __forceinline__ void mfma_in_place(f32x4& c, const i32x8& b, const i32x8& a, int bytes_b, int bytes_a) {
  asm volatile(
      "s_nop 1\n\t"
      "v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%7,%8,0] op_sel_hi:[%9,%10,0] cbsz:%5 blgp:%6"
      : "+v"(c)
      : "v"(b), "v"(a), "v"(bytes_b), "v"(bytes_a), "n"(FB), "n"(FA), "n"(BYTE_B & 1), "n"(BYTE_A & 1), "n"(BYTE_B >> 1), "n"(BYTE_A >> 1));
}
// acc[i][j] += b[j] a[i] for every i, j; the exponents of four fragments are the bytes of one register
template <int FA, int FB, int FM, int FN, int... K>
__device__ __forceinline__ void mfma_all(f32x4 (&acc)[FM][FN], const i32x8 (&b)[FN], const i32x8 (&a)[FM], const int (&eb)[FN / 4],
                                         const int (&ea)[FM / 4], std::integer_sequence<int, K...>) {
  (mfma_in_place<FA, FB, K % FN % 4, K / FN % 4>(acc[K / FN][K % FN], b[K % FN], a[K / FN], eb[K % FN / 4], ea[K / FN / 4]), ...);
}
__device__ __forceinline__ void settled(f32x4& c) { asm volatile("" : "+v"(c)); }

// 256 x 256 outputs, eight waves of 128 x 64, the 8-bit instruction.  Two waves share a SIMD and take turns: while the waves of one
// half of the workgroup read the fragments of a block from LDS (24 reads of 16 bytes a lane: 768 cycles of the CU's 128 bytes a
// cycle for four waves), the other half multiplies the block before (32 instructions of 32 cycles), with a rendezvous between; the
// matrix pipe has work in both halves of a block's time.  16384 x 4096 x 4096: 231 us, 2.38 PFLOP/s; 4096 x 4096 x 8192: 100 us, 2.74
// (a library product of 8-bit matrices of 8192 reaches 2.69).  Stamped in a run of 1500 calls: 2.07 GHz, a tile of 32 blocks 4600 cycles
// to begin, 107000 for its blocks, 4400 to store; the matrix cores' 2048 cycles a block are 0.61 of those.  What the rest is: with
// reads, fetches and stores left out a call still took 205 of the 243 us it took then, so most of it is the way an instruction with
// two exponent registers issues and the rendezvous between the halves, a sixth the fragments and fetches that show through.
template <typename O, int FA, int FB>
__global__ __launch_bounds__(512) void f8_big_kernel(Args g) {
  using T = Tile<O, 256, 256, 128, 64, 2>;
  __shared__ __align__(1024) uint8_t lds[T::kLds];
  const Place at(g, 256, 256);
  const int64_t m0 = at.m0, n0 = at.n0;
  const T t(g, lds, m0, n0);

  f32x4 acc[T::kFm][T::kFn];
#pragma unroll
  for (int i = 0; i < T::kFm; ++i)
#pragma unroll
    for (int j = 0; j < T::kFn; ++j) acc[i][j] = (f32x4)(0.f);
  i32x8 a[T::kFm], b[T::kFn];
  int ea[T::kFm / 4], eb[T::kFn / 4];

  auto read = [&](int kb) {
    const int slot = kb & 1;
#pragma unroll
    for (int j = 0; j < T::kFn; ++j) b[j] = t.bytes_b(slot, j);
#pragma unroll
    for (int i = 0; i < T::kFm; ++i) a[i] = t.bytes_a(slot, i);
#pragma unroll
    for (int i = 0; i < T::kFm; i += 4)
      ea[i / 4] = t.exponent_a(kb, i) | t.exponent_a(kb, i + 1) << 8 | t.exponent_a(kb, i + 2) << 16 | t.exponent_a(kb, i + 3) << 24;
#pragma unroll
    for (int j = 0; j < T::kFn; j += 4)
      eb[j / 4] = t.exponent_b(kb, j) | t.exponent_b(kb, j + 1) << 8 | t.exponent_b(kb, j + 2) << 16 | t.exponent_b(kb, j + 3) << 24;
  };
  auto multiply = [&]() {
    __builtin_amdgcn_s_setprio(1);
    mfma_all<FA, FB>(acc, b, a, eb, ea, std::make_integer_sequence<int, T::kFm * T::kFn>());
    __builtin_amdgcn_s_setprio(0);
  };
  auto fetch = [&](int kb) {
    if (kb >= g.blocks) return;
    t.fetch(kb, 0, kb & 1);
  };
  auto meet = [&](bool landed) {      // my reads have arrived and, with `landed`, what I fetched lies in LDS
    __builtin_amdgcn_sched_barrier(0);
    if (landed) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  };

  // Both halves run one program, the second one rendezvous behind: rendezvous 2 kb + 1 ends the first half's reads of block kb and
  // the second's multiplication of kb - 1, rendezvous 2 kb + 2 the second's reads of kb and the first's multiplication.  Behind
  // rendezvous 2 kb nobody reads block kb - 1 any more, so both halves fetch kb + 1 into its place there, and it has to lie there
  // at rendezvous 2 kb + 2.
  const bool late = t.wave >= 4;      // waves w and w + 4 share a SIMD
  fetch(0);
  meet(true);
  if (late) {
    fetch(1);
    meet(false);
  }
  for (int kb = 0; kb < g.blocks; ++kb) {
    read(kb);
    if (!late) fetch(kb + 1);      // behind the reads: the address unit takes longer over these than LDS over those
    meet(late);
    if (late) fetch(kb + 2);
    multiply();
    meet(!late);
  }
  if (!late) meet(false);
  asm volatile("s_nop 15\n\ts_nop 15");      // the last accumulators, before anything reads them
#pragma unroll
  for (int i = 0; i < T::kFm; ++i)
#pragma unroll
    for (int j = 0; j < T::kFn; ++j) settled(acc[i][j]);
  t.store(g, m0, n0, acc);
}

// the parts of a split contraction, added in order
template <typename O>
__global__ __launch_bounds__(256) void f8_fold_kernel(const float* __restrict__ part, O* out, int64_t count, int splits, int accumulate) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (int64_t)gridDim.x * 256) {
    float v = accumulate ? (float)out[i] : 0.f;
    for (int s = 0; s < splits; ++s) v += part[s * count + i];
    out[i] = (O)v;
  }
}

enum { kDot, kThin, kTile64, kTile128, kTile256 };      // kTile256: 256 x 256, EXACT 256 x 128

struct Plan {
  int form, splits, per_split;
};

// One or two rows: dot products (2 x 4096 x 4096: 5.7 us, thin 6.5; 2 x 16384 x 4096: 17.7, thin 17.0).  Otherwise the cheapest
// estimate.  A CU takes 0.7 us for a block of 128 x 128 outputs (EXACT 1.06), 0.4 times that for one of 64 x 64 (EXACT 0.36), twice
// for one of 256 x 256 (EXACT 1.56 times for one of 256 x 128), whichever its neighbours do, and four blocks' time to begin and end a
// tile; the CUs take tiles in rounds of 256.  A contraction split in s has s times the tiles with 1 / s of the blocks, and 3 us and a write and a read of its partial results more.
// The thin kernel (up to 16 rows) takes 0.08 us and 4.2 ns a row for a block of 16 columns, 256 of them together.
// Measured, in us.  64 | 128 | 256, 16-bit outputs:  1024 x 1024 x 1024: 5.5 | 8.1;  2048 x 1024 x 4096: 19 | 25 | 48;  2048 x 2048 x
// 4096: 33 | 24 | 48;  4096 x 2048 x 4096: 63 | 47 | 50;  4096 x 2560 x 4096: 128: 68, 256: 52;  16384 x 1024 x 1024: 39 | 31 | 21.
// 128 x 128 | 256 x 128, fp32 outputs:  4096 x 4096 x 4096: 142 | 127;  16384 x 4096 x 4096: 550 | 458;  2048 x 2048 x 4096: 36 | 48;
// 1024 x 1024 x 16384 in 4 | 8 parts: 48 | 46.
// fp32 outputs in 1 | 2 | 4 | 8 parts:  1024 x 1024 x 16384: 112 | 65 | 43 | 50 (128), 57 | 47 | 49 (64);  512 x 512 x 2048: 9.1 |
// 9.1 | 8.6 | 11.6 (64).
// Thin | 64 in parts:  16 x 512 x 8192: 12.7 | 9.3;  16 x 4096 x 4096: 8.0 | 9.3;  16 x 1000 x 1000: 3.7 | 5.2;  with 17 to 64 rows
// the thin form lost nearly everywhere (64 x 512 x 8192: 28.8 | 9.8).
Plan make_plan(int64_t m, int64_t n, int blocks, bool exact) {
  Plan p = {m <= 2 ? kDot : kThin, 1, blocks};
  if (m <= 2) return p;
  const double block_us = exact ? 1.06 : 0.7, fold_us = 8.0 * m * n / 5e6;
  double best = m <= 16 ? (0.08 + 0.0042 * m) * blocks * ceil_div(n, 16 * 256) : 1e30;
  const int64_t sides[] = {64, 128, 256}, wide = exact ? 128 : 256;      // the largest tile: 256 x wide
  const double costs[] = {exact ? 0.36 : 0.4, 1.0, exact ? 1.56 : 2.0};
  for (int form = kTile64; form <= kTile256; ++form) {
    const int64_t side = sides[form - kTile64], tiles = ceil_div(m, side) * ceil_div(n, form == kTile256 ? wide : side);
    const int most = form == kTile256 && !exact ? 1 : 16;
    for (int s = 1; s == 1 || (s <= most && s <= blocks / 8); s *= 2) {
      const int per = (int)ceil_div(blocks, s), parts = (int)ceil_div(blocks, per);
      const double us = block_us * costs[form - kTile64] * ceil_div(tiles * parts, 256) * (per + 4) + (parts > 1 ? 3.0 + fold_us * parts : 0.0);
      if (us < best) best = us, p = {form, parts, per};
    }
  }
  return p;
}

unsigned thin_waves(int blocks) { return blocks >= 16 ? 16 : blocks >= 8 ? 8 : blocks >= 4 ? 4 : 2; }

// A launch ends at 2^32 - 1 work-items.  (m and n are at most 2^31 each and less than 2^42 tiles of 64 x 64 together: no overflow.)
bool launch_ok(const Plan& p, int64_t m, int64_t n, int blocks, bool exact) {
  int64_t items = 0;
  switch (p.form) {
    case kDot: items = ceil_div(n, 4) * 256; break;
    case kThin: items = ceil_div(n, 16) * 64 * thin_waves(blocks); break;
    case kTile64: items = ceil_div(m, 64) * ceil_div(n, 64) * p.splits * 256; break;
    case kTile128: items = ceil_div(m, 128) * ceil_div(n, 128) * p.splits * 512; break;
    case kTile256: items = ceil_div(m, 256) * ceil_div(n, exact ? 128 : 256) * p.splits * 512; break;
  }
  return items <= 0xffffffffLL;
}

template <typename O, bool EXACT, int FA, int FB, int BM, int BN, int WM, int WN, int S, bool SPLIT>
int run_tile(const Args& g, int splits, hipStream_t stream) {
  constexpr int kThreads = BM / WM * (BN / WN) * 64;
  const dim3 grid((unsigned)(ceil_div(g.m, BM) * ceil_div(g.n, BN) * splits));
  hipLaunchKernelGGL((f8_tile_kernel<O, EXACT, FA, FB, BM, BN, WM, WN, S, SPLIT>), grid, dim3(kThreads), 0, stream, g);
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

template <typename O, bool EXACT, int FA, int FB, bool SPLIT>
int run_form(const Args& g, const Plan& p, hipStream_t stream) {
  if constexpr (EXACT)
    if (p.form == kTile256) return run_tile<O, EXACT, FA, FB, 256, 128, 64, 64, 3, SPLIT>(g, p.splits, stream);
  return p.form == kTile128 ? run_tile<O, EXACT, FA, FB, 128, 128, 64, 32, 4, SPLIT>(g, p.splits, stream)
                            : run_tile<O, EXACT, FA, FB, 64, 64, 32, 32, 4, SPLIT>(g, p.splits, stream);
}

template <typename O, bool EXACT, int FA, int FB>
int run(const Args& g, const Plan& p, hipStream_t stream) {
  ADVOC_CLEAR_LAUNCH_ERROR();
  if (p.form == kThin) {
    const unsigned waves = thin_waves(g.blocks);
    hipLaunchKernelGGL((f8_thin_kernel<O, EXACT, FA, FB>), dim3((unsigned)ceil_div(g.n, 16)), dim3(64 * waves), waves * 1024, stream, g);
    ADVOC_RETURN_IF_LAUNCH_FAILED();
    return ADVOC_OK;
  }
  if (p.form == kDot) {
    const dim3 grid((unsigned)ceil_div(g.n, 4));
    if (g.m == 1) hipLaunchKernelGGL((f8_dot_kernel<O, FA, FB, 1>), grid, dim3(256), 0, stream, g);
    else hipLaunchKernelGGL((f8_dot_kernel<O, FA, FB, 2>), grid, dim3(256), 0, stream, g);
    ADVOC_RETURN_IF_LAUNCH_FAILED();
    return ADVOC_OK;
  }
  if constexpr (!EXACT) {
    if (p.form == kTile256) {
      const dim3 grid((unsigned)(ceil_div(g.m, 256) * ceil_div(g.n, 256)));
      hipLaunchKernelGGL((f8_big_kernel<O, FA, FB>), grid, dim3(512), 0, stream, g);
      ADVOC_RETURN_IF_LAUNCH_FAILED();
      return ADVOC_OK;
    }
  }
  const int rc = p.splits == 1 ? run_form<O, EXACT, FA, FB, false>(g, p, stream) : run_form<float, EXACT, FA, FB, true>(g, p, stream);
  if (rc != ADVOC_OK || p.splits == 1) return rc;
  const int64_t count = g.m * g.n, blocks = ceil_div(count, 256);
  ADVOC_CLEAR_LAUNCH_ERROR();
  hipLaunchKernelGGL(f8_fold_kernel<O>, dim3((unsigned)(blocks > 4096 ? 4096 : blocks)), dim3(256), 0, stream, g.part, (O*)g.out, count,
                     p.splits, g.accumulate);
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

template <typename O>
int run_formats(const Args& g, const Plan& p, int fa, int fb, hipStream_t stream) {
  constexpr bool kExact = sizeof(O) == 4;
  if (fa == ADVOC_E4M3)
    return fb == ADVOC_E4M3 ? run<O, kExact, ADVOC_E4M3, ADVOC_E4M3>(g, p, stream) : run<O, kExact, ADVOC_E4M3, ADVOC_E5M2>(g, p, stream);
  return fb == ADVOC_E4M3 ? run<O, kExact, ADVOC_E5M2, ADVOC_E4M3>(g, p, stream) : run<O, kExact, ADVOC_E5M2, ADVOC_E5M2>(g, p, stream);
}

}  // namespace

extern "C" int64_t advoc_matmul_nt_f8_workspace_bytes(int64_t m, int64_t n, int64_t k, int32_t out_dtype) {
  if (m <= 0 || n <= 0 || k <= 0 || k > 0x7fffff00LL) return 0;
  const Plan p = make_plan(m, n, (int)ceil_div(k, kBlock), out_dtype == ADVOC_F32);
  return p.splits > 1 ? 4 * p.splits * m * n : 0;
}

extern "C" int advoc_matmul_nt_f8(const uint8_t* a, const uint8_t* a_scale, int32_t a_format, const uint8_t* b, const uint8_t* b_scale,
                                  int32_t b_format, void* out, int32_t out_dtype, int32_t accumulate, int64_t m, int64_t n, int64_t k,
                                  void* workspace, int64_t workspace_bytes, advoc_stream_t stream) {
  if (m < 0 || n < 0 || k <= 0) return ADVOC_ERR_BAD_SHAPE;
  if (m == 0 || n == 0) return ADVOC_OK;
  if (!a || !a_scale || !b || !b_scale || !out) return ADVOC_ERR_NULL;
  if ((a_format != ADVOC_E4M3 && a_format != ADVOC_E5M2) || (b_format != ADVOC_E4M3 && b_format != ADVOC_E5M2))
    return ADVOC_ERR_UNSUPPORTED;
  if (!advoc::dtype_ok(out_dtype) || (accumulate && out_dtype != ADVOC_F32)) return ADVOC_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) return ADVOC_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(a_scale) | reinterpret_cast<uintptr_t>(b_scale)) & 3) return ADVOC_ERR_UNSUPPORTED;
  // 256 rows of an operand lie behind one 32-bit descriptor; tiles are numbered in 31 bits
  if (k > 8000000 || m > (1LL << 31) || n > (1LL << 31) || ceil_div(m, 64) * ceil_div(n, 64) > 0x3fffffff) return ADVOC_ERR_UNSUPPORTED;
  Args g = {a, a_scale, b, b_scale, out, static_cast<float*>(workspace), m, n};
  g.blocks = (int)ceil_div(k, kBlock);
  g.kp = (int64_t)g.blocks * kBlock;
  g.sp = ceil_div(g.blocks, 4) * 4;
  g.accumulate = accumulate != 0;
  Plan p = make_plan(m, n, g.blocks, out_dtype == ADVOC_F32);
  if (p.splits > 1 && (!workspace || workspace_bytes < 4 * p.splits * m * n)) p.splits = 1, p.per_split = g.blocks;
  if (p.splits > 1 && (reinterpret_cast<uintptr_t>(workspace) & 3)) return ADVOC_ERR_UNSUPPORTED;
  if (!launch_ok(p, m, n, g.blocks, out_dtype == ADVOC_F32)) return ADVOC_ERR_UNSUPPORTED;
  g.per_split = p.per_split;
  if (out_dtype == ADVOC_F32) return run_formats<float>(g, p, a_format, b_format, advoc::as_stream(stream));
  if (out_dtype == ADVOC_BF16) return run_formats<__bf16>(g, p, a_format, b_format, advoc::as_stream(stream));
  return run_formats<_Float16>(g, p, a_format, b_format, advoc::as_stream(stream));
}

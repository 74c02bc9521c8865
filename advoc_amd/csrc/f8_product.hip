// Products of 8-bit block-scaled matrices (gfx950): out[m, n] = sum_kb 2^(ea[m, kb] + eb[n, kb]) sum_{k in block kb} a[m, k] b[n, k].
//
// v_mfma_scale_f32_16x16x128_f8f6f4 multiplies 16 x 128 by 128 x 16 values and applies an exponent byte per row and 32 values of k
// to each operand: one instruction per block of 128, the block's byte in all four lane groups, accumulation in its fp32 registers
// across blocks.  Which of the 128 positions of k a lane's 32 bytes are does not matter as long as both operands agree, so a lane
// takes 32 consecutive bytes.
// What that instruction adds up is not quite fp32: it aligns the products of eight consecutive k to the largest of them and drops
// what is below 2^-13 of it (measured, also of the unscaled 16x16x32 form).  Against the definition the result is 1.5e-5 off in norm
// -- 1/100 of the rounding of a 16-bit output, so those take it.  An fp32 output is computed EXACTly: the bytes become bf16 with the
// block's power of two applied (v_cvt_scalef32_pk_bf16_fp8; every 8-bit value is a bf16 value) and go through
// v_mfma_f32_16x16x32_bf16, whose sums are fp32's: 4e-8 off in norm, at half the rate.
// The operand with n rows is the instruction's first: the four accumulators of a lane are then four consecutive n of one output
// row, and the n that a wave's fragments stand for are dealt so that a lane's fragments continue them (16 consecutive n with four
// fragments): the output leaves in 32- or 64-byte pieces without a turn through LDS.
#include "rows.h"
#include "lds_dma.h"

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

// c consecutive values of one output row
template <typename O>
__device__ __forceinline__ void store_run(const Args& g, int64_t row, int64_t col, const float* v, int c) {
  if (row >= g.m) return;
  O* p = (O*)g.out + row * g.n + col;
  for (int k = 0; k < c; ++k)
    if (col + k < g.n) p[k] = (O)((g.accumulate ? (float)p[k] : 0.f) + v[k]);
}

// ---- few rows (m <= 64): the weights are read once, by whoever multiplies them ----
// A workgroup is 16 rows of b; its waves take the blocks of the contraction in turn, straight from memory to registers (a lane's 32
// bytes; 16 lanes x 4 groups cover 16 lines), and meet in LDS in wave order.
template <typename O, bool EXACT, int FA, int FB, int MF>
__global__ __launch_bounds__(1024) void f8_thin_kernel(Args g) {
  extern __shared__ f32x4 red[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
  const int64_t n0 = (int64_t)blockIdx.x * 16;
  const int64_t nrow = n0 + (lane & 15) < g.n ? n0 + (lane & 15) : g.n - 1;
  const uint8_t* bp = g.b + nrow * g.kp + (lane >> 4) * 32;
  const uint8_t* bs = g.b_scale + nrow * g.sp;
  const uint8_t *ap[MF], *as[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) {
    const int64_t r = i * 16 + (lane & 15) < g.m ? i * 16 + (lane & 15) : g.m - 1;
    ap[i] = g.a + r * g.kp + (lane >> 4) * 32;
    as[i] = g.a_scale + r * g.sp;
  }
  f32x4 acc[MF];
#pragma unroll
  for (int i = 0; i < MF; ++i) acc[i] = (f32x4)(0.f);
#pragma unroll 2
  for (int kb = wave; kb < g.blocks; kb += waves) {
    const int4* p = reinterpret_cast<const int4*>(bp + (int64_t)kb * kBlock);
    const Frag<FB, EXACT> b(join(p[0], p[1]), bs[kb]);
#pragma unroll
    for (int i = 0; i < MF; ++i) {
      const int4* q = reinterpret_cast<const int4*>(ap[i] + (int64_t)kb * kBlock);
      acc[i] = mfma<FA, FB>(b, Frag<FA, EXACT>(join(q[0], q[1]), as[i][kb]), acc[i]);
    }
  }
#pragma unroll
  for (int i = 0; i < MF; ++i) red[(wave * MF + i) * 64 + lane] = acc[i];
  __syncthreads();
  for (int e = threadIdx.x; e < MF * 64; e += blockDim.x) {
    f32x4 v = red[e];
    for (int w = 1; w < waves; ++w) v += red[w * MF * 64 + e];
    const int l = e & 63;
    const float o[4] = {v[0], v[1], v[2], v[3]};
    store_run<O>(g, (e >> 6) * 16 + (l & 15), n0 + (l >> 4) * 4, o, 4);
  }
}

// ---- tiles ----
// BM x BN outputs per workgroup, WM x WN per wave.  A block of the contraction of both operands is a stage of LDS, fetched by
// LDS-DMA while the stage before is multiplied.  A row's eight 16-byte pieces lie at piece ^ key(row): the 16 rows that a
// fragment reads together have keys 0 ... 7 twice, so its reads spread over all banks.
template <typename O, bool EXACT, int FA, int FB, int BM, int BN, int WM, int WN, bool SPLIT>
__global__ __launch_bounds__(BM / WM * (BN / WN) * 64) void f8_tile_kernel(Args g) {
  constexpr int kWaves = BM / WM * (BN / WN), kFm = WM / 16, kFn = WN / 16;
  constexpr int kShift = kFn == 4 ? 4 : 3;                       // rows of b four apart in the instruction are 4 kFn apart
  static_assert(kFn == 2 || kFn == 4, "a wave is two or four fragments of b wide");
  constexpr int kStage = (BM + BN) * kBlock;
  constexpr int kDma = (BM + BN) / 8 / kWaves;                   // a DMA instruction fetches 8 rows
  static_assert(kDma * 8 * kWaves == BM + BN && BM % (8 * kWaves) == 0, "whole DMA instructions per wave and operand");
  __shared__ __align__(1024) uint8_t lds[2 * kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t m0 = (int64_t)blockIdx.x * BM, n0 = (int64_t)blockIdx.y * BN;
  const int kb0 = SPLIT ? blockIdx.z * g.per_split : 0;
  const int kb1 = SPLIT ? (kb0 + g.per_split < g.blocks ? kb0 + g.per_split : g.blocks) : g.blocks;
  const int wm = (wave / (BN / WN)) * WM, wn = (wave % (BN / WN)) * WN;

  // rows behind the last one read as zeros: their offsets are behind the descriptor's end
  const int64_t mrows = g.m - m0 < BM ? g.m - m0 : BM, nrows = g.n - n0 < BN ? g.n - n0 : BN;
  const advoc::u32x4s ra = advoc::dma_rsrc(g.a + m0 * g.kp, (unsigned)(mrows * g.kp));
  const advoc::u32x4s rb = advoc::dma_rsrc(g.b + n0 * g.kp, (unsigned)(nrows * g.kp));
  const unsigned base = advoc::lds_address(lds);
  int voff[kDma];
#pragma unroll
  for (int t = 0; t < kDma; ++t) {
    const int row = (t * kWaves + wave) * 8 + (lane >> 3);       // of a, then of b
    const int r = row < BM ? row : row - BM;
    const int key = row < BM ? r & 7 : (r & 3) | ((r >> kShift) & 1) << 2;
    voff[t] = r * (int)g.kp + (((lane & 7) ^ key) << 4);
  }
  auto fetch = [&](int kb, int stage) {
#pragma unroll
    for (int t = 0; t < kDma; ++t) {
      const bool is_a = t * 8 * kWaves < BM;
      advoc::dma16(is_a ? ra : rb, base + stage * kStage + (t * kWaves + wave) * 1024, voff[t], kb * kBlock);
    }
  };

  // exponents: a dword is four blocks of a row
  const uint8_t *as[kFm], *bs[kFn];
  int arow[kFm], brow[kFn];
#pragma unroll
  for (int i = 0; i < kFm; ++i) {
    arow[i] = wm + i * 16 + (lane & 15);
    const int64_t r = m0 + arow[i] < g.m ? m0 + arow[i] : g.m - 1;
    as[i] = g.a_scale + r * g.sp;
  }
#pragma unroll
  for (int j = 0; j < kFn; ++j) {
    brow[j] = wn + ((lane & 15) >> 2) * 4 * kFn + j * 4 + (lane & 3);
    const int64_t r = n0 + brow[j] < g.n ? n0 + brow[j] : g.n - 1;
    bs[j] = g.b_scale + r * g.sp;
  }

  f32x4 acc[kFm][kFn];
#pragma unroll
  for (int i = 0; i < kFm; ++i)
#pragma unroll
    for (int j = 0; j < kFn; ++j) acc[i][j] = (f32x4)(0.f);

  if (kb0 < kb1) fetch(kb0, 0);
  for (int kb = kb0; kb < kb1; ++kb) {
    const int stage = (kb - kb0) & 1;
    advoc::dma_ring_barrier<0>();
    int sa[kFm], sb[kFn];
#pragma unroll
    for (int i = 0; i < kFm; ++i) sa[i] = as[i][kb];
#pragma unroll
    for (int j = 0; j < kFn; ++j) sb[j] = bs[j][kb];
    if (kb + 1 < kb1) fetch(kb + 1, stage ^ 1);
    const uint8_t* s = lds + stage * kStage;
    const int piece = (lane >> 4) * 2;
    auto bytes = [&](int row, int key) {
      const uint8_t* p = s + row * kBlock;
      return join(*reinterpret_cast<const int4*>(p + ((piece ^ key) << 4)), *reinterpret_cast<const int4*>(p + (((piece + 1) ^ key) << 4)));
    };
    auto frag_b = [&](int j) {
      return Frag<FB, EXACT>(bytes(BM + brow[j], (brow[j] & 3) | ((brow[j] >> kShift) & 1) << 2), sb[j]);
    };
    auto multiply = [&](const auto&... b) {
#pragma unroll
      for (int i = 0; i < kFm; ++i) {
        const Frag<FA, EXACT> a(bytes(arow[i], arow[i] & 7), sa[i]);
        int j = 0;
        ((acc[i][j] = mfma<FA, FB>(b, a, acc[i][j]), ++j), ...);
      }
    };
    if constexpr (kFn == 2) multiply(frag_b(0), frag_b(1));
    else multiply(frag_b(0), frag_b(1), frag_b(2), frag_b(3));
  }

  Args o = g;
  if constexpr (SPLIT) {
    o.out = g.part + (int64_t)blockIdx.z * g.m * g.n;
    o.accumulate = 0;
  }
#pragma unroll
  for (int i = 0; i < kFm; ++i) {
    float v[4 * kFn];
#pragma unroll
    for (int j = 0; j < kFn; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[4 * j + e] = acc[i][j][e];
    store_run<O>(o, m0 + arow[i], n0 + wn + (lane >> 4) * 4 * kFn, v, 4 * kFn);
  }
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

enum { kThin, kTile64, kTile128, kTile256 };

struct Plan {
  int form, splits, per_split;
};

Plan make_plan(int64_t m, int64_t n, int blocks) {
  Plan p = {kThin, 1, blocks};
  if (m <= 64) return p;
  const int64_t t256 = ceil_div(m, 256) * ceil_div(n, 256), t128 = ceil_div(m, 128) * ceil_div(n, 128);
  p.form = t256 >= 192 ? kTile256 : t128 >= 64 ? kTile128 : kTile64;
  const int64_t tiles = p.form == kTile256 ? t256 : p.form == kTile128 ? t128 : ceil_div(m, 64) * ceil_div(n, 64);
  int64_t splits = 512 / tiles;
  if (splits > blocks / 8) splits = blocks / 8;
  if (splits > 1 && p.form != kTile256) {
    p.per_split = (int)ceil_div(blocks, splits);
    p.splits = (int)ceil_div(blocks, p.per_split);
  }
  return p;
}

template <typename O, bool EXACT, int FA, int FB, int BM, int BN, int WM, int WN, bool SPLIT>
int run_tile(const Args& g, int splits, hipStream_t stream) {
  constexpr int kThreads = BM / WM * (BN / WN) * 64;
  const dim3 grid((unsigned)ceil_div(g.m, BM), (unsigned)ceil_div(g.n, BN), (unsigned)splits);
  hipLaunchKernelGGL((f8_tile_kernel<O, EXACT, FA, FB, BM, BN, WM, WN, SPLIT>), grid, dim3(kThreads), 0, stream, g);
  ADVOC_RETURN_IF_LAUNCH_FAILED();
  return ADVOC_OK;
}

template <typename O, bool EXACT, int FA, int FB>
int run(const Args& g, const Plan& p, hipStream_t stream) {
  ADVOC_CLEAR_LAUNCH_ERROR();
  if (p.form == kThin) {
    const unsigned waves = g.blocks >= 16 ? 16 : g.blocks >= 8 ? 8 : g.blocks >= 4 ? 4 : 2;
    const int mf = g.m <= 16 ? 1 : g.m <= 32 ? 2 : 4;
    const dim3 grid((unsigned)ceil_div(g.n, 16)), block(64 * waves);
    const unsigned lds = waves * mf * 1024;
    if (mf == 1) hipLaunchKernelGGL((f8_thin_kernel<O, EXACT, FA, FB, 1>), grid, block, lds, stream, g);
    else if (mf == 2) hipLaunchKernelGGL((f8_thin_kernel<O, EXACT, FA, FB, 2>), grid, block, lds, stream, g);
    else hipLaunchKernelGGL((f8_thin_kernel<O, EXACT, FA, FB, 4>), grid, block, lds, stream, g);
    ADVOC_RETURN_IF_LAUNCH_FAILED();
    return ADVOC_OK;
  }
  if (p.form == kTile256) return run_tile<O, EXACT, FA, FB, 256, 256, 128, 64, false>(g, 1, stream);
  if (p.splits == 1)
    return p.form == kTile128 ? run_tile<O, EXACT, FA, FB, 128, 128, 64, 64, false>(g, 1, stream)
                              : run_tile<O, EXACT, FA, FB, 64, 64, 32, 32, false>(g, 1, stream);
  const int rc = p.form == kTile128 ? run_tile<float, EXACT, FA, FB, 128, 128, 64, 64, true>(g, p.splits, stream)
                                    : run_tile<float, EXACT, FA, FB, 64, 64, 32, 32, true>(g, p.splits, stream);
  if (rc != ADVOC_OK) return rc;
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

extern "C" int64_t advoc_matmul_nt_f8_workspace_bytes(int64_t m, int64_t n, int64_t k) {
  if (m <= 0 || n <= 0 || k <= 0 || k > 0x7fffff00LL) return 0;
  const Plan p = make_plan(m, n, (int)ceil_div(k, kBlock));
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
  // 256 rows of an operand lie behind one 32-bit descriptor; tiles of n are a grid's second dimension
  if (k > 8000000 || m > 64LL * 0x7fffffff || n > 64LL * 65535) return ADVOC_ERR_UNSUPPORTED;
  Args g = {a, a_scale, b, b_scale, out, static_cast<float*>(workspace), m, n};
  g.blocks = (int)ceil_div(k, kBlock);
  g.kp = (int64_t)g.blocks * kBlock;
  g.sp = ceil_div(g.blocks, 4) * 4;
  g.accumulate = accumulate != 0;
  Plan p = make_plan(m, n, g.blocks);
  if (p.splits > 1 && (!workspace || workspace_bytes < 4 * p.splits * m * n)) p.splits = 1, p.per_split = g.blocks;
  if (p.splits > 1 && (reinterpret_cast<uintptr_t>(workspace) & 3)) return ADVOC_ERR_UNSUPPORTED;
  g.per_split = p.per_split;
  if (out_dtype == ADVOC_F32) return run_formats<float>(g, p, a_format, b_format, advoc::as_stream(stream));
  if (out_dtype == ADVOC_BF16) return run_formats<__bf16>(g, p, a_format, b_format, advoc::as_stream(stream));
  return run_formats<_Float16>(g, p, a_format, b_format, advoc::as_stream(stream));
}

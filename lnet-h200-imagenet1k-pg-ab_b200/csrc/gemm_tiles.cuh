// Tiled matrix product on tcgen05 with an epilogue:
//   C[m, n] = sum_k A(m, k) B(n, k),  y = f(C * scales + bias) + residual,
// for operands stored with k contiguous (K-major) or with m or n contiguous
// (MN-major), in bf16 or (K-major) e4m3, fp32 accumulators in TMEM.
//
// A persistent CTA, or a pair of CTAs on two SMs (cta_group::2), walks output
// tiles.  Warp 0 loads: 128-byte wide k blocks by TMA (128-byte swizzle) into a
// ring of stages.  Warp 1 issues the MMAs, one elected thread of the pair's
// first CTA.  Warps 2 to 9 take finished accumulators out of TMEM (two
// accumulators, so that the next tile's MMAs run meanwhile) through the
// epilogue.
//
// Why a pair: a 128 x 256 tile of one SM reads 48 KB per 512 clocks of MMA, 94
// bytes a clock, more than an SM's share of L2; the pair's 256 x 256 tile splits
// B between the two SMs, 64 bytes a clock for the same work.
//
// A last wave that would leave SMs idle is split along k: those tiles' fp32 sums
// go to memory and a second kernel joins them.
//
// Bound by the tensor cores: 16384 x 2048 -> 8192 bf16 with GELU and the stored
// pre-activation, and the gradient's two products, take 345 us each (1590 of 1661
// TFLOP/s measured; tensor pipe 0.90 active without GELU).  The epilogue takes 2.9 us a 256 x 256 tile (5.9 with GELU and
// pre-activation) behind the next tile's MMAs, and bounds the kernel where K is
// below about 768 (1536).
//
// Every wait is bounded: a role whose wait gives up marks the CTA as failed, all
// roles leave their loops, and tiles that were not finished are written as NaN.
#pragma once

#include <cuda.h>
#include <cuda_fp8.h>

#include "rows.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace lnet {

constexpr int kTileM = 128;             // rows of A a CTA holds
// 8 warps leave shared memory for 6 stages: 16, with 5, cost 4 % at K = 2048 and took 8 % off GELU at
// K = 96.  Asking for the next block from TMEM before working on one changed nothing.
constexpr int kEpiWarps = 8;
constexpr int kTileThreads = 64 + 32 * kEpiWarps;  // loader, MMA issuer, epilogue warps
// A try of 1 us suspends the waiting threads; shorter ones changed no time, and their polling takes
// power from the tensor cores.
constexpr uint32_t kTileWaitHint = 1000u;
constexpr uint32_t kTileWaitLimit = 1000000u;  // tries: about a second
constexpr int kTileSmemLimit = 227 * 1024;

enum LinearActivation { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// rcp.approx (1 ulp) of both values
__device__ __forceinline__ Pair rcp_fast(Pair x) {
  float a, b;
  unpair(x, a, b);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(a));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(b));
  return pair(a, b);
}
__device__ __forceinline__ Pair pair_of(float v) { return pair(v, v); }

// The normal distribution's tail Q(|a|) and the exponential e = e^(-a^2 / 2) that it shares with
// the density: Q = p(t) e / 2, t = 1 / (1 + 0.3275911 |a| / sqrt 2), with the polynomial 7.1.26 of
// Abramowitz and Stegun, Handbook of Mathematical Functions (absolute error of erf below 1.5e-7).
// With erff and expf an epilogue took longer than the MMAs of K = 2048.
__device__ __forceinline__ Pair normal_tail(Pair a, Pair &e) {
  float x, y;
  unpair(a, x, y);
  e = exp2_fast(a * a * pair_of(-0.72134752f));
  const Pair t = rcp_fast(fma(pair(fabsf(x), fabsf(y)), pair_of(0.23164190f), pair_of(1.f)));
  Pair p = fma(pair_of(0.5307027145f), t, pair_of(-0.7265760135f));
  p = fma(p, t, pair_of(0.7107068705f));
  p = fma(p, t, pair_of(-0.142248368f));
  p = fma(p, t, pair_of(0.127414796f));
  return p * t * e;
}

// f(a): SiLU a / (1 + e^-a), GELU a Phi(a) = a (1 + erf(a / sqrt 2)) / 2, in fp32.
template <int ACT>
__device__ __forceinline__ Pair act_value(Pair a) {
  float x, y;
  if (ACT == kActRelu) {
    unpair(a, x, y);
    return pair(x < 0.f ? 0.f : x, y < 0.f ? 0.f : y);  // keeps NaN
  }
  if (ACT == kActSilu)
    return a * rcp_fast(exp2_fast(a * pair_of(-kLog2e)) + pair_of(1.f));
  if (ACT == kActGelu) {
    Pair e;
    const Pair q = normal_tail(a, e), above = fma(q, pair_of(-1.f), pair_of(1.f));
    float q0, q1, u0, u1;
    unpair(a, x, y), unpair(q, q0, q1), unpair(above, u0, u1);
    return a * pair(x < 0.f ? q0 : u0, y < 0.f ? q1 : u1);
  }
  return a;
}
// f'(a)
template <int ACT>
__device__ __forceinline__ Pair act_slope(Pair a) {
  float x, y;
  if (ACT == kActRelu) {
    unpair(a, x, y);
    return pair(x > 0.f ? 1.f : (x != x ? x : 0.f), y > 0.f ? 1.f : (y != y ? y : 0.f));
  }
  if (ACT == kActSilu) {
    const Pair s = rcp_fast(exp2_fast(a * pair_of(-kLog2e)) + pair_of(1.f));
    return s * fma(a, fma(s, pair_of(-1.f), pair_of(1.f)), pair_of(1.f));
  }
  if (ACT == kActGelu) {
    Pair e;
    const Pair q = normal_tail(a, e), half = fma(q, pair_of(-1.f), pair_of(0.5f));
    float h0, h1;
    unpair(a, x, y), unpair(half, h0, h1);
    const Pair phi = e * pair_of(0.39894228f);  // Phi = 1/2 +- (1/2 - Q)
    return fma(a, phi, pair(copysignf(h0, x), copysignf(h1, y)) + pair_of(0.5f));
  }
  return pair_of(1.f);
}

// f of N values (N even): the choice of f is made once, outside the loop over them.
template <int N, int ACT>
__device__ __forceinline__ void act_each(float *v) {
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const Pair r = act_value<ACT>(pair(v[i], v[i + 1]));
    unpair(r, v[i], v[i + 1]);
  }
}
template <int N>
__device__ __forceinline__ void act_values(float *v, int act) {
  switch (act) {
    case kActRelu: act_each<N, kActRelu>(v); break;
    case kActSilu: act_each<N, kActSilu>(v); break;
    case kActGelu: act_each<N, kActGelu>(v); break;
    default: break;
  }
}

struct TileEpilogue {
  __nv_bfloat16 *out;             // [M, N]
  __nv_bfloat16 *pre;             // C * scales + bias in bf16, or null
  const __nv_bfloat16 *bias;      // [N] or null
  const __nv_bfloat16 *residual;  // [M, N] or null
  const float *row_scale, *col_scale;  // [M], [N] or both null
  int act;
};

// Division of n < 2^31 by a number known before the launch (Granlund and Montgomery, Division by
// Invariant Integers using Multiplication): the roles find their next tile with it, and the loader,
// one thread, was held up by the dozens of dependent instructions of plain divisions.
struct FastDiv {
  uint32_t d, m;
  int s;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div), s(0) {
    while ((1ull << s) < div) ++s;
    m = (uint32_t)(((1ull << 32) * ((1ull << s) - div)) / div + 1);
  }
  __device__ __forceinline__ int quotient(int n) const {
    return (int)((__umulhi(m, (uint32_t)n) + (uint32_t)n) >> s);
  }
};

struct TileArgs {
  CUtensorMap a, b;
  TileEpilogue e;
  int64_t M, N;
  FastDiv by_band, by_last, by_splits;  // 8 n_tiles, rows of the last band, splits
  // Tiles 0 to full - 1 take all of k; the others are split into `splits` ranges of k each, whose
  // fp32 sums go to `partial` [tile - full][split][CTA][BN / 4][128 rows][4].
  int m_tiles, n_tiles, full, splits, kblocks;
  float *partial;
};

template <int CTAS, int BN, bool FP8>
struct TileShape {
  static constexpr int NB = BN / CTAS;  // rows of B a CTA holds
  static constexpr int A_BYTES = kTileM * 128, B_BYTES = NB * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  // a warp's 32 x 32 bf16 block on its way to memory, and its columns' bias and scale (fp32)
  static constexpr int WARP_COLS = BN / (kEpiWarps / 4) >= 32 ? BN / (kEpiWarps / 4) : 32;
  static constexpr int WARP_BYTES = 2048 + 2 * WARP_COLS * 4;
  static constexpr int OTHER = 1024 /* alignment */ + 512 /* barriers */ + kEpiWarps * WARP_BYTES;
  static constexpr int STAGES =
      (kTileSmemLimit - OTHER) / STAGE > 8 ? 8 : (kTileSmemLimit - OTHER) / STAGE;
  static constexpr int SMEM = STAGES * STAGE + OTHER;
  static constexpr int TMEM = 2 * BN < 32 ? 32 : 2 * BN;
};

// ---------------------------------------------------------------- epilogue
// A warp holds a 32 x 32 block of a, a lane a row.  Rows of a block lie N elements apart, so a lane
// that moved its own row would touch 32 lines an instruction; the block goes through shared memory
// (64-byte rows, 16-byte units exchanged so that neither side has bank conflicts) and moves as 4
// lanes a row, or, where rows are not 16-byte aligned, as 8, 16 or 32 lanes a row.
__device__ __forceinline__ uint4 *block_unit(uint8_t *block, int row, int unit) {
  return reinterpret_cast<uint4 *>(block + row * 64 + ((unit ^ ((row >> 1) & 3)) << 4));
}
__device__ __forceinline__ __nv_bfloat16 *block_element(uint8_t *block, int row, int col) {
  return reinterpret_cast<__nv_bfloat16 *>(block_unit(block, row, col >> 3)) + (col & 7);
}
// Where a lane's units of a warp's rows lie: row (lane / 4) + 8 i, unit lane % 4 of 32 columns.
struct BlockRows {
  int64_t at;   // element offset of the lane's first unit in column 0
  int64_t row0, M, N;
  uint32_t ok;  // bit i: row i of the lane is inside
};
__device__ __forceinline__ BlockRows block_rows(int64_t row0, int64_t M, int64_t N) {
  const int lane = threadIdx.x & 31;
  BlockRows b{(row0 + (lane >> 2)) * N + (lane & 3) * 8, row0, M, N, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) b.ok |= (row0 + (lane >> 2) + 8 * i < M ? 1u : 0u) << i;
  return b;
}
// The block to or from memory, U (4, 2 or 1) elements a lane, U rows an instruction.
template <int U>
using UnitWord = std::conditional_t<U == 4, uint2, std::conditional_t<U == 2, uint32_t, uint16_t>>;
template <int U>
__device__ __forceinline__ void block_out(uint8_t *block, __nv_bfloat16 *dst, const BlockRows &b,
                                          int64_t col) {
  using W = UnitWord<U>;
  const int lane = threadIdx.x & 31, r0 = lane / (32 / U), c = lane % (32 / U) * U;
  if (col + c >= b.N) return;
  const int rows = (int)min((int64_t)32, b.M - b.row0);
  __nv_bfloat16 *p = dst + (b.row0 + r0) * b.N + col + c;
#pragma unroll 8
  for (int r = r0; r < rows; r += U, p += U * b.N)
    *reinterpret_cast<W *>(p) = *reinterpret_cast<const W *>(block_element(block, r, c));
}
template <int U>
__device__ __forceinline__ void block_in(uint8_t *block, const __nv_bfloat16 *src, const BlockRows &b,
                                         int64_t col) {
  using W = UnitWord<U>;
  constexpr int Q = U == 1 ? 16 : 32 / U;  // loads on their way at once
  const int lane = threadIdx.x & 31, r0 = lane / (32 / U), c = lane % (32 / U) * U;
  if (col + c >= b.N) return;
  const int rows = (int)min((int64_t)32, b.M - b.row0);
  const __nv_bfloat16 *p = src + (b.row0 + r0) * b.N + col + c;
#pragma unroll
  for (int s = 0; s < 32; s += Q * U) {
    W q[Q];
#pragma unroll
    for (int i = 0; i < Q; ++i)
      q[i] = r0 + s + i * U < rows
                 ? __ldg(reinterpret_cast<const W *>(p + (int64_t)(s + i * U) * b.N))
                 : W{};
#pragma unroll
    for (int i = 0; i < Q; ++i)
      *reinterpret_cast<W *>(block_element(block, r0 + s + i * U, c)) = q[i];
  }
}
template <int UNIT>
__device__ __forceinline__ void block_store(uint8_t *block, const float *v, __nv_bfloat16 *dst,
                                            const BlockRows &b, int64_t col) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    RowChunk<__nv_bfloat16, 8> c;
    c.put(v + 8 * u);
    *block_unit(block, lane, u) = c.raw;
  }
  __syncwarp();
  if constexpr (UNIT == 8) {
    __nv_bfloat16 *p = dst + b.at + col;
    const bool in = col + (lane & 3) * 8 < b.N;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (in && (b.ok >> i & 1))
        *reinterpret_cast<uint4 *>(p) = *block_unit(block, i * 8 + (lane >> 2), lane & 3);
      p += 8 * b.N;
    }
  } else {
    block_out<UNIT>(block, dst, b, col);
  }
  __syncwarp();
}
// 16-byte units of a block of `src`: issued early, used by block_add.
__device__ __forceinline__ void block_fetch(const __nv_bfloat16 *src, uint4 *u, const BlockRows &b,
                                            int64_t col) {
  const __nv_bfloat16 *p = src + b.at + col;
  const bool in = col + (threadIdx.x & 3) * 8 < b.N;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    u[i] = make_uint4(0, 0, 0, 0);
    if (in && (b.ok >> i & 1)) u[i] = __ldg(reinterpret_cast<const uint4 *>(p));
    p += 8 * b.N;
  }
}
// v += the block of `src`, whose units are in `u` where UNIT is 8.
template <int UNIT>
__device__ __forceinline__ void block_add(uint8_t *block, const __nv_bfloat16 *src, const uint4 *u,
                                          float *v, const BlockRows &b, int64_t col) {
  const int lane = threadIdx.x & 31;
  if constexpr (UNIT == 8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) *block_unit(block, i * 8 + (lane >> 2), lane & 3) = u[i];
  } else {
    block_in<UNIT>(block, src, b, col);
  }
  __syncwarp();
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    RowChunk<__nv_bfloat16, 8> c;
    c.raw = *block_unit(block, lane, k);
    float w[8];
    c.get(w);
#pragma unroll
    for (int i = 0; i < 8; i += 2)
      unpair(pair(v[8 * k + i], v[8 * k + i + 1]) + pair(w[i], w[i + 1]), v[8 * k + i],
             v[8 * k + i + 1]);
  }
  __syncwarp();
}

// The block's 32 columns of bias and scale come from shared memory (`bias`, `scale`; scale only
// with row scales); `res` holds the residual's units.  Every lane of the warp takes part.
template <int UNIT>
__device__ __forceinline__ void tile_epilogue(const TileEpilogue &e, const BlockRows &b,
                                              float *v, int64_t col, float row_scale,
                                              const float *bias, const float *scale,
                                              uint8_t *block, const uint4 *res) {
  if (e.col_scale) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 s = *reinterpret_cast<const float4 *>(scale + j);
      const Pair rs = pair(row_scale, row_scale);
      unpair(pair(v[j], v[j + 1]) * rs * pair(s.x, s.y), v[j], v[j + 1]);
      unpair(pair(v[j + 2], v[j + 3]) * rs * pair(s.z, s.w), v[j + 2], v[j + 3]);
    }
  }
  if (e.bias) {
#pragma unroll
    for (int j = 0; j < 32; j += 4) {
      const float4 q = *reinterpret_cast<const float4 *>(bias + j);
      unpair(pair(v[j], v[j + 1]) + pair(q.x, q.y), v[j], v[j + 1]);
      unpair(pair(v[j + 2], v[j + 3]) + pair(q.z, q.w), v[j + 2], v[j + 3]);
    }
  }
  if (e.pre) block_store<UNIT>(block, v, e.pre, b, col);
  act_values<32>(v, e.act);
  if (e.residual) block_add<UNIT>(block, e.residual, res, v, b, col);
  block_store<UNIT>(block, v, e.out, b, col);
}

// Bias and scale of `n` columns from `col` on into a warp's shared memory (0 past N).
__device__ __forceinline__ void stage_columns(const TileEpilogue &e, int64_t N, int64_t col, int n,
                                              float *bias, float *scale) {
  for (int c = threadIdx.x & 31; c < n; c += 32) {
    if (e.bias) bias[c] = col + c < N ? load_f(e.bias, col + c) : 0.f;
    if (e.col_scale) scale[c] = col + c < N ? __ldg(e.col_scale + col + c) : 0.f;
  }
}

// Unit t of the work: tile, and its k blocks [k0, k1) (split < 0: all of them).
struct TileUnit {
  int tile, split, k0, k1;
};
__device__ __forceinline__ TileUnit unit_at(const TileArgs &p, int t) {
  if (t < p.full) return TileUnit{t, -1, 0, p.kblocks};
  const int u = t - p.full, tile = p.by_splits.quotient(u), split = u - tile * p.splits;
  return TileUnit{p.full + tile, split, (int)((int64_t)p.kblocks * split / p.splits),
                  (int)((int64_t)p.kblocks * (split + 1) / p.splits)};
}

// Tile order: bands of 8 row tiles, down the rows inside a column, so that a
// wave of CTAs shares few operand tiles in L2.
constexpr int kBand = 8;
__device__ __forceinline__ void tile_at(const TileArgs &p, int t, int &m, int &n) {
  const int band = p.by_band.quotient(t);
  t -= band * kBand * p.n_tiles;
  const bool last = p.m_tiles - band * kBand < kBand;
  n = last ? p.by_last.quotient(t) : t / kBand;
  m = band * kBand + t - n * (last ? (int)p.by_last.d : kBand);
}

// UNIT: elements that [M, N] tensors are moved by (8, 4, 2 or 1), of which N is a multiple and to which
// they are aligned.  In one kernel the paths of the four slowed one another: 6329 x 2010 -> 4557 with
// residual and pre-activation took 203 us, and takes 155 (4558 columns 118, 4556 111, 4560 103).
template <int CTAS, int BN, bool A_MN, bool B_MN, bool FP8, int UNIT>
__global__ void __launch_bounds__(kTileThreads, 1)
tile_gemm_kernel(const __grid_constant__ TileArgs p) {
  using S = TileShape<CTAS, BN, FP8>;
  constexpr int NB = S::NB, STAGES = S::STAGES;
  constexpr int KB = FP8 ? 128 : 64;  // elements of a k block (128 bytes)
  static_assert(!B_MN || NB % 64 == 0, "an MN-major operand comes in panels of 64");
  extern __shared__ uint8_t smem_raw[];
  uint8_t *smem = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                              ~(uintptr_t)1023);
  uint64_t *bars = reinterpret_cast<uint64_t *>(smem + STAGES * S::STAGE);
  uint64_t *full = bars, *empty = bars + STAGES, *acc_full = bars + 2 * STAGES,
           *acc_empty = acc_full + 2, *drain = acc_empty + 2;
  uint32_t *tslot = reinterpret_cast<uint32_t *>(drain + 1);
  uint8_t *warp_smem = smem + STAGES * S::STAGE + 512;
  volatile uint32_t *failed = tslot + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CTAS == 2 ? sm100::cluster_rank() : 0;
  const bool leader = rank == 0;
  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      sm100::mbar_init(full + i, 1);
      sm100::mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      sm100::mbar_init(acc_full + i, 1);
      sm100::mbar_init(acc_empty + i, CTAS * kEpiWarps);
    }
    sm100::mbar_init(drain, 1);
    *failed = 0;
    sm100::fence_barrier_init();
  }
  __syncwarp();
  if (warp == 1) {
    if (CTAS == 2) {
      sm100::tmem_alloc_pair(tslot, S::TMEM);
      sm100::tmem_relinquish_pair();
    } else {
      sm100::tmem_alloc(tslot, S::TMEM);
      sm100::tmem_relinquish();
    }
  }
  sm100::tc_fence_before();
  if (CTAS == 2) sm100::cluster_sync();
  __syncthreads();
  sm100::tc_fence_after();
  const uint32_t tmem = *tslot;
  const int units = p.full + (p.m_tiles * p.n_tiles - p.full) * p.splits;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    bool ok = sm100::mbar_try_wait(bar, parity, kTileWaitHint);
    for (uint32_t i = 0; i < kTileWaitLimit && !ok && !*failed; ++i)
      ok = sm100::mbar_try_wait(bar, parity, kTileWaitHint);
    if (!ok) *failed = 1;
    return ok;
  };

  if (warp == 0 && lane == 0) {  // ---------------------------------------- loader
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    // the barriers of the pair's first CTA
    const uint32_t full0 = CTAS == 2 ? sm100::map_to_rank(full, 0) : sm100::smem_u32(full);
    for (int t = first; t < units && ok; t += step) {
      const TileUnit w = unit_at(p, t);
      int m, n;
      tile_at(p, w.tile, m, n);
      const int am = (m * CTAS + (int)rank) * kTileM, bn = n * BN + (int)rank * NB;
      for (int k = w.k0; k < w.k1; ++k) {
        if (issued >= STAGES && !(ok = wait(empty + stage, phase ^ 1))) break;
        if (leader) sm100::mbar_arrive_expect_tx(full + stage, CTAS * S::STAGE);
        const uint32_t bar = full0 + stage * 8;
        const uint32_t da = sm100::smem_u32(smem + stage * S::STAGE), db = da + S::A_BYTES;
        if (A_MN) {
#pragma unroll
          for (int q = 0; q < kTileM / 64; ++q)
            sm100::tma_load_2d_group<CTAS>(da + q * 8192, &p.a, bar, am + 64 * q, k * KB);
        } else {
          sm100::tma_load_2d_group<CTAS>(da, &p.a, bar, k * KB, am);
        }
        if (B_MN) {
#pragma unroll
          for (int q = 0; q < (NB >= 64 ? NB / 64 : 1); ++q)
            sm100::tma_load_2d_group<CTAS>(db + q * 8192, &p.b, bar, bn + 64 * q, k * KB);
        } else {
          sm100::tma_load_2d_group<CTAS>(db, &p.b, bar, k * KB, bn);
        }
        ++issued;
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
    }
    // No CTA leaves while a copy or an arrival is on its way to it: every stage in use is
    // waited for once more (after a failure, its copies alone, again with a limit).
    for (int i = 0; i < min(issued, STAGES); ++i) {
      const int back = issued - 1 - i;
      uint64_t *e = empty + back % STAGES, *f = full + back % STAGES;
      const uint32_t par = (uint32_t)(back / STAGES) & 1;
      if (!(ok && wait(e, par)) && leader)
        sm100::mbar_wait_bounded(f, par, 100000u);
    }
  } else if (warp == 1 && lane == 0 && leader) {  // ------------------------ MMA issuer
    constexpr uint32_t idesc =
        (1u << 4) | (FP8 ? 0u : (1u << 7) | (1u << 10)) | ((A_MN ? 1u : 0u) << 15) |
        ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) |
        ((uint32_t)((CTAS * kTileM) >> 4) << 24);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int t = first; t < units && ok; t += step) {
      const TileUnit w = unit_at(p, t);
      if (!(ok = wait(acc_empty + acc, acc_phase ^ 1))) break;
      sm100::tc_fence_after();
      for (int k = w.k0; k < w.k1; ++k) {
        if (!(ok = wait(full + stage, phase))) break;
        sm100::tc_fence_after();
        const uint32_t da = sm100::smem_u32(smem + stage * S::STAGE), db = da + S::A_BYTES;
        const uint64_t ad = A_MN ? sm100::make_desc_sw128_mn(da, 8192) : sm100::make_desc_sw128(da);
        const uint64_t bd = B_MN ? sm100::make_desc_sw128_mn(db, 8192) : sm100::make_desc_sw128(db);
#pragma unroll
        for (int s = 0; s < 4; ++s)  // 32 bytes of k, or 16 k rows of 128 bytes
          sm100::mma_group<CTAS, FP8>(tmem + acc * BN, ad + s * (A_MN ? 128 : 2),
                                      bd + s * (B_MN ? 128 : 2), idesc, k > w.k0 || s > 0);
        sm100::mma_commit_group<CTAS>(empty + stage);
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
      if (!ok) break;
      sm100::mma_commit_group<CTAS>(acc_full + acc);
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
    if (!ok) {  // the MMAs in flight end before TMEM is freed
      sm100::mma_commit_group<CTAS>(drain);
      sm100::mbar_wait_bounded(drain, 0, 100000u);
    }
  } else if (warp >= 2) {  // ----------------------------------------------- epilogue
    const int ew = warp - 2, quad = warp & 3, group = ew >> 2;
    constexpr int COLS = S::WARP_COLS;
    const bool mine = group * COLS < BN;
    uint8_t *block = warp_smem + ew * S::WARP_BYTES;
    float *bias = reinterpret_cast<float *>(block + 2048), *scale = bias + COLS;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = first; t < units; t += step) {
      const TileUnit w = unit_at(p, t);
      int m, n;
      tile_at(p, w.tile, m, n);
      const int64_t row0 = (int64_t)(m * CTAS + (int)rank) * kTileM + quad * 32;
      const int64_t col0 = (int64_t)n * BN + group * COLS;
      const bool in = mine && row0 < p.M && col0 < p.N;
      const BlockRows rows = block_rows(row0, p.M, p.N);
      float rs = 1.f;
      if (in && w.split < 0) {  // while the accumulators are not there yet
        stage_columns(p.e, p.N, col0, COLS, bias, scale);
        if (p.e.row_scale && row0 + lane < p.M) rs = __ldg(p.e.row_scale + row0 + lane);
        if (p.e.residual && row0 + lane < p.M) {  // the residual's lines on their way to L2
          const __nv_bfloat16 *line = p.e.residual + (row0 + lane) * p.N + col0;
          for (int c = 0; c < COLS && col0 + c < p.N; c += 64)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(line + c));
        }
      }
      __syncwarp();
      if (ok) ok = wait(acc_full + acc, acc_phase);
      ok = __all_sync(0xFFFFFFFFu, ok);
      sm100::tc_fence_after();
      // The accumulators are free once they are in registers, before the stores.
      auto release = [&] {
        sm100::tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CTAS == 2)
            sm100::mbar_arrive_rank(acc_empty + acc, 0);
          else
            sm100::mbar_arrive(acc_empty + acc);
        }
      };
      if (!in) release();
#pragma unroll 1
      for (int c = 0; in && c < COLS && col0 + c < p.N; c += 32) {
        uint4 ru[4];
        if (w.split < 0 && UNIT == 8 && p.e.residual) block_fetch(p.e.residual, ru, rows, col0 + c);
        float v[32];
        if (ok) {
          sm100::tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + acc * BN + group * COLS + c, v);
          sm100::tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(0x7FC00000u);
        }
        if (c + 32 >= COLS || col0 + c + 32 >= p.N) release();
        if (w.split < 0) {
          tile_epilogue<UNIT>(p.e, rows, v, col0 + c, rs, bias + c, scale + c, block, ru);
        } else {
          float4 *out = reinterpret_cast<float4 *>(p.partial) +
                        (((int64_t)(w.tile - p.full) * p.splits + w.split) * CTAS + rank) *
                            (BN / 4 * kTileM) +
                        (group * COLS + c) / 4 * kTileM + quad * 32 + lane;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            out[j * kTileM] = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        }
        __syncwarp();
      }
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
  }
  __syncwarp();
  sm100::tc_fence_before();
  __syncthreads();
  if (CTAS == 2) sm100::cluster_sync();  // the pair's barriers and TMEM stay until both are done
  if (warp == 1) {
    sm100::tc_fence_after();
    if (CTAS == 2)
      sm100::tmem_dealloc_pair(tmem, S::TMEM);
    else
      sm100::tmem_dealloc(tmem, S::TMEM);
  }
}

// The tiles whose k was split: their sums, added in split order, through the epilogue.  A warp takes
// a 32 x 32 block.
constexpr int kJoinThreads = 128;
template <int CTAS, int BN, int UNIT>
__global__ void __launch_bounds__(kJoinThreads) tile_join_kernel(const __grid_constant__ TileArgs p) {
  constexpr int BLOCKS = CTAS * 4 * (BN / 32);  // of a tile
  __shared__ __align__(16) uint8_t smem[kJoinThreads / 32][2048 + 2 * 32 * 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int id = blockIdx.x * (kJoinThreads / 32) + warp;
  const int tile = id / BLOCKS, b = id - tile * BLOCKS;
  if (p.full + tile >= p.m_tiles * p.n_tiles) return;
  const int cta = b / (4 * (BN / 32)), quad = b / (BN / 32) % 4, c = b % (BN / 32) * 32;
  int m, n;
  tile_at(p, p.full + tile, m, n);
  const int64_t row0 = (int64_t)(m * CTAS + cta) * kTileM + quad * 32;
  const int64_t col = (int64_t)n * BN + c;
  if (row0 >= p.M || col >= p.N) return;
  uint8_t *block = smem[warp];
  float *bias = reinterpret_cast<float *>(block + 2048), *scale = bias + 32;
  stage_columns(p.e, p.N, col, 32, bias, scale);
  __syncwarp();
  uint4 ru[4];
  const BlockRows rows = block_rows(row0, p.M, p.N);
  if (UNIT == 8 && p.e.residual) block_fetch(p.e.residual, ru, rows, col);
  const float rs = p.e.row_scale && row0 + lane < p.M ? __ldg(p.e.row_scale + row0 + lane) : 1.f;
  float v[32];
#pragma unroll
  for (int j = 0; j < 32; ++j) v[j] = 0.f;
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s) {
    const float4 *in = reinterpret_cast<const float4 *>(p.partial) +
                       (((int64_t)tile * p.splits + s) * CTAS + cta) * (BN / 4 * kTileM) +
                       c / 4 * kTileM + quad * 32 + lane;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float4 u = __ldg(in + j * kTileM);
      v[4 * j] += u.x, v[4 * j + 1] += u.y, v[4 * j + 2] += u.z, v[4 * j + 3] += u.w;
    }
  }
  tile_epilogue<UNIT>(p.e, rows, v, col, rs, bias, scale, block, ru);
}

// ---------------------------------------------------------------- host side
// One operand: `mn` rows (or columns) by `k`, `pitch` elements between rows of memory.
struct TileOperand {
  const void *ptr;
  int64_t mn, k, pitch;
  bool mn_major;
};

inline int tile_tensor_map(CUtensorMap *map, const TileOperand &o, bool fp8, int box_mn) {
  PFN_cuTensorMapEncodeTiled_v12000 encode;
  LNET_TRY(tensor_map_encoder(&encode));
  const int elem = fp8 ? 1 : 2;
  const cuuint64_t dims[2] = {(cuuint64_t)(o.mn_major ? o.mn : o.k),
                              (cuuint64_t)(o.mn_major ? o.k : o.mn)};
  const cuuint64_t strides[1] = {(cuuint64_t)(o.pitch * elem)};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / elem), (cuuint32_t)(o.mn_major ? 64 : box_mn)};
  const cuuint32_t ones[2] = {1, 1};
  const CUresult r = encode(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                            2, const_cast<void *>(o.ptr), dims, strides, box, ones,
                            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                            CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS)
    return fail(LNET_ERR_CUDA, "tensor map of a %lld x %lld operand (pitch %lld) failed: %d",
                (long long)o.mn, (long long)o.k, (long long)o.pitch, (int)r);
  return LNET_OK;
}

}  // namespace lnet

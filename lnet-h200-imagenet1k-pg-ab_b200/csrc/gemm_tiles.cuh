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
// Every wait is bounded: a role whose wait gives up marks the CTA as failed, all
// roles leave their loops, and tiles that were not finished are written as NaN.
#pragma once

#include <cuda.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "sm100.cuh"
#include "tmap.cuh"

namespace lnet {

constexpr int kTileM = 128;             // rows of A a CTA holds
constexpr int kTileThreads = 320;       // loader, MMA issuer, 8 epilogue warps
constexpr int kEpiWarps = 8;
constexpr uint32_t kTileWaitLimit = 1000000u;  // about 1 s of 1 us tries
constexpr int kTileSmemLimit = 227 * 1024;

enum LinearActivation { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// f(a); SiLU and GELU (0.5 a (1 + erf(a / sqrt 2))) in fp32.
__device__ __forceinline__ float act_value(float a, int act) {
  if (act == kActRelu) return a < 0.f ? 0.f : a;  // keeps NaN
  if (act == kActSilu) return a / (1.f + __expf(-a));
  if (act == kActGelu) return 0.5f * a * (1.f + erff(a * 0.70710678118654752f));
  return a;
}
// f'(a)
__device__ __forceinline__ float act_slope(float a, int act) {
  if (act == kActRelu) return a > 0.f ? 1.f : (a != a ? a : 0.f);
  if (act == kActSilu) {
    const float s = 1.f / (1.f + __expf(-a));
    return s * (1.f + a * (1.f - s));
  }
  if (act == kActGelu)
    return 0.5f * (1.f + erff(a * 0.70710678118654752f)) +
           a * __expf(-0.5f * a * a) * 0.39894228040143268f;
  return 1.f;
}

struct TileEpilogue {
  void *out;                      // bf16 [M, N], or fp32 partial sums [splits, M, N]
  __nv_bfloat16 *pre;             // C * scales + bias in bf16, or null
  const __nv_bfloat16 *bias;      // [N] or null
  const __nv_bfloat16 *residual;  // [M, N] or null
  const float *row_scale, *col_scale;  // [M], [N] or both null
  int act;
};

struct TileArgs {
  CUtensorMap a, b;
  TileEpilogue e;
  int64_t M, N;
  int m_tiles, n_tiles, splits, kblocks;
  int partial;  // write fp32 sums of this split
  int vec;      // 16-byte accesses to every [M, N] and [N] tensor
};

template <int CTAS, int BN, bool FP8>
struct TileShape {
  static constexpr int NB = BN / CTAS;  // rows of B a CTA holds
  static constexpr int A_BYTES = kTileM * 128, B_BYTES = NB * 128;
  static constexpr int STAGE = A_BYTES + B_BYTES;
  static constexpr int STAGES = (kTileSmemLimit - 2048) / STAGE > 8 ? 8
                                                                   : (kTileSmemLimit - 2048) / STAGE;
  static constexpr int SMEM = STAGES * STAGE + 1024 /* alignment */ + 512 /* barriers */;
  static constexpr int TMEM = 2 * BN < 32 ? 32 : 2 * BN;
};

// 32 columns of one row through the epilogue.  Loads bias, scales and residual
// 16 bytes at a time where the row's columns are all there and aligned.
__device__ __forceinline__ void tile_epilogue(const TileArgs &p, float *v, int64_t row,
                                              int64_t col, float row_scale, int64_t split) {
  const TileEpilogue &e = p.e;
  const bool full = col + 32 <= p.N;
  if (p.partial) {
    float *out = reinterpret_cast<float *>(e.out) + (split * p.M + row) * p.N + col;
    if (full && p.vec) {
#pragma unroll
      for (int j = 0; j < 32; j += 4)
        *reinterpret_cast<float4 *>(out + j) = make_float4(v[j], v[j + 1], v[j + 2], v[j + 3]);
    } else {
      for (int j = 0; j < 32; ++j)
        if (col + j < p.N) out[j] = v[j];
    }
    return;
  }
  const int64_t off = row * p.N + col;
  __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(e.out) + off;
  if (full && p.vec) {
#pragma unroll
    for (int j = 0; j < 32; j += 8) {
      float w[8];
      if (e.col_scale) {
        const float4 s0 = __ldg(reinterpret_cast<const float4 *>(e.col_scale + col + j));
        const float4 s1 = __ldg(reinterpret_cast<const float4 *>(e.col_scale + col + j + 4));
        const float s[8] = {s0.x, s0.y, s0.z, s0.w, s1.x, s1.y, s1.z, s1.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j + i] = v[j + i] * row_scale * s[i];
      }
      auto unpack = [&](const __nv_bfloat16 *src) {
        const uint4 u = __ldg(reinterpret_cast<const uint4 *>(src));
        const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          w[2 * i] = __uint_as_float(q[i] << 16);
          w[2 * i + 1] = __uint_as_float(q[i] & 0xFFFF0000u);
        }
      };
      auto pack = [&](__nv_bfloat16 *dst) {
        uint32_t q[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const __nv_bfloat162 b = __floats2bfloat162_rn(v[j + 2 * i], v[j + 2 * i + 1]);
          q[i] = *reinterpret_cast<const uint32_t *>(&b);
        }
        *reinterpret_cast<uint4 *>(dst) = make_uint4(q[0], q[1], q[2], q[3]);
      };
      if (e.bias) {
        unpack(e.bias + col + j);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j + i] += w[i];
      }
      if (e.pre) pack(e.pre + off + j);
      if (e.act != kActNone) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j + i] = act_value(v[j + i], e.act);
      }
      if (e.residual) {
        unpack(e.residual + off + j);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[j + i] += w[i];
      }
      pack(out + j);
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 32; ++j) {
    if (col + j >= p.N) break;
    float a = v[j];
    if (e.col_scale) a = a * row_scale * __ldg(e.col_scale + col + j);
    if (e.bias) a += load_f(e.bias, col + j);
    if (e.pre) store_f(e.pre, off + j, a);
    a = act_value(a, e.act);
    if (e.residual) a += load_f(e.residual, off + j);
    store_f(out, j, a);
  }
}

// The k blocks of one split: [k0, k1).
__device__ __forceinline__ void split_range(const TileArgs &p, int split, int &k0, int &k1) {
  k0 = (int)((int64_t)p.kblocks * split / p.splits);
  k1 = (int)((int64_t)p.kblocks * (split + 1) / p.splits);
}

// Tile order: bands of 8 row tiles, down the rows inside a column, so that a
// wave of CTAs shares few operand tiles in L2.
__device__ __forceinline__ void tile_at(const TileArgs &p, int t, int &m, int &n, int &split) {
  const int per = p.m_tiles * p.n_tiles;
  split = t / per;
  t -= split * per;
  constexpr int kBand = 8;
  const int band = t / (kBand * p.n_tiles);
  const int height = min(kBand, p.m_tiles - band * kBand);
  t -= band * kBand * p.n_tiles;
  n = t / height;
  m = band * kBand + t % height;
}

template <int CTAS, int BN, bool A_MN, bool B_MN, bool FP8>
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
  const int tiles = p.m_tiles * p.n_tiles * p.splits;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;
  auto wait = [&](uint64_t *bar, uint32_t parity) {
    bool ok = sm100::mbar_try_wait_cluster(bar, parity, 1000u);
    for (uint32_t i = 0; i < kTileWaitLimit && !ok && !*failed; ++i)
      ok = sm100::mbar_try_wait_cluster(bar, parity, 1000u);
    if (!ok) *failed = 1;
    return ok;
  };

  if (warp == 0 && lane == 0) {  // ---------------------------------------- loader
    int stage = 0, issued = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int m, n, split, k0, k1;
      tile_at(p, t, m, n, split);
      split_range(p, split, k0, k1);
      const int am = (m * CTAS + (int)rank) * kTileM, bn = n * BN + (int)rank * NB;
      for (int k = k0; k < k1; ++k) {
        if (issued >= STAGES && !(ok = wait(empty + stage, phase ^ 1))) break;
        if (leader) sm100::mbar_arrive_expect_tx(full + stage, CTAS * S::STAGE);
        const uint32_t bar = CTAS == 2 ? sm100::map_to_rank(full + stage, 0)
                                       : sm100::smem_u32(full + stage);
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
        sm100::mbar_wait_bounded(f, par, kTileWaitLimit / 10);
    }
  } else if (warp == 1 && lane == 0 && leader) {  // ------------------------ MMA issuer
    constexpr uint32_t idesc =
        (1u << 4) | (FP8 ? 0u : (1u << 7) | (1u << 10)) | ((A_MN ? 1u : 0u) << 15) |
        ((B_MN ? 1u : 0u) << 16) | ((uint32_t)(BN >> 3) << 17) |
        ((uint32_t)((CTAS * kTileM) >> 4) << 24);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    for (int t = first; t < tiles && ok; t += step) {
      int m, n, split, k0, k1;
      tile_at(p, t, m, n, split);
      split_range(p, split, k0, k1);
      if (!(ok = wait(acc_empty + acc, acc_phase ^ 1))) break;
      sm100::tc_fence_after();
      for (int k = k0; k < k1; ++k) {
        if (!(ok = wait(full + stage, phase))) break;
        sm100::tc_fence_after();
        const uint32_t da = sm100::smem_u32(smem + stage * S::STAGE), db = da + S::A_BYTES;
        const uint64_t ad = A_MN ? sm100::make_desc_sw128_mn(da, 8192) : sm100::make_desc_sw128(da);
        const uint64_t bd = B_MN ? sm100::make_desc_sw128_mn(db, 8192) : sm100::make_desc_sw128(db);
#pragma unroll
        for (int s = 0; s < 4; ++s)  // 32 bytes of k, or 16 k rows of 128 bytes
          sm100::mma_group<CTAS, FP8>(tmem + acc * BN, ad + s * (A_MN ? 128 : 2),
                                      bd + s * (B_MN ? 128 : 2), idesc, k > k0 || s > 0);
        sm100::mma_commit_group<CTAS>(empty + stage);
        if (++stage == STAGES) stage = 0, phase ^= 1;
      }
      if (!ok) break;
      sm100::mma_commit_group<CTAS>(acc_full + acc);
      if (++acc == 2) acc = 0, acc_phase ^= 1;
    }
    if (!ok) {  // the MMAs in flight end before TMEM is freed
      sm100::mma_commit_group<CTAS>(drain);
      sm100::mbar_wait_bounded(drain, 0, kTileWaitLimit / 10);
    }
  } else if (warp >= 2) {  // ----------------------------------------------- epilogue
    const int ew = warp - 2, quad = warp & 3, half = ew >> 2;
    constexpr int COLS = BN / 2 >= 32 ? BN / 2 : 32;  // columns of a warp
    const bool mine = half * COLS < BN;
    int acc = 0;
    uint32_t acc_phase = 0;
    bool ok = true;
    for (int t = first; t < tiles; t += step) {
      int m, n, split;
      tile_at(p, t, m, n, split);
      if (ok) ok = wait(acc_full + acc, acc_phase);
      ok = __all_sync(0xFFFFFFFFu, ok);
      sm100::tc_fence_after();
      const int64_t row = (int64_t)(m * CTAS + (int)rank) * kTileM + quad * 32 + lane;
      const float rs = p.e.row_scale && row < p.M ? __ldg(p.e.row_scale + row) : 1.f;
#pragma unroll 1
      for (int c = 0; mine && c < COLS; c += 32) {
        const int64_t col = (int64_t)n * BN + half * COLS + c;
        float v[32];
        if (ok) {
          sm100::tmem_ld32(tmem + ((uint32_t)(quad * 32) << 16) + acc * BN + half * COLS + c, v);
          sm100::tmem_ld_wait();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(0x7FC00000u);
        }
        if (row < p.M && col < p.N) tile_epilogue(p, v, row, col, rs, split);
      }
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2)
          sm100::mbar_arrive_rank(acc_empty + acc, 0);
        else
          sm100::mbar_arrive(acc_empty + acc);
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

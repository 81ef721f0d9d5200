// Matrix product with bias, activation and residual in its epilogue, its
// gradient, and its 8-bit form.
//
//   a = x W^T (* x_scale[row] weight_scale[col]) + bias,  y = f(a) + residual
//   gradient: da = dy f'(a),  dx = da W,  dW = da^T x,  dbias = sum over rows of da
//
// Three shapes of work:
//   * up to 8 rows: every weight is used once or a few times, so the call is
//     bound by reading them; a warp takes a column, 16 bytes of weights a lane
//     and step, and multiplies on the CUDA cores (vector_kernel);
//   * more rows: tensor cores (gemm_tiles.cuh); where the output has fewer tiles
//     than SMs and k is long, k is split and the fp32 partial sums are joined,
//     with the epilogue, in a second kernel;
//   * the elementwise slope da, rounded to bf16 as the operand of the two
//     products (fp32 on the way, and in the bias' column sums).
// TMA wants 16-byte aligned rows: an operand with other rows is first copied to
// the workspace with its rows padded.
#include <string.h>

#include <algorithm>
#include <type_traits>

#include "gemm_tiles.cuh"
#include "rows.cuh"

namespace lnet {
namespace {

constexpr int kVectorRows = 8;
constexpr int kVectorThreads = 256;
constexpr int kPackThreads = 256;
constexpr int kSlopeLanes = 8, kSlopeBlocks = 4;  // row lanes and resident blocks of the slope kernel

struct VectorArgs {
  const void *x, *w;
  TileEpilogue e;
  int64_t N, K, x_pitch, w_pitch;
  int rows, split;  // warps that share a column's k: 1, 2, 4 or 8
};

__device__ __forceinline__ float2 e4m3_pair_value(uint16_t q) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)q, __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2 *>(&h));
}

// 16 bytes of operand: 8 bf16 or 16 e4m3.
template <bool FP8>
__device__ __forceinline__ void operand_values(const uint4 &u, float *v) {
  const uint32_t q[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (FP8) {
      const float2 a = e4m3_pair_value((uint16_t)(q[i] & 0xFFFF));
      const float2 b = e4m3_pair_value((uint16_t)(q[i] >> 16));
      v[4 * i] = a.x, v[4 * i + 1] = a.y, v[4 * i + 2] = b.x, v[4 * i + 3] = b.y;
    } else {
      v[2 * i] = __uint_as_float(q[i] << 16);
      v[2 * i + 1] = __uint_as_float(q[i] & 0xFFFF0000u);
    }
  }
}
template <bool FP8>
__device__ __forceinline__ float operand_value(const void *p, int64_t i) {
  if (FP8) return e4m3_pair_value(reinterpret_cast<const uint8_t *>(p)[i]).x;
  return load_f(reinterpret_cast<const __nv_bfloat16 *>(p), i);
}

// The epilogue of one value.
__device__ __forceinline__ void scalar_epilogue(const TileEpilogue &e, float a, int64_t row,
                                                int64_t col, int64_t N) {
  if (e.col_scale) a = a * __ldg(e.row_scale + row) * __ldg(e.col_scale + col);
  if (e.bias) a += load_f(e.bias, col);
  const int64_t off = row * N + col;
  if (e.pre) store_f(e.pre, off, a);
  float v[2] = {a, 0.f};
  act_values<2>(v, e.act);
  a = v[0];
  if (e.residual) a += load_f(e.residual, off);
  store_f(e.out, off, a);
}

// R rows of x against every weight row.  A warp a column, or, where columns are few, a block's warps
// share its k in turns and the sums are added in order.  Bound by the weights' bytes for one row: 1 x
// 1024 -> 4096 bf16 (8.4 MB, 1.3 us at the peak) takes 5 us, the rest launch, first loads and shuffles.
template <bool FP8, int R, bool VEC>
__global__ void __launch_bounds__(kVectorThreads) vector_kernel(const VectorArgs p) {
  constexpr int E = FP8 ? 16 : 8, ES = FP8 ? 1 : 2;
  constexpr int U = R <= 2 ? 4 : 2;
  constexpr int WARPS = kVectorThreads / 32;
  __shared__ float parts[WARPS][R];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int turn = warp & (p.split - 1), stride = 32 * p.split, first = turn * 32 + lane;
  const int64_t col = (int64_t)blockIdx.x * (WARPS / p.split) + warp / p.split;
  const bool live = col < p.N;
  float acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.f;
  if (!live) {
  } else if (VEC) {
    const uint4 *w = reinterpret_cast<const uint4 *>(reinterpret_cast<const uint8_t *>(p.w) +
                                                     col * p.w_pitch * ES);
    const uint4 *x = reinterpret_cast<const uint4 *>(p.x);
    const int nc = (int)(p.K / E);
    for (int c0 = first; c0 < nc; c0 += stride * U) {
      uint4 wu[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        wu[u] = c0 + stride * u < nc ? __ldg(w + c0 + stride * u) : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c0 + stride * u >= nc) break;
        float wv[E];
        operand_values<FP8>(wu[u], wv);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          if (r >= p.rows) break;
          float xv[E];
          operand_values<FP8>(__ldg(x + r * (p.x_pitch / E) + c0 + stride * u), xv);
#pragma unroll
          for (int i = 0; i < E; ++i) acc[r] = fmaf(xv[i], wv[i], acc[r]);
        }
      }
    }
  } else {
    constexpr int S = 8;  // loads in flight: an element each
    for (int64_t k0 = first; k0 < p.K; k0 += (int64_t)stride * S) {
      float wv[S];
#pragma unroll
      for (int u = 0; u < S; ++u) {
        const int64_t k = k0 + stride * u;
        wv[u] = k < p.K ? operand_value<FP8>(p.w, col * p.w_pitch + k) : 0.f;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (r >= p.rows) break;
        float xv[S];
#pragma unroll
        for (int u = 0; u < S; ++u) {
          const int64_t k = k0 + stride * u;
          xv[u] = k < p.K ? operand_value<FP8>(p.x, r * p.x_pitch + k) : 0.f;
        }
#pragma unroll
        for (int u = 0; u < S; ++u) acc[r] = fmaf(xv[u], wv[u], acc[r]);
      }
    }
  }
  float mine = 0.f;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float s = group_reduce<32, SumOp>(acc[r], nullptr);
    if (lane == r) mine = s;
  }
  if (p.split > 1) {
    if (lane < R) parts[warp][lane] = mine;
    __syncthreads();
    if (turn) return;
    if (lane < R)
      for (int s = 1; s < p.split; ++s) mine += parts[warp + s][lane];
  }
  if (live && lane < p.rows) scalar_epilogue(p.e, mine, lane, col, p.N);
}

// Rows copied to a padded pitch (elements of ES bytes; the padding is zero).  A lane writes 16 bytes,
// a warp a stretch of a row.
template <int ES>
__global__ void __launch_bounds__(kPackThreads)
pack_kernel(const uint8_t *__restrict__ src, int64_t rows, int64_t cols, int64_t src_pitch,
            uint8_t *__restrict__ dst, int64_t pitch) {
  using E = std::conditional_t<ES == 2, uint16_t, uint8_t>;
  constexpr int PER = 16 / ES;
  const int lane = threadIdx.x & 31;
  const int64_t stretches = (pitch + 32 * PER - 1) / (32 * PER), total = rows * stretches;
  for (int64_t s = (int64_t)blockIdx.x * (kPackThreads / 32) + (threadIdx.x >> 5); s < total;
       s += (int64_t)gridDim.x * (kPackThreads / 32)) {
    const int64_t r = s / stretches, c0 = ((s - r * stretches) * 32 + lane) * PER;
    if (c0 >= pitch) continue;
    const E *from = reinterpret_cast<const E *>(src) + r * src_pitch + c0;
    E v[PER];
    if (c0 + PER <= cols) {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = __ldg(from + i);
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) v[i] = c0 + i < cols ? __ldg(from + i) : (E)0;
    }
    E *to = reinterpret_cast<E *>(dst) + r * pitch + c0;
    if (c0 + PER <= pitch && (reinterpret_cast<uintptr_t>(to) & 15) == 0) {
      uint4 u;
      memcpy(&u, v, 16);
      *reinterpret_cast<uint4 *>(to) = u;
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i)
        if (c0 + i < pitch) to[i] = v[i];
    }
  }
}

// da = dy f'(pre) in bf16 (pitch `pitch`, its padding zero; null: not wanted), and the blocks'
// column sums of the unrounded da (null: not wanted).  A thread holds VEC columns of every
// kSlopeLanes-th row of its block's rows.  16384 x 8192, GELU: 171 us for 805 MB (0.73 of a copy's
// rate), bound by the exponential and the polynomial (1.7 instructions a clock) next to HBM.  Rows off
// 16-byte boundaries take pairs of columns where they are even, else one: 6329 x 4558, ReLU, 40 us,
// 4557 columns 74, 4560 31.
template <int VEC, int ACT>
__global__ void __launch_bounds__(32 * kSlopeLanes, kSlopeBlocks)
slope_kernel(const __nv_bfloat16 *__restrict__ dy, const __nv_bfloat16 *__restrict__ pre, int64_t M,
             int64_t N, __nv_bfloat16 *__restrict__ da, int64_t pitch,
             float *__restrict__ partial) {
  __shared__ float sums[kSlopeLanes][32 * VEC];
  // rows in flight; four of 8 columns held registers that a fourth block needs, and eight of one or
  // two columns took twice as long
  constexpr int R = 2;
  const int64_t col = ((int64_t)blockIdx.x * 32 + threadIdx.x) * VEC;
  float s[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) s[i] = 0.f;
  const int64_t r0 = M * blockIdx.y / gridDim.y, r1 = M * (blockIdx.y + 1) / gridDim.y;
  if (col < N) {
    for (int64_t r = r0 + threadIdx.y; r < r1; r += kSlopeLanes * R) {
      RowChunk<__nv_bfloat16, VEC> c[R], q[R];
#pragma unroll
      for (int k = 0; k < R; ++k) {
        c[k].zero(), q[k].zero();
        if (r + k * kSlopeLanes >= r1) continue;
        c[k].load(dy + (r + k * kSlopeLanes) * N + col);
        if (ACT != kActNone) q[k].load(pre + (r + k * kSlopeLanes) * N + col);
      }
#pragma unroll
      for (int k = 0; k < R; ++k) {
        float g[VEC + 1], a[VEC + 1];
        c[k].get(g), q[k].get(a);
        if (VEC == 1) g[1] = 0.f, a[1] = 0.f;
#pragma unroll
        for (int i = 0; i < VEC; i += 2) {
          const Pair d = pair(g[i], g[i + 1]) * act_slope<ACT>(pair(a[i], a[i + 1]));
          unpair(d, g[i], g[i + 1]);
        }
        const bool live = r + k * kSlopeLanes < r1;
        if (live) {
#pragma unroll
          for (int i = 0; i < VEC; ++i) s[i] += g[i];
        }
        if (da && live) {
          c[k].put(g);
          c[k].store(da + (r + k * kSlopeLanes) * pitch + col);
        }
      }
    }
  } else if (da && col < pitch) {
    RowChunk<__nv_bfloat16, VEC> c;
    c.zero();
    for (int64_t r = r0 + threadIdx.y; r < r1; r += kSlopeLanes) c.store(da + r * pitch + col);
  }
  if (!partial) return;
#pragma unroll
  for (int i = 0; i < VEC; ++i) sums[threadIdx.y][threadIdx.x * VEC + i] = s[i];
  __syncthreads();
  for (int c = threadIdx.y * 32 + threadIdx.x; c < 32 * VEC; c += 32 * kSlopeLanes) {
    const int64_t out = (int64_t)blockIdx.x * 32 * VEC + c;
    if (out >= N) continue;
    float t = 0.f;
#pragma unroll
    for (int l = 0; l < kSlopeLanes; ++l) t += sums[l][c];
    partial[(int64_t)blockIdx.y * N + out] = t;
  }
}

template <int VEC>
void launch_slope(dim3 grid, dim3 block, int act, const __nv_bfloat16 *dy, const __nv_bfloat16 *pre,
                  int64_t M, int64_t N, __nv_bfloat16 *da, int64_t pitch, float *columns,
                  cudaStream_t s) {
  switch (act) {
    case kActRelu:
      slope_kernel<VEC, kActRelu><<<grid, block, 0, s>>>(dy, pre, M, N, da, pitch, columns);
      break;
    case kActSilu:
      slope_kernel<VEC, kActSilu><<<grid, block, 0, s>>>(dy, pre, M, N, da, pitch, columns);
      break;
    case kActGelu:
      slope_kernel<VEC, kActGelu><<<grid, block, 0, s>>>(dy, pre, M, N, da, pitch, columns);
      break;
    default:
      slope_kernel<VEC, kActNone><<<grid, block, 0, s>>>(dy, pre, M, N, da, pitch, columns);
  }
}

// dbias from the blocks' column sums, in block order (32 columns by 32 lanes).
__global__ void __launch_bounds__(1024)
column_sum_kernel(const float *__restrict__ partial, int blocks, int64_t N,
                  __nv_bfloat16 *__restrict__ out) {
  __shared__ float part[32][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < N)
    for (int b = threadIdx.y; b < blocks; b += 32) s += partial[(int64_t)b * N + c];
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < N) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += part[i][threadIdx.x];
    store_f(out, c, s);
  }
}

// ---------------------------------------------------------------- plans
enum TileKind { kPair256, kPair128, kOne128, kOne64 };

struct ProductPlan {
  TileKind kind;
  int m_tiles, n_tiles, full, splits, grid;
  int64_t partial_floats;
};

// Tile shape and split of an [M, N] product over `kblocks` blocks of 128 bytes.  Time in units of
// 128 clocks, about 70 ns: a k block of a 128 x 64 tile's MMAs.
ProductPlan product_plan(int64_t M, int64_t N, int kblocks) {
  const int sms = sm_count();
  struct Shape {
    TileKind kind;
    int ctas, bn;
    double block;  // a k block, measured at 16384 x 8192 x 2048 and its gradient's products
  };
  static const Shape shapes[] = {
      {kPair256, 2, 256, 4.0}, {kPair128, 2, 128, 2.8}, {kOne128, 1, 128, 2.85}, {kOne64, 1, 64, 1.8}};
  ProductPlan best{};
  double best_cost = 0;
  for (const Shape &s : shapes) {
    const int64_t mt = cdiv(M, (int64_t)kTileM * s.ctas), nt = cdiv(N, s.bn), tiles = mt * nt;
    const int slots = sms / s.ctas;
    const int64_t waves = tiles / slots, tail = tiles % slots;
    constexpr double kFill = 24;  // pipeline fill and the last epilogue, once
    const double whole = s.block * kblocks + 6;
    for (int splits = 1; splits <= 64; ++splits) {
      // every split keeps 4 k blocks, and the splits take 3 rounds at most
      if (splits > 1 && (tail == 0 || tail * splits > 3 * slots || kblocks / splits < 4)) break;
      double cost = kFill + waves * whole;
      if (tail) cost += cdiv(tail * splits, slots) * (s.block * cdiv(kblocks, splits) + 6);
      // the sums are written and read once (about 6 TB/s), and one more kernel runs (5 us on the
      // GPU and 3 on the host)
      const int64_t floats = splits > 1 ? tail * splits * s.ctas * kTileM * s.bn : 0;
      if (splits > 1) cost += 90 + floats * 8 / 4.2e5;
      if (best_cost == 0 || cost < best_cost) {
        best_cost = cost;
        const int64_t full = splits > 1 ? waves * slots : tiles;
        const int64_t units = full + (tiles - full) * splits;
        best = ProductPlan{s.kind, (int)mt, (int)nt, (int)full, splits,
                           (int)std::min<int64_t>(units, slots) * s.ctas, floats};
      }
    }
  }
  return best;
}

template <int CTAS, int BN, bool A_MN, bool B_MN, bool FP8, int UNIT>
int launch_unit(const ProductPlan &q, const TileOperand &a, const TileOperand &b, TileArgs &args,
                cudaStream_t stream) {
  using S = TileShape<CTAS, BN, FP8>;
  constexpr auto kernel = &tile_gemm_kernel<CTAS, BN, A_MN, B_MN, FP8, UNIT>;
  LNET_TRY(raise_shared_memory<kernel>(S::SMEM, "tile_gemm_kernel shared memory"));
  LNET_TRY(tile_tensor_map(&args.a, a, FP8, kTileM));
  LNET_TRY(tile_tensor_map(&args.b, b, FP8, S::NB));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)q.grid);
  cfg.blockDim = dim3(kTileThreads);
  cfg.dynamicSmemBytes = S::SMEM;
  cfg.stream = stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = CTAS;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  cfg.attrs = &cluster;
  cfg.numAttrs = 1;
  LNET_TRY(cuda_check(cudaLaunchKernelEx(&cfg, kernel, args), "tile_gemm_kernel"));
  LNET_TRY(after_launch("tile_gemm_kernel"));
  if (q.splits == 1) return LNET_OK;
  const int blocks = (q.m_tiles * q.n_tiles - q.full) * CTAS * 4 * (BN / 32);
  tile_join_kernel<CTAS, BN, UNIT><<<(unsigned)cdiv(blocks, kJoinThreads / 32), kJoinThreads, 0, stream>>>(
      args);
  return after_launch("tile_join_kernel");
}

template <int CTAS, int BN, bool A_MN, bool B_MN, bool FP8>
int launch_tiles(const ProductPlan &q, const TileOperand &a, const TileOperand &b, TileArgs &args,
                 cudaStream_t s) {
  const uintptr_t where = reinterpret_cast<uintptr_t>(args.e.out) |
                          reinterpret_cast<uintptr_t>(args.e.pre) |
                          reinterpret_cast<uintptr_t>(args.e.residual);
  int unit = 8;
  while (unit > 1 && (args.N % unit || where % (2 * unit))) unit /= 2;
  switch (unit) {
    case 8: return launch_unit<CTAS, BN, A_MN, B_MN, FP8, 8>(q, a, b, args, s);
    case 4: return launch_unit<CTAS, BN, A_MN, B_MN, FP8, 4>(q, a, b, args, s);
    case 2: return launch_unit<CTAS, BN, A_MN, B_MN, FP8, 2>(q, a, b, args, s);
    default: return launch_unit<CTAS, BN, A_MN, B_MN, FP8, 1>(q, a, b, args, s);
  }
}

template <bool A_MN, bool B_MN, bool FP8>
int launch_kind(const ProductPlan &q, const TileOperand &a, const TileOperand &b, TileArgs &args,
                cudaStream_t s) {
  switch (q.kind) {
    case kPair256: return launch_tiles<2, 256, A_MN, B_MN, FP8>(q, a, b, args, s);
    case kPair128: return launch_tiles<2, 128, A_MN, B_MN, FP8>(q, a, b, args, s);
    case kOne128: return launch_tiles<1, 128, A_MN, B_MN, FP8>(q, a, b, args, s);
    default: return launch_tiles<1, 64, A_MN, B_MN, FP8>(q, a, b, args, s);
  }
}

// C = A B^T through the epilogue; `partial` holds plan.partial_floats.
template <bool A_MN, bool B_MN, bool FP8>
int product(const TileOperand &a, const TileOperand &b, const TileEpilogue &e, float *partial,
            cudaStream_t s) {
  const int64_t M = a.mn, N = b.mn;
  const int kblocks = (int)cdiv(a.k, FP8 ? 128 : 64);
  const ProductPlan q = product_plan(M, N, kblocks);
  TileArgs args{};
  args.e = e;
  args.M = M, args.N = N;
  args.m_tiles = q.m_tiles, args.n_tiles = q.n_tiles, args.full = q.full;
  args.splits = q.splits, args.kblocks = kblocks;
  args.partial = partial;
  args.by_band = FastDiv(kBand * q.n_tiles);
  args.by_last = FastDiv(q.m_tiles % kBand ? q.m_tiles % kBand : kBand);
  args.by_splits = FastDiv(q.splits);
  return launch_kind<A_MN, B_MN, FP8>(q, a, b, args, s);
}

bool tma_rows(const void *p, int64_t pitch_bytes) { return aligned16(p) && pitch_bytes % 16 == 0; }

int launch_pack(const void *src, int64_t rows, int64_t cols, int64_t src_pitch, int elem, void *dst,
                int64_t pitch, cudaStream_t s) {
  const int64_t warps = rows * cdiv(pitch, 32 * 16 / elem);
  const int blocks =
      (int)std::min<int64_t>(cdiv(warps, kPackThreads / 32), (int64_t)sm_count() * 32);
  const auto *from = reinterpret_cast<const uint8_t *>(src);
  auto *to = reinterpret_cast<uint8_t *>(dst);
  if (elem == 2)
    pack_kernel<2><<<blocks, kPackThreads, 0, s>>>(from, rows, cols, src_pitch, to, pitch);
  else
    pack_kernel<1><<<blocks, kPackThreads, 0, s>>>(from, rows, cols, src_pitch, to, pitch);
  return after_launch("linear_pack_kernel");
}

// `o` itself, or its copy with padded rows (a rows x cols matrix in memory).
int packed(TileOperand &o, int64_t rows, int64_t cols, int elem, void *copy, cudaStream_t s) {
  if (!copy) return LNET_OK;
  const int64_t pitch = (int64_t)align_up((size_t)cols * elem, 16) / elem;
  LNET_TRY(launch_pack(o.ptr, rows, cols, o.pitch, elem, copy, pitch, s));
  o.ptr = copy;
  o.pitch = pitch;
  return LNET_OK;
}

int64_t x_pitch(const lnet_b200_linear_request *q) { return q->x_pitch ? q->x_pitch : q->inner; }
int64_t w_pitch(const lnet_b200_linear_request *q) {
  return q->weight_pitch ? q->weight_pitch : q->inner;
}

int check_linear(const char *what, const lnet_b200_linear_request *q) {
  if (!q) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: request must not be NULL", what);
  if (q->rows < 0 || q->inner < 1 || q->outer < 1)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: rows %lld, inner %lld, outer %lld", what,
                (long long)q->rows, (long long)q->inner, (long long)q->outer);
  const int64_t most = (int64_t)1 << 30;
  if (q->rows > most || q->inner > most || q->outer > most)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: an extent is above 2^30", what);
  if (cdiv(q->rows, 128) * cdiv(q->outer, 64) > most || cdiv(q->rows, 128) * cdiv(q->inner, 64) > most ||
      cdiv(q->outer, 128) * cdiv(q->inner, 64) > most)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: a product has more than 2^30 tiles", what);
  for (int64_t pitch : {x_pitch(q), w_pitch(q)})
    if (pitch < q->inner || pitch > (int64_t)1 << 36)
      return fail(LNET_ERR_INVALID_ARGUMENT, "%s: a pitch of %lld, inner %lld", what,
                  (long long)pitch, (long long)q->inner);
  if (q->dtype != LNET_BF16 && q->dtype != LNET_E4M3)
    return fail(LNET_ERR_UNSUPPORTED, "%s: operands must be bf16 or e4m3", what);
  if (q->activation < kActNone || q->activation > kActGelu)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: activation must be 0 to 3", what);
  if (q->rows > 0 && (!q->x || !q->weight))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: x and weight must not be NULL", what);
  if (q->rows > 0 && q->dtype == LNET_E4M3 && (!q->x_scale || !q->weight_scale))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: 8-bit operands need x_scale and weight_scale",
                what);
  return LNET_OK;
}

// Workspace of the forward pass: operands that TMA cannot address, partial sums.
struct ForwardWork {
  void *x, *w;
  float *partial;
};
ForwardWork forward_work(Arena &ar, const lnet_b200_linear_request *q) {
  ForwardWork f{};
  if (q->rows <= kVectorRows) return f;
  const int elem = q->dtype == LNET_BF16 ? 2 : 1;
  const size_t pitch = align_up((size_t)q->inner * elem, 16);
  if (!tma_rows(q->x, x_pitch(q) * elem)) f.x = ar.take<uint8_t>(q->rows * pitch);
  if (!tma_rows(q->weight, w_pitch(q) * elem)) f.w = ar.take<uint8_t>(q->outer * pitch);
  const ProductPlan p = product_plan(q->rows, q->outer, (int)cdiv(q->inner * elem, 128));
  if (p.partial_floats) f.partial = ar.take<float>(p.partial_floats);
  return f;
}

int slope_row_blocks(int64_t M, int64_t N, int vec) {
  const int64_t across = cdiv(N, 32 * vec);
  const int64_t want = (int64_t)sm_count() * kSlopeBlocks / across;  // all of them at once
  return (int)std::max<int64_t>(1, std::min<int64_t>(want, cdiv(M, kSlopeLanes * 2)));
}
int slope_vec(const lnet_b200_linear_request *q, const void *pre, const void *dy) {
  const uintptr_t where = reinterpret_cast<uintptr_t>(pre) | reinterpret_cast<uintptr_t>(dy);
  return q->outer % 8 == 0 && where % 16 == 0 ? 8 : q->outer % 2 == 0 && where % 4 == 0 ? 2 : 1;
}

// Workspace of the gradient.
struct BackwardWork {
  __nv_bfloat16 *da;  // null: dy itself serves
  void *x, *w;
  float *partial, *columns;
};
BackwardWork backward_work(Arena &ar, const lnet_b200_linear_request *q, const void *pre,
                           const void *dy, bool want_dx, bool want_dw, bool want_db) {
  BackwardWork b{};
  const size_t pitch_in = align_up((size_t)q->inner * 2, 16);
  const size_t pitch_out = align_up((size_t)q->outer * 2, 16);
  if ((want_dx || want_dw) && (pre || !tma_rows(dy, q->outer * 2)))
    b.da = ar.take<__nv_bfloat16>(q->rows * pitch_out / 2);
  if (want_dw && !tma_rows(q->x, x_pitch(q) * 2)) b.x = ar.take<uint8_t>(q->rows * pitch_in);
  if (want_dx && !tma_rows(q->weight, w_pitch(q) * 2)) b.w = ar.take<uint8_t>(q->outer * pitch_in);
  int64_t partial = 0;
  if (want_dx)
    partial = product_plan(q->rows, q->inner, (int)cdiv(q->outer, 64)).partial_floats;
  if (want_dw)
    partial = std::max(partial,
                       product_plan(q->outer, q->inner, (int)cdiv(q->rows, 64)).partial_floats);
  if (partial) b.partial = ar.take<float>(partial);
  if (want_db)
    b.columns = ar.take<float>((size_t)slope_row_blocks(q->rows, q->outer, slope_vec(q, pre, dy)) *
                               q->outer);
  return b;
}

template <bool FP8, bool VEC>
void launch_vector(const VectorArgs &v, cudaStream_t s) {
  const unsigned blocks = (unsigned)cdiv(v.N, kVectorThreads / 32 / v.split);
  if (v.rows == 1)
    vector_kernel<FP8, 1, VEC><<<blocks, kVectorThreads, 0, s>>>(v);
  else if (v.rows == 2)
    vector_kernel<FP8, 2, VEC><<<blocks, kVectorThreads, 0, s>>>(v);
  else if (v.rows <= 4)
    vector_kernel<FP8, 4, VEC><<<blocks, kVectorThreads, 0, s>>>(v);
  else
    vector_kernel<FP8, 8, VEC><<<blocks, kVectorThreads, 0, s>>>(v);
}

}  // namespace
}  // namespace lnet

using namespace lnet;

extern "C" int lnet_b200_linear_workspace_size(const lnet_b200_linear_request *req,
                                               size_t *bytes) {
  const char *what = "linear_workspace_size";
  LNET_TRY(check_linear(what, req));
  if (!bytes) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: bytes must not be NULL", what);
  Arena ar(nullptr, 0);
  if (req->rows > 0) forward_work(ar, req);
  *bytes = ar.used;
  return LNET_OK;
}

extern "C" int lnet_b200_linear_forward(const lnet_b200_linear_request *req, void *workspace,
                                        size_t workspace_bytes, void *y, void *preact,
                                        lnet_stream_t stream) {
  const char *what = "linear_forward";
  LNET_TRY(check_linear(what, req));
  reset_launches();
  if (req->rows == 0) return LNET_OK;
  if (!y) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: y must not be NULL", what);
  Arena ar(workspace, workspace_bytes);
  const ForwardWork f = forward_work(ar, req);
  if (ar.used > workspace_bytes || (ar.used && !workspace))
    return fail(LNET_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", what, ar.used,
                workspace_bytes);
  begin_entry(stream);
  const bool fp8 = req->dtype == LNET_E4M3;
  const int elem = fp8 ? 1 : 2;
  TileEpilogue e{};
  e.out = reinterpret_cast<__nv_bfloat16 *>(y);
  e.pre = reinterpret_cast<__nv_bfloat16 *>(preact);
  e.bias = reinterpret_cast<const __nv_bfloat16 *>(req->bias);
  e.residual = reinterpret_cast<const __nv_bfloat16 *>(req->residual);
  e.row_scale = fp8 ? req->x_scale : nullptr;
  e.col_scale = fp8 ? req->weight_scale : nullptr;
  e.act = req->activation;
  if (req->rows <= kVectorRows) {
    VectorArgs v{req->x,       req->weight,  e,           req->outer, req->inner,
                 x_pitch(req), w_pitch(req), (int)req->rows, 1};
    const bool vec = req->inner * elem % 16 == 0 && tma_rows(req->x, x_pitch(req) * elem) &&
                     tma_rows(req->weight, w_pitch(req) * elem);
    // two blocks an SM, as long as every warp keeps a load a lane
    const int64_t loads = req->inner * elem / (vec ? 16 : elem);
    while (v.split < kVectorThreads / 32 && v.N * v.split < (int64_t)sm_count() * 16 &&
           loads >= 64 * v.split)
      v.split *= 2;
    if (fp8)
      vec ? launch_vector<true, true>(v, stream) : launch_vector<true, false>(v, stream);
    else
      vec ? launch_vector<false, true>(v, stream) : launch_vector<false, false>(v, stream);
    return after_launch("linear_vector_kernel");
  }
  TileOperand a{req->x, req->rows, req->inner, x_pitch(req), false};
  TileOperand b{req->weight, req->outer, req->inner, w_pitch(req), false};
  LNET_TRY(packed(a, req->rows, req->inner, elem, f.x, stream));
  LNET_TRY(packed(b, req->outer, req->inner, elem, f.w, stream));
  return fp8 ? product<false, false, true>(a, b, e, f.partial, stream)
             : product<false, false, false>(a, b, e, f.partial, stream);
}

extern "C" int lnet_b200_linear_pack(const void *src, int32_t dtype, int64_t rows, int64_t cols,
                                     int64_t src_pitch, void *dst, int64_t dst_pitch,
                                     lnet_stream_t stream) {
  const char *what = "linear_pack";
  const int64_t most = (int64_t)1 << 36;
  if (rows < 0 || cols < 1 || src_pitch < cols || dst_pitch < cols || src_pitch > most ||
      dst_pitch > most || rows > (int64_t)1 << 30 ||
      (rows > 0 && std::max(src_pitch, dst_pitch) > ((int64_t)1 << 46) / rows))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: rows %lld, cols %lld, pitches %lld and %lld", what,
                (long long)rows, (long long)cols, (long long)src_pitch, (long long)dst_pitch);
  if (dtype != LNET_BF16 && dtype != LNET_E4M3)
    return fail(LNET_ERR_UNSUPPORTED, "%s: operands must be bf16 or e4m3", what);
  reset_launches();
  if (rows == 0) return LNET_OK;
  if (!src || !dst) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: a NULL pointer", what);
  begin_entry(stream);
  return launch_pack(src, rows, cols, src_pitch, dtype == LNET_BF16 ? 2 : 1, dst, dst_pitch,
                     stream);
}

static int check_backward(const char *what, const lnet_b200_linear_request *req,
                          const void *preact, const void *dy) {
  LNET_TRY(check_linear(what, req));
  if (req->dtype != LNET_BF16)
    return fail(LNET_ERR_UNSUPPORTED, "%s: the gradient wants bf16 operands", what);
  if (req->rows > 0 && (!dy || (req->activation != kActNone && !preact)))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: dy%s must not be NULL", what,
                req->activation != kActNone ? ", preact" : "");
  return LNET_OK;
}

extern "C" int lnet_b200_linear_backward_workspace_size(const lnet_b200_linear_request *req,
                                                        const void *preact, const void *dy,
                                                        int32_t want_dx, int32_t want_dweight,
                                                        int32_t want_dbias, size_t *bytes) {
  const char *what = "linear_backward_workspace_size";
  LNET_TRY(check_backward(what, req, preact, dy));
  if (!bytes) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: bytes must not be NULL", what);
  Arena ar(nullptr, 0);
  if (req->rows > 0)
    backward_work(ar, req, req->activation ? preact : nullptr, dy, want_dx, want_dweight,
                  want_dbias);
  *bytes = ar.used;
  return LNET_OK;
}

extern "C" int lnet_b200_linear_backward(const lnet_b200_linear_request *req, const void *preact,
                                         const void *dy, void *workspace, size_t workspace_bytes,
                                         void *dx, void *dweight, void *dbias,
                                         lnet_stream_t stream) {
  const char *what = "linear_backward";
  LNET_TRY(check_backward(what, req, preact, dy));
  reset_launches();
  begin_entry(stream);
  const int64_t M = req->rows, N = req->outer, K = req->inner;
  if (M == 0) {
    if (dweight) LNET_TRY(cuda_check(cudaMemsetAsync(dweight, 0, N * K * 2, stream), what));
    if (dbias) LNET_TRY(cuda_check(cudaMemsetAsync(dbias, 0, N * 2, stream), what));
    return LNET_OK;
  }
  if (!req->activation) preact = nullptr;
  Arena ar(workspace, workspace_bytes);
  const BackwardWork w = backward_work(ar, req, preact, dy, dx != nullptr, dweight != nullptr,
                                       dbias != nullptr);
  if (ar.used > workspace_bytes || (ar.used && !workspace))
    return fail(LNET_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", what, ar.used,
                workspace_bytes);
  const auto *dyp = reinterpret_cast<const __nv_bfloat16 *>(dy);
  const auto *pre = reinterpret_cast<const __nv_bfloat16 *>(preact);
  const int64_t pitch = w.da ? (int64_t)align_up((size_t)N * 2, 16) / 2 : N;
  if (w.da || w.columns) {
    const int vec = slope_vec(req, preact, dy);
    const int64_t width = w.da ? pitch : N;
    const dim3 grid((unsigned)cdiv(width, 32 * vec), (unsigned)slope_row_blocks(M, N, vec));
    const dim3 block(32, kSlopeLanes);
    if (vec == 8)
      launch_slope<8>(grid, block, req->activation, dyp, pre, M, N, w.da, pitch, w.columns, stream);
    else if (vec == 2)
      launch_slope<2>(grid, block, req->activation, dyp, pre, M, N, w.da, pitch, w.columns, stream);
    else
      launch_slope<1>(grid, block, req->activation, dyp, pre, M, N, w.da, pitch, w.columns, stream);
    LNET_TRY(after_launch("linear_slope_kernel"));
    if (w.columns) {
      column_sum_kernel<<<(unsigned)cdiv(N, 32), dim3(32, 32), 0, stream>>>(
          w.columns, (int)grid.y, N, reinterpret_cast<__nv_bfloat16 *>(dbias));
      LNET_TRY(after_launch("linear_column_sum_kernel"));
    }
  }
  const void *da = w.da ? (const void *)w.da : dy;
  if (dx) {
    TileOperand a{da, M, N, pitch, false};
    TileOperand b{req->weight, K, N, w_pitch(req), true};
    LNET_TRY(packed(b, N, K, 2, w.w, stream));
    TileEpilogue e{};
    e.out = reinterpret_cast<__nv_bfloat16 *>(dx);
    LNET_TRY((product<false, true, false>(a, b, e, w.partial, stream)));
  }
  if (dweight) {
    TileOperand a{da, N, M, pitch, true};
    TileOperand b{req->x, K, M, x_pitch(req), true};
    LNET_TRY(packed(b, M, K, 2, w.x, stream));
    TileEpilogue e{};
    e.out = reinterpret_cast<__nv_bfloat16 *>(dweight);
    LNET_TRY((product<true, true, false>(a, b, e, w.partial, stream)));
  }
  return LNET_OK;
}

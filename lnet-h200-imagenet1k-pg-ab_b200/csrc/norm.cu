// Residual addition + RMSNorm, its gradient, and its 8-bit output.
//
//   h = round(x + r)              the stream, in the inputs' type
//   rstd = (mean(h^2) + eps)^-1/2 fp32, over the stream as it is stored
//   y = h rstd w
//   8 bits: s = max|y| / 448, q = e4m3(y / s)   (s = 0: q = 0)
//   gradient: g = dy w, c = mean(g h rstd),
//     dx = dr = rstd (g - h rstd c) + dh,  dw = sum over rows of dy h rstd
//
// Every pass is bound by HBM: a row is read once, held in registers (packed
// loads of 16 bytes, up to 4 a thread) through both of its reductions, and
// written once.  A row of up to 128 chunks belongs to 4, 8, 16 or 32 lanes of a
// warp (the fewest that hold it in 4 chunks each, so that a 96-wide bf16 row
// uses 4 lanes x 3 chunks and no lane idles); a longer one to a block of up to
// 512 threads; one that 512 threads cannot hold is read again from L2 (wide
// kernels).  Rows of other lengths than a multiple of 16 bytes keep the 16-byte
// loads, shifted to the boundaries (SHIFT).
//
// Measured, of the 6448 GB/s of a copy: 16384 x 4096 bf16 + residual to e4m3 76
// us on the same inputs again and 82 on others in turn (0.96, 0.89); 802816 x 96 bf16 with gradient 101 + 102 us for 616 MB each (0.94)
// and 6 us of column sums.
#include <cuda_fp8.h>

#include <algorithm>
#include <atomic>
#include <initializer_list>

#include "rows.cuh"
#include "sm100.cuh"

namespace lnet {
namespace {

constexpr float kE4m3Max = 448.f;
constexpr int kSubThreads = 256;    // block of the kernels that put several rows in a warp
constexpr int kBlockThreads = 512;  // largest block of the row-per-block kernels
constexpr int kWideThreads = 1024;
constexpr int kReduceLanes = 32;

// chunks a thread may hold
template <int VEC>
__host__ __device__ constexpr int chunks_of() {
  return VEC == 1 ? 16 : 4;
}

__device__ __forceinline__ float weight_at(const void *w, bool w_bf16, int64_t i) {
  return w_bf16 ? load_f(reinterpret_cast<const __nv_bfloat16 *>(w), i)
                : __ldg(reinterpret_cast<const float *>(w) + i);
}

// VEC weights from column c * VEC on, in fp32 (16-byte loads where the plan is vectorised).
template <int VEC>
__device__ __forceinline__ void weight_chunk(const void *w, bool w_bf16, int c, float *v) {
  if (VEC == 1) {
    v[0] = weight_at(w, w_bf16, c);
  } else if (w_bf16) {
    const uint16_t *p = reinterpret_cast<const uint16_t *>(w) + c * VEC;
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const uint2 u = __ldg(reinterpret_cast<const uint2 *>(p) + i);
      v[4 * i] = __uint_as_float(u.x << 16);
      v[4 * i + 1] = __uint_as_float(u.x & 0xFFFF0000u);
      v[4 * i + 2] = __uint_as_float(u.y << 16);
      v[4 * i + 3] = __uint_as_float(u.y & 0xFFFF0000u);
    }
  } else {
    const float *p = reinterpret_cast<const float *>(w) + c * VEC;
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float4 u = __ldg(reinterpret_cast<const float4 *>(p) + i);
      v[4 * i] = u.x, v[4 * i + 1] = u.y, v[4 * i + 2] = u.z, v[4 * i + 3] = u.w;
    }
  }
}

template <int VEC>
__device__ __forceinline__ void weight_lanes(const void *w, bool w_bf16, int c, Lanes<VEC> *p) {
  float v[VEC];
  weight_chunk<VEC>(w, w_bf16, c, v);
  to_lanes<VEC>(v, p);
}

__device__ __forceinline__ uint32_t e4m3_pair(float a, float b) {
  return (uint32_t)__nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
// A chunk's 8 codes of which only those inside the row are stored.  The row covers the chunk's end or
// its start (rows have two chunks and more), so that pieces of 4, 2 and 1 codes are aligned to their
// size: 47611 x 123 bf16 38 us, 50 with 8 stores of a byte.  (4 codes of an fp32 chunk, or the 16-bit
// elements of a bf16 one, took longer in pieces: 33 us against 22, 39 against 35.)
__device__ __forceinline__ void store_cut8(uint8_t *p, uint64_t codes, int e0, int dim) {
  const int count = e0 < 0 ? 8 + e0 : dim - e0;
#pragma unroll
  for (int s = 4; s >= 1; s /= 2) {
    if (!(count & s)) continue;
    const int at = e0 < 0 ? 8 - (count & ~(s - 1)) : count & ~(2 * s - 1);
    const uint32_t v = (uint32_t)(codes >> (8 * at));
    if (s == 4) *reinterpret_cast<uint32_t *>(p + at) = v;
    if (s == 2) *reinterpret_cast<uint16_t *>(p + at) = (uint16_t)v;
    if (s == 1) p[at] = (uint8_t)v;
  }
}
// e4m3(v k) of the chunk of a row that starts at element e0, saturating.
template <int VEC, bool SHIFT = false>
__device__ __forceinline__ void store_e4m3(uint8_t *row, const Lanes<VEC> *l, float k, int64_t e0,
                                           int dim) {
  Lanes<VEC> s[lanes_of<VEC>()];
  float v[VEC];
#pragma unroll
  for (int i = 0; i < lanes_of<VEC>(); ++i) s[i] = l[i] * splat<VEC>(k);
  from_lanes<VEC>(s, v);
  uint8_t *p = row + e0;
  if constexpr (VEC == 1) {
    *p = (uint8_t)e4m3_pair(v[0], 0.f);
  } else {
    uint32_t q[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i)
      q[i] = e4m3_pair(v[4 * i], v[4 * i + 1]) | (e4m3_pair(v[4 * i + 2], v[4 * i + 3]) << 16);
    // A chunk's codes are as aligned as the chunk where the tensors' first elements are.
    const bool cut = e0 < 0 || e0 + VEC > dim;
    if (SHIFT && ((VEC == 4 && cut) || (reinterpret_cast<uintptr_t>(p) & (VEC - 1)))) {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (e0 + i >= 0 && e0 + i < dim) p[i] = (uint8_t)(q[i / 4] >> (8 * (i % 4)));
    } else if (SHIFT && VEC == 8 && cut) {
      store_cut8(p, q[0] | (uint64_t)q[VEC / 4 - 1] << 32, e0, dim);
    } else if constexpr (VEC == 8) {
      *reinterpret_cast<uint2 *>(p) = make_uint2(q[0], q[1]);
    } else {
      *reinterpret_cast<uint32_t *>(p) = q[0];
    }
  }
}
// A row's scale s = m / 448, m = max|y|, and how its codes e4m3(y / s) are taken: y (448 / m), two fp32
// roundings from the quotient, 2^-20 of a code's step.  Where s is below the normal numbers 448 / m
// overflows and is no inverse of the s that is stored; there y is lifted by 2^64 first, exactly, and
// multiplied by the inverse of the lifted s.  A zero row (or one so small that s is 0) has codes 0; a
// scale that is not finite takes its row along.
struct E4m3Scale {
  float s, k;
  bool low;
};
constexpr float kLift = 18446744073709551616.f;  // 2^64
__device__ __forceinline__ E4m3Scale e4m3_scale(float m) {
  E4m3Scale c{m / kE4m3Max, kE4m3Max / m, false};
  if (c.s < 1.17549435e-38f) c.k = c.s == 0.f ? 0.f : 1.f / (c.s * kLift), c.low = true;
  if (c.s == INFINITY) c.k = 0.f;
  return c;
}
template <int VEC>
__device__ __forceinline__ void e4m3_lift(Lanes<VEC> *l, float lift = kLift) {
#pragma unroll
  for (int i = 0; i < lanes_of<VEC>(); ++i) l[i] = l[i] * splat<VEC>(lift);
}
// Largest magnitude of a chunk so far.
template <int VEC>
__device__ __forceinline__ float chunk_magnitude(float m, const Lanes<VEC> *l) {
  float v[VEC];
  from_lanes<VEC>(l, v);
#pragma unroll
  for (int i = 0; i < VEC; ++i) m = MaxMagnitudeOp::of(m, fabsf(v[i]));
  return m;
}

struct NormArgs {
  const void *x, *r, *w;
  void *y, *h;
  uint8_t *q;
  float *scales, *rstd;
  int64_t rows, dim;
  float eps;
  int w_bf16;
};

// Brings the rows of a block's next turn, which lie together, to L2 (whole 16-byte units): one
// instruction a tensor, and the next turn waits for L2 in place of HBM.
template <typename T, int VEC>
__device__ __forceinline__ void prefetch_rows(const T *p, int64_t base, int per, int64_t rows,
                                              int64_t dim) {
  if (VEC == 1 || p == nullptr || base >= rows) return;
  const uintptr_t from = (reinterpret_cast<uintptr_t>(p + base * dim) + 15) & ~(uintptr_t)15;
  const uintptr_t to =
      reinterpret_cast<uintptr_t>(p + (base + min((int64_t)per, rows - base)) * dim) &
      ~(uintptr_t)15;
  if (to > from) sm100::bulk_prefetch_l2(reinterpret_cast<const void *>(from), (uint32_t)(to - from));
}

// Rows whose length is no multiple of 16 bytes (SHIFT): a row's chunks start at the 16-byte boundary
// before it, so chunk c holds elements c VEC - shift on, and its first and last may be cut.  Every
// tensor of a call has the same shift in a row, and a thread's rows are a multiple of VEC apart, so
// its shift, its columns and their weights are the same in every row that it takes.
template <typename T, int VEC>
__device__ __forceinline__ int row_shift(const T *row) {
  return (int)((reinterpret_cast<uintptr_t>(row) & 15) / sizeof(T));
}
// A cut chunk is loaded whole, with elements of the rows beside it, which clear_outside makes 0 once
// every load of the row is on its way; where it reaches out of the tensor's `size` elements, by
// elements.
template <typename T, int VEC, bool SHIFT>
__device__ __forceinline__ void load_part(RowChunk<T, VEC> &k, const T *t, int64_t off, int e0, int dim,
                                          int64_t size) {
  if (!SHIFT || (off + e0 >= 0 && off + e0 + VEC <= size)) {
    k.load(t + off + e0);
  } else {
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      v[i] = e0 + i >= 0 && e0 + i < dim ? load_f(t, off + e0 + i) : 0.f;
    k.put(v);
  }
}
template <typename T, int VEC, bool SHIFT>
__device__ __forceinline__ void clear_outside(RowChunk<T, VEC> &k, int e0, int dim) {
  if (!SHIFT || (e0 >= 0 && e0 + VEC <= dim)) return;
  float v[VEC];
  k.get(v);
#pragma unroll
  for (int i = 0; i < VEC; ++i)
    if (e0 + i < 0 || e0 + i >= dim) v[i] = 0.f;
  k.put(v);
}
template <typename T, int VEC, bool SHIFT>
__device__ __forceinline__ void store_part(const RowChunk<T, VEC> &k, T *row, int e0, int dim) {
  if (!SHIFT || (e0 >= 0 && e0 + VEC <= dim)) {
    k.store(row + e0);
  } else {
    float v[VEC];
    k.get(v);
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      if (e0 + i >= 0 && e0 + i < dim) store_f(row, e0 + i, v[i]);
  }
}
template <int VEC, bool SHIFT>
__device__ __forceinline__ void weight_part(const void *w, bool w_bf16, int c, int e0, int dim,
                                            Lanes<VEC> *p) {
  if (!SHIFT) {
    weight_lanes<VEC>(w, w_bf16, c, p);
  } else {
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC; ++i)
      v[i] = e0 + i >= 0 && e0 + i < dim ? weight_at(w, w_bf16, e0 + i) : 0.f;
    to_lanes<VEC>(v, p);
  }
}

// G lanes a row (0: the block).  8 bits at 16384 x 4096 is near two bounds, HBM and 2.1 instructions a
// clock: a block of 128 threads a row took 95 us where a warp of 16 chunks a lane took 114, and with
// the arithmetic in packed pairs it takes 80 (82 since its largest value waits for rstd: of y, not of h w).
template <typename T, int VEC, int G, bool FP8, bool SHIFT>
__global__ void __launch_bounds__(G ? kSubThreads : kBlockThreads)
norm_forward_kernel(const NormArgs a) {
  constexpr int NV = chunks_of<VEC>();
  __shared__ float scratch[33];
  const int g = G ? G : blockDim.x;
  const int lane = threadIdx.x % g, sub = threadIdx.x / g, per = blockDim.x / g;
  const T *x = reinterpret_cast<const T *>(a.x), *r = reinterpret_cast<const T *>(a.r);
  const int dim = (int)a.dim;
  const int64_t size = a.rows * a.dim;
  const int shift =
      SHIFT ? row_shift<T, VEC>(x + ((int64_t)blockIdx.x * per + sub) * a.dim) : 0;
  const int nvec = (dim + shift + VEC - 1) / VEC;
  constexpr int NP = lanes_of<VEC>();
  using L = Lanes<VEC>;
  L w[NV][NP];  // a thread's columns are the same in every row
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int c = lane + j * g;
    if (c < nvec) weight_part<VEC, SHIFT>(a.w, a.w_bf16, c, c * VEC - shift, dim, w[j]);
  }
  for (int64_t base = (int64_t)blockIdx.x * per; base < a.rows;
       base += (int64_t)gridDim.x * per) {
    const int64_t row = base + sub;
    const bool live = row < a.rows;
    const int64_t off = row * a.dim;
    const int64_t next = base + (int64_t)gridDim.x * per;
    // (with several rows a block the loads in flight suffice, and the copies cost a sixth)
    if (G == 0 && threadIdx.x == 0) prefetch_rows<T, VEC>(x, next, per, a.rows, a.dim);
    if (G == 0 && threadIdx.x == blockDim.x - 1) prefetch_rows<T, VEC>(r, next, per, a.rows, a.dim);
    RowChunk<T, VEC> cx[NV], cr[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * g;
      cx[j].zero();
      if (live && c < nvec) load_part<T, VEC, SHIFT>(cx[j], x, off, c * VEC - shift, dim, size);
    }
    if (r) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = lane + j * g;
        cr[j].zero();
        if (live && c < nvec) load_part<T, VEC, SHIFT>(cr[j], r, off, c * VEC - shift, dim, size);
      }
    }
    L sum = splat<VEC>(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * g;
      L v[NP];
      clear_outside<T, VEC, SHIFT>(cx[j], c * VEC - shift, dim);
      get_lanes(cx[j], v);
      if (r) {
        L u[NP];
        clear_outside<T, VEC, SHIFT>(cr[j], c * VEC - shift, dim);
        get_lanes(cr[j], u);
#pragma unroll
        for (int i = 0; i < NP; ++i) v[i] = v[i] + u[i];
        put_lanes(cx[j], v);  // the stream, rounded to its type
        if (live && c < nvec)
          store_part<T, VEC, SHIFT>(cx[j], reinterpret_cast<T *>(a.h) + off, c * VEC - shift, dim);
        get_lanes(cx[j], v);
      }
#pragma unroll
      for (int i = 0; i < NP; ++i) sum = fma(v[i], v[i], sum);
    }
    const float ss = group_reduce<G, SumOp>(lane_sum(sum), scratch);
    const float rstd = 1.f / sqrtf(ss / (float)a.dim + a.eps);
    if (a.rstd && live && lane == 0) a.rstd[row] = rstd;
    if (FP8) {
      L t[NV][NP];  // y
      const L f = splat<VEC>(rstd);
      float m = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (lane + j * g >= nvec) continue;
        get_lanes(cx[j], t[j]);
#pragma unroll
        for (int i = 0; i < NP; ++i) t[j][i] = t[j][i] * f * w[j][i];
        m = chunk_magnitude<VEC>(m, t[j]);
      }
      m = group_reduce<G, MaxMagnitudeOp>(m, scratch);
      const E4m3Scale scale = e4m3_scale(m);
      if (live && lane == 0) a.scales[row] = scale.s;
      if (scale.low) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
          if (lane + j * g < nvec) e4m3_lift<VEC>(t[j]);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = lane + j * g;
        if (live && c < nvec)
          store_e4m3<VEC, SHIFT>(a.q + off, t[j], scale.k, c * VEC - shift, dim);
      }
    } else {
      const L f = splat<VEC>(rstd);
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = lane + j * g;
        if (!live || c >= nvec) continue;
        L v[NP];
        get_lanes(cx[j], v);
#pragma unroll
        for (int i = 0; i < NP; ++i) v[i] = v[i] * f * w[j][i];
        put_lanes(cx[j], v);
        store_part<T, VEC, SHIFT>(cx[j], reinterpret_cast<T *>(a.y) + off, c * VEC - shift, dim);
      }
    }
  }
}

// Rows that a block cannot hold: three sweeps, the later ones over the stream (or x) in L2.
template <typename T, bool FP8>
__global__ void __launch_bounds__(kWideThreads) norm_forward_wide_kernel(const NormArgs a) {
  __shared__ float scratch[33];
  const T *x = reinterpret_cast<const T *>(a.x), *r = reinterpret_cast<const T *>(a.r);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t off = row * a.dim;
    const T *h = r ? reinterpret_cast<const T *>(a.h) : x;
    float ss = 0.f;
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
      float v = load_f(x, off + c);
      if (r) {
        RowChunk<T, 1> k;
        v += load_f(r, off + c);
        k.put(&v);
        k.store(reinterpret_cast<T *>(a.h) + off + c);
        k.get(&v);
      }
      ss = fmaf(v, v, ss);
    }
    ss = group_reduce<0, SumOp>(ss, scratch);
    const float rstd = 1.f / sqrtf(ss / (float)a.dim + a.eps);
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = rstd;
    E4m3Scale scale{};
    if (FP8) {
      float m = 0.f;
      for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x)
        m = MaxMagnitudeOp::of(m, fabsf(load_f(h, off + c) * rstd * weight_at(a.w, a.w_bf16, c)));
      m = group_reduce<0, MaxMagnitudeOp>(m, scratch);
      scale = e4m3_scale(m);
      if (threadIdx.x == 0) a.scales[row] = scale.s;
    }
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const float y = load_f(h, off + c) * rstd * weight_at(a.w, a.w_bf16, c);
      if (FP8) {
        Single t{y};
        if (scale.low) e4m3_lift<1>(&t);
        store_e4m3<1>(a.q + off, &t, scale.k, c, 0);
      } else {
        store_f(reinterpret_cast<T *>(a.y), off + c, y);
      }
    }
  }
}

// A matrix's rows in e4m3 with the scale max|row| / 448: a serving program's weights, once, and the
// activations between two 8-bit products.  A block a row, the second sweep from L1 or L2.  The
// grid is what runs at once: 16384 x 4096 bf16 46 us, and 62 with a block an SM more than fits.
template <typename T, int VEC>
__global__ void __launch_bounds__(256)
quantize_rows_kernel(const T *__restrict__ x, int64_t rows, int64_t dim, uint8_t *q,
                     float *scales) {
  __shared__ float scratch[33];
  const int64_t nvec = dim / VEC;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *p = x + row * dim;
    float m = 0.f;
    for (int64_t c = threadIdx.x; c < nvec; c += blockDim.x) {
      RowChunk<T, VEC> u;
      Lanes<VEC> l[lanes_of<VEC>()];
      u.load(p + c * VEC);
      get_lanes(u, l);
      m = chunk_magnitude<VEC>(m, l);
    }
    m = group_reduce<0, MaxMagnitudeOp>(m, scratch);
    const E4m3Scale scale = e4m3_scale(m);
    if (threadIdx.x == 0) scales[row] = scale.s;
    const float lift = scale.low ? kLift : 1.f;
    for (int64_t c = threadIdx.x; c < nvec; c += blockDim.x) {
      RowChunk<T, VEC> u;
      Lanes<VEC> l[lanes_of<VEC>()];
      u.load(p + c * VEC);
      get_lanes(u, l);
      e4m3_lift<VEC>(l, lift);
      store_e4m3<VEC>(q + row * dim, l, scale.k, c * VEC, 0);
    }
  }
}

struct NormGradArgs {
  const void *h, *w, *dy, *dh;
  const float *rstd;
  void *dx;
  float *partial;  // [grid, dim] column sums of the blocks, or null
  int64_t rows, dim;
  int w_bf16;
};

// A thread keeps its columns' part of dw in registers over all of its block's rows; the blocks' sums
// are joined in block order by norm_columns_kernel, so the bits are the same every time.
// (In a block, a warp after another added to one row of sums, a shifted row after another: 64 turns, 30 us
// of any call of narrow odd rows; side by side, 102 x 74 takes 12 us for 33 and 28559 x 212 bf16 29 for 39.)
template <typename T, int VEC, int G, bool SHIFT>
__global__ void __launch_bounds__(G || (SHIFT && VEC == 8) ? kSubThreads : kBlockThreads)
norm_backward_kernel(const NormGradArgs a) {
  constexpr int NV = chunks_of<VEC>();
  __shared__ float scratch[33];
  // the block's sums of dw: a row of `dim` <= G NV VEC columns a warp, or a shifted row
  __shared__ float columns[!G ? 1 : (SHIFT ? kSubThreads / (G ? G : 1) : kSubThreads / 32) * G * NV * VEC];
  const int g = G ? G : blockDim.x;
  const int lane = threadIdx.x % g, sub = threadIdx.x / g, per = blockDim.x / g;
  const T *hp = reinterpret_cast<const T *>(a.h), *dyp = reinterpret_cast<const T *>(a.dy);
  const T *dhp = reinterpret_cast<const T *>(a.dh);
  const int dim = (int)a.dim;
  const int64_t size = a.rows * a.dim;
  const int shift =
      SHIFT ? row_shift<T, VEC>(hp + ((int64_t)blockIdx.x * per + sub) * a.dim) : 0;
  const int nvec = (dim + shift + VEC - 1) / VEC;
  constexpr int NP = lanes_of<VEC>();
  using L = Lanes<VEC>;
  L kept[SHIFT ? NV : 1][NP];  // weights that are no whole chunk of memory stay in registers
  if (SHIFT) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * g;
      if (c < nvec) weight_part<VEC, SHIFT>(a.w, a.w_bf16, c, c * VEC - shift, dim, kept[SHIFT ? j : 0]);
    }
  }
  auto weights = [&](int j, int c, L *w) {
    if (SHIFT) {
#pragma unroll
      for (int i = 0; i < NP; ++i) w[i] = kept[SHIFT ? j : 0][i];
    } else {
      weight_lanes<VEC>(a.w, a.w_bf16, c, w);
    }
  };
  L dwp[NV][NP];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < NP; ++i) dwp[j][i] = splat<VEC>(0.f);
  for (int64_t base = (int64_t)blockIdx.x * per; base < a.rows;
       base += (int64_t)gridDim.x * per) {
    const int64_t row = base + sub;
    const bool live = row < a.rows;
    const int64_t off = row * a.dim;
    const int64_t next = base + (int64_t)gridDim.x * per;
    if (threadIdx.x == 0) prefetch_rows<T, VEC>(hp, next, per, a.rows, a.dim);
    if (threadIdx.x == 32) prefetch_rows<T, VEC>(dyp, next, per, a.rows, a.dim);
    if (threadIdx.x == blockDim.x - 1) prefetch_rows<T, VEC>(dhp, next, per, a.rows, a.dim);
    RowChunk<T, VEC> ch[NV], cy[NV], cs[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * g;
      ch[j].zero(), cy[j].zero(), cs[j].zero();
      if (live && c < nvec) {
        const int e0 = c * VEC - shift;
        load_part<T, VEC, SHIFT>(ch[j], hp, off, e0, dim, size);
        load_part<T, VEC, SHIFT>(cy[j], dyp, off, e0, dim, size);
        if (dhp) load_part<T, VEC, SHIFT>(cs[j], dhp, off, e0, dim, size);
      }
    }
    const float rstd = live ? __ldg(a.rstd + row) : 0.f;
    const L f = splat<VEC>(rstd);
    L sum = splat<VEC>(0.f);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * g;
      if (c >= nvec) continue;
      clear_outside<T, VEC, SHIFT>(ch[j], c * VEC - shift, dim);
      clear_outside<T, VEC, SHIFT>(cy[j], c * VEC - shift, dim);
      L h[NP], dy[NP], w[NP];
      get_lanes(ch[j], h), get_lanes(cy[j], dy);
      weights(j, c, w);
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        const L t = dy[i] * (h[i] * f);
        dwp[j][i] = dwp[j][i] + t;
        sum = fma(t, w[i], sum);
      }
    }
    const float dot = group_reduce<G, SumOp>(lane_sum(sum), scratch);
    const float k = -dot / (float)a.dim * rstd;
    const L minus = splat<VEC>(k);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * g;
      if (!live || c >= nvec) continue;
      L h[NP], dy[NP], s[NP], w[NP];
      get_lanes(ch[j], h), get_lanes(cy[j], dy), get_lanes(cs[j], s);
      weights(j, c, w);
#pragma unroll
      for (int i = 0; i < NP; ++i) s[i] = fma(f, fma(h[i], minus, dy[i] * w[i]), s[i]);
      put_lanes(cs[j], s);
      store_part<T, VEC, SHIFT>(cs[j], reinterpret_cast<T *>(a.dx) + off, c * VEC - shift, dim);
    }
  }
  if (!a.partial) return;
  float dw[NV][VEC];
#pragma unroll
  for (int j = 0; j < NV; ++j) from_lanes<VEC>(dwp[j], dw[j]);
  float *out = a.partial + (int64_t)blockIdx.x * a.dim;
  auto each_column = [&](auto &&f) {  // (column, sum) of the thread's own
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int c = lane + j * g;
      if (c >= nvec) continue;
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const int col = c * VEC - shift + i;
        if (!SHIFT || (col >= 0 && col < dim)) f(col, dw[j][i]);
      }
    }
  };
  if (G == 0) {
    each_column([&](int col, float v) { out[col] = v; });
  } else {
    // A warp's rows are joined by shuffles, where their lanes hold the same columns, and its sums (or
    // each shifted row's) put side by side and added in order.
    if (!SHIFT) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < VEC; ++i)
#pragma unroll
          for (int o = 16; o >= (G ? G : 32); o >>= 1)
            dw[j][i] += __shfl_xor_sync(0xFFFFFFFFu, dw[j][i], o);
    }
    const int slots = SHIFT ? per : (int)blockDim.x / 32, slot = SHIFT ? sub : threadIdx.x / 32;
    if (SHIFT || (threadIdx.x & 31) < G)
      each_column([&](int col, float v) { columns[slot * dim + col] = v; });
    __syncthreads();
    for (int c = threadIdx.x; c < dim; c += blockDim.x) {
      float s = 0.f;
#pragma unroll 8
      for (int k = 0; k < slots; ++k) s += columns[k * dim + c];
      out[c] = s;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWideThreads) norm_backward_wide_kernel(const NormGradArgs a) {
  __shared__ float scratch[33];
  const T *hp = reinterpret_cast<const T *>(a.h), *dyp = reinterpret_cast<const T *>(a.dy);
  const T *dhp = reinterpret_cast<const T *>(a.dh);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t off = row * a.dim;
    const float rstd = __ldg(a.rstd + row);
    const bool first = row == blockIdx.x;
    float dot = 0.f;
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const float t = load_f(dyp, off + c) * (load_f(hp, off + c) * rstd);
      dot = fmaf(t, weight_at(a.w, a.w_bf16, c), dot);
      if (a.partial) {  // a thread's own columns
        float *p = a.partial + (int64_t)blockIdx.x * a.dim + c;
        *p = first ? t : *p + t;
      }
    }
    dot = group_reduce<0, SumOp>(dot, scratch);
    const float k = dot / (float)a.dim * rstd;
    for (int64_t c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const float gi = load_f(dyp, off + c) * weight_at(a.w, a.w_bf16, c);
      const float s = dhp ? load_f(dhp, off + c) : 0.f;
      store_f(reinterpret_cast<T *>(a.dx), off + c,
              fmaf(rstd, gi - load_f(hp, off + c) * k, s));
    }
  }
}

// dw = column sums of the blocks' partial sums, in block order.
__global__ void __launch_bounds__(32 * kReduceLanes)
norm_columns_kernel(const float *__restrict__ partial, int blocks, int64_t dim, void *dw,
                    int w_bf16) {
  __shared__ float part[kReduceLanes][33];
  const int64_t c = (int64_t)blockIdx.x * 32 + threadIdx.x;
  float s = 0.f;
  if (c < dim) {
#pragma unroll 4
    for (int b = threadIdx.y; b < blocks; b += kReduceLanes) s += partial[(int64_t)b * dim + c];
  }
  part[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.y == 0 && c < dim) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < kReduceLanes; ++i) s += part[i][threadIdx.x];
    if (w_bf16)
      store_f(reinterpret_cast<__nv_bfloat16 *>(dw), c, s);
    else
      reinterpret_cast<float *>(dw)[c] = s;
  }
}

// How rows are read: an element at a time, in chunks, or in chunks shifted to their boundaries.
enum RowAccess { kScalarRows, kChunkRows, kShiftedRows };

// Threads, lanes a row, row groups and blocks (at most) of a call (lanes 0: a block a row).
struct NormPlan {
  int lanes, threads, blocks;
  int64_t groups;
  RowAccess access;
  bool wide;
};

// Shifted rows: up to 512 threads, 256 for the gradient of bf16 rows, whose registers allow no more.
NormPlan norm_plan(int64_t rows, int64_t dim, int elem, RowAccess access, int blocks_per_sm,
                   int shifted_threads) {
  NormPlan p{};
  const int vec = 16 / elem;
  p.access = access;
  const int nv = access == kScalarRows ? 16 : 4;
  const int64_t nvec = access == kScalarRows  ? dim
                       : access == kChunkRows ? dim / vec
                                              : cdiv(dim + vec - 1, vec);
  int64_t per = 1;
  if (nvec <= (int64_t)32 * nv) {
    p.lanes = 4;
    while ((int64_t)p.lanes * nv < nvec) p.lanes *= 2;
    p.threads = kSubThreads;
    per = kSubThreads / p.lanes;
  } else if (nvec <= (int64_t)(access == kShiftedRows ? shifted_threads : kBlockThreads) * nv) {
    p.threads = (int)((cdiv(nvec, nv) + 31) / 32 * 32);
  } else if (access == kShiftedRows) {
    return norm_plan(rows, dim, elem, kScalarRows, blocks_per_sm, shifted_threads);
  } else {
    p.wide = true;
    p.threads = kWideThreads;
  }
  p.groups = cdiv(rows, per);
  // more blocks of few threads
  const int most = blocks_per_sm * std::max(1, 256 / p.threads);
  p.blocks = (int)std::min<int64_t>(p.groups, (int64_t)sm_count() * most);
  return p;
}

// `first` and `others`: the call's tensors of rows (null: none); w: its weight.
RowAccess row_access(int64_t dim, int elem, const void *w, const void *first,
                     std::initializer_list<const void *> others) {
  const int vec = 16 / elem;
  for (const void *p : others)
    if (p && ((reinterpret_cast<uintptr_t>(p) ^ reinterpret_cast<uintptr_t>(first)) & 15))
      return kScalarRows;
  if (dim % vec == 0 && aligned16(first) && aligned16(w)) return kChunkRows;
  return dim >= 2 * vec ? kShiftedRows : kScalarRows;
}

// The grid of a persistent kernel: as many blocks as run at once (a second, shorter wave would
// leave most of the GPU idle), at most p.blocks.
template <auto KERNEL>
int resident_blocks(const NormPlan &p) {
  static std::atomic<int> known[kWideThreads / 32 + 1];  // by threads
  std::atomic<int> &k = known[p.threads / 32];
  int n = k.load();
  if (n == 0) {
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, KERNEL, p.threads, 0) != cudaSuccess ||
        n < 1)
      n = 1;
    k.store(n);
  }
  const int64_t blocks = std::min<int64_t>(p.blocks, (int64_t)sm_count() * n);
  // shifted rows of a thread lie a multiple of 8 apart (several rows a block always do)
  return (int)(p.access == kShiftedRows && p.lanes == 0 && blocks < p.groups ? blocks / 8 * 8
                                                                             : blocks);
}

// most blocks of an SM; each of the gradient's writes its column sums
constexpr int kForwardBlocks = 32, kBackwardBlocks = 4;

template <auto KERNEL, typename A>
int launch_rows(const NormPlan &p, const A &a, cudaStream_t s) {
  const int blocks = resident_blocks<KERNEL>(p);
  KERNEL<<<blocks, p.threads, 0, s>>>(a);
  return blocks;
}

template <typename T, int VEC, bool FP8, bool SHIFT>
void launch_forward(const NormPlan &p, const NormArgs &a, cudaStream_t s) {
  switch (p.lanes) {
    case 4: launch_rows<norm_forward_kernel<T, VEC, 4, FP8, SHIFT>>(p, a, s); break;
    case 8: launch_rows<norm_forward_kernel<T, VEC, 8, FP8, SHIFT>>(p, a, s); break;
    case 16: launch_rows<norm_forward_kernel<T, VEC, 16, FP8, SHIFT>>(p, a, s); break;
    case 32: launch_rows<norm_forward_kernel<T, VEC, 32, FP8, SHIFT>>(p, a, s); break;
    default: launch_rows<norm_forward_kernel<T, VEC, 0, FP8, SHIFT>>(p, a, s); break;
  }
}

template <typename T, bool FP8>
int forward_typed(const NormArgs &a, cudaStream_t s) {
  RowAccess access = row_access(a.dim, sizeof(T), a.w, a.x, {a.r, a.h, a.y});
  if (access == kChunkRows && !aligned16(a.q)) access = kShiftedRows;
  const NormPlan p = norm_plan(a.rows, a.dim, sizeof(T), access, kForwardBlocks, kBlockThreads);
  if (p.wide)
    launch_rows<norm_forward_wide_kernel<T, FP8>>(p, a, s);
  else if (p.access == kChunkRows)
    launch_forward<T, vec_of<T>(), FP8, false>(p, a, s);
  else if (p.access == kShiftedRows)
    launch_forward<T, vec_of<T>(), FP8, true>(p, a, s);
  else
    launch_forward<T, 1, FP8, false>(p, a, s);
  return after_launch("norm_forward_kernel");
}

template <typename T>
int quantize_typed(const T *x, int64_t rows, int64_t dim, uint8_t *q, float *scales,
                   cudaStream_t s) {
  constexpr int VEC = vec_of<T>();
  const bool vec = dim % VEC == 0 && aligned16(x) && aligned16(q);
  const int64_t nvec = vec ? dim / VEC : dim;
  NormPlan p{};
  p.access = vec ? kChunkRows : kScalarRows;
  p.threads = (int)std::min<int64_t>(256, (nvec + 31) / 32 * 32);
  p.groups = rows;
  p.blocks = (int)std::min<int64_t>(rows, (int64_t)sm_count() * (2048 / p.threads));
  if (vec)
    quantize_rows_kernel<T, VEC><<<resident_blocks<quantize_rows_kernel<T, VEC>>(p), p.threads, 0, s>>>(
        x, rows, dim, q, scales);
  else
    quantize_rows_kernel<T, 1><<<resident_blocks<quantize_rows_kernel<T, 1>>(p), p.threads, 0, s>>>(
        x, rows, dim, q, scales);
  return after_launch("quantize_rows_kernel");
}

// The gradient's kernel; returns its blocks.
template <typename T, int VEC, bool SHIFT>
int launch_backward(const NormPlan &p, const NormGradArgs &a, cudaStream_t s) {
  switch (p.lanes) {
    case 4: return launch_rows<norm_backward_kernel<T, VEC, 4, SHIFT>>(p, a, s);
    case 8: return launch_rows<norm_backward_kernel<T, VEC, 8, SHIFT>>(p, a, s);
    case 16: return launch_rows<norm_backward_kernel<T, VEC, 16, SHIFT>>(p, a, s);
    case 32: return launch_rows<norm_backward_kernel<T, VEC, 32, SHIFT>>(p, a, s);
    default: return launch_rows<norm_backward_kernel<T, VEC, 0, SHIFT>>(p, a, s);
  }
}

template <typename T>
int backward_typed(const NormPlan &p, const NormGradArgs &a, cudaStream_t s) {
  if (p.wide) return launch_rows<norm_backward_wide_kernel<T>>(p, a, s);
  switch (p.access) {
    case kChunkRows: return launch_backward<T, vec_of<T>(), false>(p, a, s);
    case kShiftedRows: return launch_backward<T, vec_of<T>(), true>(p, a, s);
    default: return launch_backward<T, 1, false>(p, a, s);
  }
}

int check_norm(const char *what, int64_t rows, int64_t dim, int dtype, int weight_dtype,
               float eps) {
  if (rows < 0 || dim < 1)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: rows %lld, dim %lld", what, (long long)rows,
                (long long)dim);
  if (dim > (int64_t)1 << 30 || (rows > 0 && dim > ((int64_t)1 << 46) / rows))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: %lld x %lld elements are too many", what,
                (long long)rows, (long long)dim);
  if (dtype != LNET_F32 && dtype != LNET_BF16)
    return fail(LNET_ERR_UNSUPPORTED, "%s: dtype must be fp32 or bf16", what);
  if (weight_dtype != LNET_F32 && weight_dtype != LNET_BF16)
    return fail(LNET_ERR_UNSUPPORTED, "%s: the weight must be fp32 or bf16", what);
  if (!(eps >= 0.f)) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: eps must be >= 0", what);
  return LNET_OK;
}

NormPlan grad_plan(int64_t rows, int64_t dim, int elem, RowAccess access) {
  return norm_plan(rows, dim, elem, access, kBackwardBlocks, elem == 2 ? kSubThreads : kBlockThreads);
}
int norm_grad_blocks(int64_t rows, int64_t dim, int elem) {
  // the most of any access: the size query does not see the pointers
  int blocks = 0;
  for (RowAccess a : {kScalarRows, kChunkRows, kShiftedRows})
    blocks = std::max(blocks, grad_plan(rows, dim, elem, a).blocks);
  return blocks;
}

}  // namespace
}  // namespace lnet

using namespace lnet;

extern "C" int lnet_b200_residual_rms_norm(const void *x, const void *residual, const void *weight,
                                           int32_t dtype, int32_t weight_dtype, int64_t rows,
                                           int64_t dim, float eps, void *y, void *stream_out,
                                           float *rstd, lnet_stream_t stream) {
  const char *what = "residual_rms_norm";
  LNET_TRY(check_norm(what, rows, dim, dtype, weight_dtype, eps));
  reset_launches();
  if (rows == 0) return LNET_OK;
  if (!x || !weight || !y || (residual && !stream_out))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: x, weight, y%s must not be NULL", what,
                residual ? ", stream_out" : "");
  begin_entry(stream);
  NormArgs a{x, residual, weight, y, stream_out, nullptr, nullptr, rstd, rows, dim, eps,
             weight_dtype == LNET_BF16};
  return dtype == LNET_BF16 ? forward_typed<__nv_bfloat16, false>(a, stream)
                            : forward_typed<float, false>(a, stream);
}

extern "C" int lnet_b200_residual_rms_norm_fp8(const void *x, const void *residual,
                                               const void *weight, int32_t dtype,
                                               int32_t weight_dtype, int64_t rows, int64_t dim,
                                               float eps, uint8_t *values, float *scales,
                                               void *stream_out, lnet_stream_t stream) {
  const char *what = "residual_rms_norm_fp8";
  LNET_TRY(check_norm(what, rows, dim, dtype, weight_dtype, eps));
  reset_launches();
  if (rows == 0) return LNET_OK;
  if (!x || !weight || !values || !scales || (residual && !stream_out))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: x, weight, values, scales%s must not be NULL",
                what, residual ? ", stream_out" : "");
  begin_entry(stream);
  NormArgs a{x, residual, weight, nullptr, stream_out, values, scales, nullptr, rows, dim, eps,
             weight_dtype == LNET_BF16};
  return dtype == LNET_BF16 ? forward_typed<__nv_bfloat16, true>(a, stream)
                            : forward_typed<float, true>(a, stream);
}

extern "C" int lnet_b200_quantize_rows_fp8(const void *x, int32_t dtype, int64_t rows,
                                           int64_t dim, uint8_t *values, float *scales,
                                           lnet_stream_t stream) {
  const char *what = "quantize_rows_fp8";
  LNET_TRY(check_norm(what, rows, dim, dtype, LNET_F32, 0.f));
  reset_launches();
  if (rows == 0) return LNET_OK;
  if (!x || !values || !scales)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: x, values, scales must not be NULL", what);
  begin_entry(stream);
  return dtype == LNET_BF16
             ? quantize_typed(reinterpret_cast<const __nv_bfloat16 *>(x), rows, dim, values, scales,
                              stream)
             : quantize_typed(reinterpret_cast<const float *>(x), rows, dim, values, scales, stream);
}

extern "C" int lnet_b200_residual_rms_norm_workspace_size(int32_t dtype, int64_t rows, int64_t dim,
                                                          size_t *bytes) {
  const char *what = "residual_rms_norm_workspace_size";
  LNET_TRY(check_norm(what, rows, dim, dtype, LNET_F32, 0.f));
  if (!bytes) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: bytes must not be NULL", what);
  *bytes = rows == 0 ? 0
                     : (size_t)norm_grad_blocks(rows, dim, dtype == LNET_BF16 ? 2 : 4) *
                           (size_t)dim * sizeof(float);
  return LNET_OK;
}

extern "C" int lnet_b200_residual_rms_norm_backward(
    const void *stream_in, const float *rstd, const void *weight, const void *dy,
    const void *dstream, int32_t dtype, int32_t weight_dtype, int64_t rows, int64_t dim, void *dx,
    void *dweight, void *workspace, size_t workspace_bytes, lnet_stream_t stream) {
  const char *what = "residual_rms_norm_backward";
  LNET_TRY(check_norm(what, rows, dim, dtype, weight_dtype, 0.f));
  reset_launches();
  if (rows > 0 && (!stream_in || !rstd || !weight || !dy || !dx))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: stream, rstd, weight, dy, dx must not be NULL",
                what);
  begin_entry(stream);
  if (rows == 0) {
    if (dweight)
      LNET_TRY(cuda_check(cudaMemsetAsync(dweight, 0, dim * (weight_dtype == LNET_BF16 ? 2 : 4),
                                          stream),
                          what));
    return LNET_OK;
  }
  const int elem = dtype == LNET_BF16 ? 2 : 4;
  const RowAccess access = row_access(dim, elem, weight, stream_in, {dy, dstream, dx});
  const NormPlan p = grad_plan(rows, dim, elem, access);
  const size_t need = dweight ? (size_t)p.blocks * (size_t)dim * sizeof(float) : 0;
  if (need > workspace_bytes || (need && !workspace))
    return fail(LNET_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", what, need,
                workspace_bytes);
  NormGradArgs a{stream_in, weight, dy, dstream, rstd, dx,
                 dweight ? reinterpret_cast<float *>(workspace) : nullptr, rows, dim,
                 weight_dtype == LNET_BF16};
  const int blocks = dtype == LNET_BF16 ? backward_typed<__nv_bfloat16>(p, a, stream)
                                        : backward_typed<float>(p, a, stream);
  LNET_TRY(after_launch("norm_backward_kernel"));
  if (dweight) {
    norm_columns_kernel<<<(unsigned)cdiv(dim, 32), dim3(32, kReduceLanes), 0, stream>>>(
        a.partial, blocks, dim, dweight, a.w_bf16);
    LNET_TRY(after_launch("norm_columns_kernel"));
  }
  return LNET_OK;
}

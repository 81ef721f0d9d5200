// Row-wise helpers of the feed-forward and distillation operators: 16-byte or
// scalar chunks of a row in fp32, reductions over a group of lanes or a block.
#pragma once

#include <atomic>
#include <type_traits>

#include "common.cuh"

namespace lnet {

constexpr float kLog2e = 1.4426950408889634f;

// VEC consecutive elements of a row: 16 bytes, or one element where the row's
// pitch or base does not keep 16-byte alignment.
template <typename T, int VEC>
struct RowChunk {
  static_assert(VEC == 1 || VEC * sizeof(T) == 16, "a chunk is one element or 16 bytes");
};

template <>
struct RowChunk<float, 1> {
  float raw;
  __device__ __forceinline__ void load(const float *p) { raw = __ldg(p); }
  __device__ __forceinline__ void store(float *p) const { *p = raw; }
  __device__ __forceinline__ void zero() { raw = 0.f; }
  __device__ __forceinline__ void get(float *v) const { v[0] = raw; }
  __device__ __forceinline__ void put(const float *v) { raw = v[0]; }
};
template <>
struct RowChunk<__nv_bfloat16, 1> {
  uint16_t raw;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
    raw = __ldg(reinterpret_cast<const uint16_t *>(p));
  }
  __device__ __forceinline__ void store(__nv_bfloat16 *p) const {
    *reinterpret_cast<uint16_t *>(p) = raw;
  }
  __device__ __forceinline__ void zero() { raw = 0; }
  __device__ __forceinline__ void get(float *v) const {
    v[0] = __uint_as_float((uint32_t)raw << 16);
  }
  __device__ __forceinline__ void put(const float *v) {
    raw = __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
  }
};
template <>  // (a pair, for bf16 rows that start on 4-byte boundaries only)
struct RowChunk<__nv_bfloat16, 2> {
  uint32_t raw;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
    raw = __ldg(reinterpret_cast<const uint32_t *>(p));
  }
  __device__ __forceinline__ void store(__nv_bfloat16 *p) const {
    *reinterpret_cast<uint32_t *>(p) = raw;
  }
  __device__ __forceinline__ void zero() { raw = 0; }
  __device__ __forceinline__ void get(float *v) const {
    v[0] = __uint_as_float(raw << 16);
    v[1] = __uint_as_float(raw & 0xFFFF0000u);
  }
  __device__ __forceinline__ void put(const float *v) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(v[0], v[1]);
    raw = *reinterpret_cast<const uint32_t *>(&b);
  }
};
template <>
struct RowChunk<float, 4> {
  float4 raw;
  __device__ __forceinline__ void load(const float *p) {
    raw = __ldg(reinterpret_cast<const float4 *>(p));
  }
  __device__ __forceinline__ void store(float *p) const { *reinterpret_cast<float4 *>(p) = raw; }
  __device__ __forceinline__ void zero() { raw = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void get(float *v) const {
    v[0] = raw.x, v[1] = raw.y, v[2] = raw.z, v[3] = raw.w;
  }
  __device__ __forceinline__ void put(const float *v) {
    raw = make_float4(v[0], v[1], v[2], v[3]);
  }
};
template <>
struct RowChunk<__nv_bfloat16, 8> {
  uint4 raw;
  __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
    raw = __ldg(reinterpret_cast<const uint4 *>(p));
  }
  __device__ __forceinline__ void store(__nv_bfloat16 *p) const {
    *reinterpret_cast<uint4 *>(p) = raw;
  }
  __device__ __forceinline__ void zero() { raw = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void get(float *v) const {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  __device__ __forceinline__ void put(const float *v) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 b = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t *>(&b);
    }
    raw = make_uint4(w[0], w[1], w[2], w[3]);
  }
};

template <typename T>
__host__ __device__ constexpr int vec_of() {
  return 16 / (int)sizeof(T);
}

struct SumOp {
  static __device__ __forceinline__ float id() { return 0.f; }
  static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
// Of magnitudes, as the integers that their bits are: a NaN is above infinity and stays.
struct MaxMagnitudeOp {
  static __device__ __forceinline__ float id() { return 0.f; }
  static __device__ __forceinline__ float of(float a, float b) {
    return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
  }
};

// Reduction over G lanes of a warp (G a power of two), or over the block where
// G = 0 (`scratch`: 33 floats of shared memory; the block's size is a multiple
// of 32).  Every thread gets the result.
template <int G, typename Op>
__device__ __forceinline__ float group_reduce(float v, float *scratch) {
  constexpr int W = G == 0 ? 32 : G;
  if (W == 32 && std::is_same<Op, MaxMagnitudeOp>::value) {
    v = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(v)));
  } else {
#pragma unroll
    for (int o = W / 2; o > 0; o >>= 1) v = Op::of(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  }
  if (G == 0) {
    const int warps = blockDim.x >> 5;
    if (warps == 1) return v;
    __syncthreads();  // the scratch of an earlier reduction has been read
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    v = (threadIdx.x & 31) < warps ? scratch[threadIdx.x & 31] : Op::id();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v = Op::of(v, __shfl_xor_sync(0xFFFFFFFFu, v, o));
  }
  return v;
}

// ex2.approx (2 ulp), results below 2^-126 flushed to zero
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Two fp32 values in one register pair: one instruction for both.
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void unpair(Pair p, float &a, float &b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v));
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair p;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair p;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(p.v) : "l"(a.v), "l"(b.v));
  return p;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair p;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(p.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return p;
}
__device__ __forceinline__ Pair exp2_fast(Pair x) {
  float a, b;
  unpair(x, a, b);
  return pair(exp2_fast(a), exp2_fast(b));
}

// A chunk in the form that is computed with: pairs, or its one element.
struct Single {
  float v;
};
__device__ __forceinline__ Single operator+(Single a, Single b) { return {a.v + b.v}; }
__device__ __forceinline__ Single operator*(Single a, Single b) { return {a.v * b.v}; }
__device__ __forceinline__ Single fma(Single a, Single b, Single c) { return {fmaf(a.v, b.v, c.v)}; }
template <int VEC>
using Lanes = std::conditional_t<VEC == 1, Single, Pair>;
template <int VEC>
__host__ __device__ constexpr int lanes_of() {
  return VEC == 1 ? 1 : VEC / 2;
}
template <int VEC>
__device__ __forceinline__ Lanes<VEC> splat(float v) {
  if constexpr (VEC == 1)
    return Single{v};
  else
    return pair(v, v);
}
template <int VEC>
__device__ __forceinline__ void to_lanes(const float *v, Lanes<VEC> *p) {
  if constexpr (VEC == 1) {
    p[0].v = v[0];
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) p[i] = pair(v[2 * i], v[2 * i + 1]);
  }
}
template <int VEC>
__device__ __forceinline__ void from_lanes(const Lanes<VEC> *p, float *v) {
  if constexpr (VEC == 1) {
    v[0] = p[0].v;
  } else {
#pragma unroll
    for (int i = 0; i < VEC / 2; ++i) unpair(p[i], v[2 * i], v[2 * i + 1]);
  }
}
__device__ __forceinline__ float lane_sum(Single a) { return a.v; }
__device__ __forceinline__ float lane_sum(Pair a) {
  float x, y;
  unpair(a, x, y);
  return x + y;
}
template <typename T, int VEC>
__device__ __forceinline__ void get_lanes(const RowChunk<T, VEC> &c, Lanes<VEC> *p) {
  float v[VEC];
  c.get(v);
  to_lanes<VEC>(v, p);
}
template <typename T, int VEC>
__device__ __forceinline__ void put_lanes(RowChunk<T, VEC> &c, const Lanes<VEC> *p) {
  float v[VEC];
  from_lanes<VEC>(p, v);
  c.put(v);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Raises a kernel's limit of dynamic shared memory on the current device, once a device.
template <auto KERNEL>
int raise_shared_memory(int bytes, const char *what) {
  static std::atomic<uint64_t> ready{0};
  int dev = 0;
  LNET_TRY(cuda_check(cudaGetDevice(&dev), what));
  const uint64_t bit = (uint64_t)1 << (dev & 63);
  if (ready.load() & bit) return LNET_OK;
  LNET_TRY(cuda_check(
      cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes), what));
  ready.fetch_or(bit);
  return LNET_OK;
}

// SMs of the current device (queried once per process; every GPU of a machine is
// the same part).
inline int sm_count() {
  static const int n = [] {
    int dev = 0, v = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1)
      v = 148;
    return v;
  }();
  return n;
}

}  // namespace lnet

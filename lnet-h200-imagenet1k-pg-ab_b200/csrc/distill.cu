// Distillation from a teacher's top logits, mixed with hard labels.
//
// Row i: entries j with index >= 0 and a teacher logit above -inf,
//   p_j = softmax(t_j / tau) over them,   q = softmax(z / tau) over all classes,
//   KL = sum_j p_j (log p_j - log q_j),   CE = logsumexp(z) - z[label],
//   loss = alpha tau^2 KL [entries] + (1 - alpha) CE [label >= 0],
//   dz = alpha tau (q - p) [entries] + (1 - alpha) (softmax(z) - onehot) [label >= 0].
// A part with weight 0 is left out.  A class at -inf has q = 0 (the loss is +inf
// where the teacher gives it mass); a row that is -inf throughout has q = 0
// everywhere.  A row with neither entries nor a label has loss and gradient 0
// whatever its logits are.  An index or label past the classes makes the row's
// loss NaN and touches nothing else.
//
// Two kernels.  With a gradient, and rows that 8 blocks hold, the row stays on
// chip (distill_resident_kernel below).  The loss alone, longer rows, and a
// gradient whose alignment differs from z's or that has more than 256 entries a row
// take distill_row_kernel: one sweep
// reads the row for its running maximum and exponential sums (one sum for each
// of the temperatures tau and 1 that the loss needs), a second one writes the
// gradient from the row in L2 or L1.  In both the few entries of the teacher and
// the label are then corrected in place, each from z again, so that every value
// is rounded once.  A row belongs to a block, or to a cluster of up to 8 blocks
// that join their sums through distributed shared memory.
#include <cooperative_groups.h>

#include <string.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "rows.cuh"
#include "sm100.cuh"

namespace cg = cooperative_groups;

namespace lnet {
namespace {

constexpr float kLowest = -3.402823466e+38f;
constexpr int kCountThreads = 256;
constexpr int kSumThreads = 1024;
constexpr int kEntries = 256;  // most entries of a row that are corrected one by one
constexpr int kWindow = 4096;  // classes whose masses a block holds at once

struct DistillArgs {
  const void *z;
  const int64_t *index, *labels;  // labels may be null
  const float *teacher;
  const int *counts;        // per-block counts of the counted rows, or null
  const float *upstream;    // gradient of the loss (one, or one a row), or null: 1
  float *loss;              // [rows], or null
  void *dz;                 // or null
  int64_t rows, classes, top;
  float tau, alpha;
  int n_counts, upstream_rows;
};

// Largest element of a chunk (NaN only where every element is).
__device__ __forceinline__ float chunk_max(const RowChunk<float, 4> &k) {
  return fmaxf(fmaxf(k.raw.x, k.raw.y), fmaxf(k.raw.z, k.raw.w));
}
__device__ __forceinline__ float chunk_max(const RowChunk<__nv_bfloat16, 8> &k) {
  const __nv_bfloat162 *w = reinterpret_cast<const __nv_bfloat162 *>(&k.raw);
  const __nv_bfloat162 m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
  return fmaxf(__low2float(m), __high2float(m));
}

// Maximum over a warp (a NaN is passed over).
__device__ __forceinline__ float warp_max(float v) {
  float m;
  asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// Running maximum m and sums of exp((z - m) / tau), exp(z - m).
struct RowStats {
  float m, st, s1;
};

template <bool TWO>
__device__ __forceinline__ void stats_join(RowStats &a, const RowStats &b, float kt) {
  const float m = fmaxf(a.m, b.m);
  a.st = a.st * exp2_fast((a.m - m) * kt) + b.st * exp2_fast((b.m - m) * kt);
  if (TWO) a.s1 = a.s1 * exp2_fast((a.m - m) * kLog2e) + b.s1 * exp2_fast((b.m - m) * kLog2e);
  a.m = m;
}

// Joined over a warp.
template <bool TWO>
__device__ __forceinline__ RowStats stats_warp(RowStats a, float kt) {
  const float m = warp_max(a.m);
  a.st *= exp2_fast((a.m - m) * kt);
  if (TWO) a.s1 *= exp2_fast((a.m - m) * kLog2e);
  a.m = m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    a.st += __shfl_xor_sync(0xFFFFFFFFu, a.st, o);
    if (TWO) a.s1 += __shfl_xor_sync(0xFFFFFFFFu, a.s1, o);
  }
  return a;
}

template <bool TWO, int N>
__device__ __forceinline__ void stats_add(RowStats &a, const float *v, float kt) {
  float m = v[0];
#pragma unroll
  for (int i = 1; i < N; ++i) m = fmaxf(m, v[i]);
  if (m > a.m) {
    a.st *= exp2_fast((a.m - m) * kt);
    if (TWO) a.s1 *= exp2_fast((a.m - m) * kLog2e);
    a.m = m;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    a.st += exp2_fast((v[i] - a.m) * kt);
    if (TWO) a.s1 += exp2_fast((v[i] - a.m) * kLog2e);
  }
}

// 5 rows of 100003 bf16 classes, two temperatures, loss alone, cold: 9.0 us with the teacher's
// entries fetched while the row is read and sums joined by warps (10.2 with the entries after the
// row's sums and one barrier a quantity); the chain of load, join over the block, join over the
// cluster bounds it.
// MANY: a gradient with more than kEntries entries, which are added up class by class; fewer are corrected
// one by one, each with a look at all of them.  296 rows of 70001 bf16 classes with 64, 256, 512, 1024
// and 4096 entries: 62, 71, 85, 117, 279 us by classes, 38, 51, 103, 298, 4067 one by one; 296 x 32768
// with 16384 415 us and 87 ms.
template <typename T, bool TWO, bool MANY>
__global__ void distill_row_kernel(const DistillArgs a) {
  constexpr int VEC = vec_of<T>();
  constexpr int U = 4;  // chunks in flight a thread
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  __shared__ RowStats warp_stats[32];
  __shared__ float3 warp_teacher[32];  // largest logit, sum of e^((t - largest) / tau), flags
  __shared__ RowStats block_stats;
  __shared__ float scratch[33];
  const int tid = threadIdx.x, nt = blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  const int64_t row = blockIdx.x / parts;
  const T *z = reinterpret_cast<const T *>(a.z) + row * a.classes;
  T *dz = reinterpret_cast<T *>(a.dz) + (a.dz ? row * a.classes : 0);
  const int64_t *index = a.index + row * a.top;
  const float *teacher = a.teacher + row * a.top;
  const bool use_kl = a.alpha != 0.f;
  const bool use_ce = a.labels != nullptr && a.alpha != 1.f;
  const float kt = kLog2e / a.tau;

  // This block's classes: [lo, hi), cut where z is 16-byte aligned; [va, vb) in chunks.
  const int64_t head0 = std::min<int64_t>(
      a.classes, (int64_t)((16 - (reinterpret_cast<uintptr_t>(z) & 15)) & 15) / sizeof(T));
  const int64_t chunks = (a.classes - head0) / VEC;
  const int64_t c0 = chunks * part / parts, c1 = chunks * (part + 1) / parts;
  const int64_t va = head0 + c0 * VEC, vb = head0 + c1 * VEC;
  const int64_t lo = part == 0 ? 0 : va, hi = part == parts - 1 ? a.classes : vb;
  const int nc = (int)(c1 - c0);

  // The thread's first entry, on its way while the row is read.
  int64_t ix0 = -1;
  float t0 = 0.f;
  if (use_kl && tid < a.top) ix0 = index[tid], t0 = teacher[tid];
  const int64_t label = use_ce ? a.labels[row] : -1;

  // ---- running maximum and sums
  RowStats st{kLowest, 0.f, 0.f};
  {
    const T *zv = z + va;
    int c = tid;
    for (; c + (U - 1) * nt < nc; c += U * nt) {
      RowChunk<T, VEC> k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) k[u].load(zv + (int64_t)(c + u * nt) * VEC);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[VEC];
        k[u].get(v);
        stats_add<TWO, VEC>(st, v, kt);
      }
    }
    for (; c < nc; c += nt) {
      RowChunk<T, VEC> k;
      k.load(zv + (int64_t)c * VEC);
      float v[VEC];
      k.get(v);
      stats_add<TWO, VEC>(st, v, kt);
    }
    for (int64_t i = lo + tid; i < va; i += nt) {
      const float v = load_f(z, i);
      stats_add<TWO, 1>(st, &v, kt);
    }
    for (int64_t i = vb + tid; i < hi; i += nt) {
      const float v = load_f(z, i);
      stats_add<TWO, 1>(st, &v, kt);
    }
  }
  // ---- the teacher's largest logit and sum, of the thread's entries
  float tmax = kLowest, tsum = 0.f;
  int flags = 0;  // 1 an entry, 2 an index past the classes
  float z0 = 0.f;
  if (use_kl) {
    for (int64_t j = tid; j < a.top; j += nt) {
      const int64_t ix = j == tid ? ix0 : index[j];
      const float t = j == tid ? t0 : teacher[j];
      if (ix < 0 || t == -INFINITY) continue;
      flags |= ix >= a.classes ? 3 : 1;
      if (j == tid && ix < a.classes && a.loss && part == 0) z0 = load_f(z, ix);
      const float m = fmaxf(tmax, t);
      tsum = tsum * exp2f((tmax - m) * kt) + exp2f((t - m) * kt);
      tmax = m;
    }
  }

  // ---- joined over the block, and the row's sums over the cluster
  st = stats_warp<TWO>(st, kt);
  auto teacher_warp = [&] {
    const float m = warp_max(tmax);
    tsum *= exp2f((tmax - m) * kt);
    tmax = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) tsum += __shfl_xor_sync(0xFFFFFFFFu, tsum, o);
    flags = __reduce_or_sync(0xFFFFFFFFu, flags);
  };
  if (use_kl) teacher_warp();
  if (lane == 0) {
    warp_stats[warp] = st;
    warp_teacher[warp] = make_float3(tmax, tsum, __int_as_float(flags));
  }
  __syncthreads();
  st = stats_warp<TWO>(lane < warps ? warp_stats[lane] : RowStats{kLowest, 0.f, 0.f}, kt);
  if (use_kl) {
    const float3 w = lane < warps ? warp_teacher[lane] : make_float3(kLowest, 0.f, 0.f);
    tmax = w.x, tsum = w.y, flags = __float_as_int(w.z);
    teacher_warp();
  }
  if (parts > 1) {
    if (tid == 0) block_stats = st;
    cluster.sync();
    if (a.dz || part == 0)
      st = stats_warp<TWO>(lane < parts ? *cluster.map_shared_rank(&block_stats, lane)
                                        : RowStats{kLowest, 0.f, 0.f},
                           kt);
    cluster.barrier_arrive();  // waited for at the end: no block leaves while another reads its sums
  }
  auto leave = [&] {
    if (parts > 1) cluster.barrier_wait();
  };
  // a row that is -inf throughout: q = 0, log q = -inf
  const float inv_t = st.st == 0.f ? 0.f : 1.f / st.st;
  const float s_one = TWO ? st.s1 : st.st;  // one temperature: tau = 1, or no label part
  const float inv_1 = s_one == 0.f ? 0.f : 1.f / s_one;
  const bool has_t = (flags & 1) != 0, has_l = label >= 0;
  const bool bad = (flags & 2) != 0 || label >= a.classes;
  const float log_st = logf(st.st), log_tsum = logf(tsum);

  // ---- the loss
  if (a.loss && part == 0) {
    float kl = 0.f;
    if (has_t && !bad) {
      for (int64_t j = tid; j < a.top; j += nt) {
        const int64_t ix = j == tid ? ix0 : index[j];
        const float t = j == tid ? t0 : teacher[j];
        if (ix < 0 || t == -INFINITY) continue;
        const float lt = (t - tmax) / a.tau;
        const float p = exp2f((t - tmax) * kt) / tsum;
        const float zq = j == tid ? z0 : load_f(z, ix);
        const float lq = zq == -INFINITY ? -INFINITY : (zq - st.m) / a.tau - log_st;
        if (p != 0.f) kl += p * ((lt - log_tsum) - lq);
      }
    }
    // (up to 32 entries are warp 0's)
    kl = a.top <= 32 ? group_reduce<32, SumOp>(kl, scratch) : group_reduce<0, SumOp>(kl, scratch);
    if (tid == 0) {
      float loss = has_t ? a.alpha * a.tau * a.tau * kl : 0.f;
      if (has_l && !bad) {
        const float zl = load_f(z, label);
        const float ce = zl == -INFINITY ? INFINITY : logf(s_one) + (st.m - zl);
        loss += (1.f - a.alpha) * ce;
      }
      a.loss[row] = bad ? NAN : loss;
    }
  }
  if (!a.dz) return leave();

  // ---- the gradient: at * e^((z - m) / tau) + a1 * e^(z - m), then the entries
  float scale = 1.f;
  if (a.counts) {
    int n = 0;
    for (int i = tid & 31; i < a.n_counts; i += 32) n += a.counts[i];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xFFFFFFFFu, n, o);
    scale = 1.f / (float)(n > 0 ? n : 1);
  }
  if (a.upstream) scale *= a.upstream[a.upstream_rows ? row : 0];
  if (bad) scale = NAN;
  const float ct = has_t ? a.alpha * a.tau * scale : 0.f;
  const float c1s = has_l ? (1.f - a.alpha) * scale : 0.f;
  const bool idle = !has_t && !has_l;  // no target: the gradient is 0 whatever the logits are
  float at = ct * inv_t, a1 = c1s * inv_1;
  if (!TWO) {
    at += a1;
    a1 = 0.f;
  }
  const float m = st.m;
  auto grad = [&](float v) {
    float g = at * exp2_fast((v - m) * kt);
    if (TWO) g = fmaf(a1, exp2_fast((v - m) * kLog2e), g);
    return idle ? 0.f : g;
  };
  const bool same_alignment =
      ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(dz)) & 15) == 0;
  if (same_alignment) {
    const T *zv = z + va;
    T *gv = dz + va;
    int c = tid;
    for (; c + (U - 1) * nt < nc; c += U * nt) {
      RowChunk<T, VEC> k[U];
#pragma unroll
      for (int u = 0; u < U; ++u) k[u].load(zv + (int64_t)(c + u * nt) * VEC);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float v[VEC];
        k[u].get(v);
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = grad(v[i]);
        k[u].put(v);
        k[u].store(gv + (int64_t)(c + u * nt) * VEC);
      }
    }
    for (; c < nc; c += nt) {
      RowChunk<T, VEC> k;
      k.load(zv + (int64_t)c * VEC);
      float v[VEC];
      k.get(v);
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = grad(v[i]);
      k.put(v);
      k.store(gv + (int64_t)c * VEC);
    }
  } else {
    for (int64_t i = va + tid; i < vb; i += nt) store_f(dz, i, grad(load_f(z, i)));
  }
  for (int64_t i = lo + tid; i < va; i += nt) store_f(dz, i, grad(load_f(z, i)));
  for (int64_t i = vb + tid; i < hi; i += nt) store_f(dz, i, grad(load_f(z, i)));
  if (bad) return leave();
  __syncthreads();  // the dense part is written
  if constexpr (MANY) {
    // The block's classes, a window at a time: the entries' masses are added up in shared memory, in
    // units of 2^-62, as integers (any order gives the same sum; what a p below 2^-38 loses is less
    // than 2^-63), and a class that has some is written anew.  top classes / kWindow looks at an entry.
    extern __shared__ unsigned long long mass[];
    const bool whole = tsum == tsum;  // a NaN among the teacher's logits makes its row's entries NaN
    for (int c = tid; c < kWindow; c += nt) mass[c] = 0;
    for (int64_t w0 = lo; w0 < hi; w0 += kWindow) {
      const int64_t n = std::min<int64_t>(kWindow, hi - w0);
      __syncthreads();
      if (has_t)
        for (int64_t j = tid; j < a.top; j += nt) {
          const int64_t at_window = index[j] - w0;
          if (at_window < 0 || at_window >= n) continue;
          const float t = teacher[j];
          if (t == -INFINITY) continue;
          const float p = exp2f((t - tmax) * kt) / tsum;
          atomicAdd(mass + at_window, whole ? __float2ull_rn(p * 0x1p62f) : 1ull);
        }
      __syncthreads();
      for (int c = tid; c < n; c += nt) {
        const bool own_label = has_l && w0 + c == label;
        const unsigned long long sum = mass[c];
        if (sum == 0 && !own_label) continue;
        mass[c] = 0;
        float g = grad(load_f(z, w0 + c)) - ct * (whole || sum == 0 ? __ull2float_rn(sum) * 0x1p-62f : NAN);
        if (own_label) g -= c1s;
        store_f(dz, w0 + c, g);
      }
    }
    return leave();
  }
  // An entry named twice gets both masses: each of its threads adds them in the same order
  // and writes the same value.
  auto corrected = [&](int64_t ix) {
    float p = 0.f;
    if (has_t)
      for (int64_t j = 0; j < a.top; ++j)
        if (index[j] == ix && teacher[j] != -INFINITY)
          p += exp2f((teacher[j] - tmax) * kt) / tsum;
    float g = grad(load_f(z, ix)) - ct * p;
    if (has_l && ix == label) g -= c1s;
    store_f(dz, ix, g);
  };
  if (has_t)
    for (int64_t j = tid; j < a.top; j += nt)
      if (index[j] >= lo && index[j] < hi) corrected(index[j]);
  if (has_l && label >= lo && label < hi && tid == nt - 1) corrected(label);
  leave();
}

// ---------------------------------------------------------------- loss and gradient, row on chip
// First, a warp a row, the teacher's side: the softmax p of the entries, an index named twice
// merged into its first place, the sums that the loss needs, and how many rows count.
constexpr int kPrepareThreads = 256;
constexpr int kHasTeacher = 1, kHasLabel = 2, kBad = 4;

struct Entry {
  int index;  // -1: nothing to do
  float p;
};
struct RowInfo {
  float plogp;  // sum p log p
  int flags;
};

// NQ: entries of a lane.
template <int NQ>
__global__ void __launch_bounds__(kPrepareThreads)
distill_prepare_kernel(const DistillArgs a, Entry *entries, RowInfo *info, int *counts,
                       unsigned *done) {
  __shared__ int warp_counts[kPrepareThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, top = (int)a.top;
  const float kt = kLog2e / a.tau;
  const bool use_kl = a.alpha != 0.f, use_ce = a.labels != nullptr && a.alpha != 1.f;
  if (blockIdx.x == 0 && threadIdx.x == 0) *done = 0;
  int counted = 0;
  for (int64_t row = (int64_t)blockIdx.x * (kPrepareThreads / 32) + warp; row < a.rows;
       row += (int64_t)gridDim.x * (kPrepareThreads / 32)) {
    const int64_t label = a.labels ? a.labels[row] : -1;
    int index[NQ];
    float t[NQ];
    int flags = 0;
    float m = kLowest;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      index[q] = -1, t[q] = 0.f;
      if (q * 32 + lane >= top) continue;
      const int64_t ix = a.index[row * a.top + q * 32 + lane];
      t[q] = a.teacher[row * a.top + q * 32 + lane];
      if (ix < 0 || t[q] == -INFINITY) continue;
      flags |= kHasTeacher;
      if (ix >= a.classes) {
        flags |= kBad;
        continue;
      }
      index[q] = (int)ix;
      m = fmaxf(m, t[q]);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
      flags |= __shfl_xor_sync(0xFFFFFFFFu, flags, o);
    }
    if (label >= 0) flags |= kHasLabel;
    counted += flags != 0;
    if (!use_kl) flags &= ~(kHasTeacher | kBad);
    if (!use_ce) flags &= ~kHasLabel;
    if (use_ce && label >= a.classes) flags |= kBad;
    float w[NQ], s = 0.f;
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      w[q] = index[q] < 0 ? 0.f : exp2f((t[q] - m) * kt);
      s += w[q];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    const float log_s = logf(s);
    float plogp = 0.f, merged[NQ];
    bool later[NQ];
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      w[q] = index[q] < 0 ? 0.f : w[q] / s;
      if (w[q] != 0.f) plogp = fmaf(w[q], (t[q] - m) / a.tau - log_s, plogp);
      merged[q] = 0.f, later[q] = false;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) plogp += __shfl_xor_sync(0xFFFFFFFFu, plogp, o);
    float p_label = 0.f;
#pragma unroll
    for (int src = 0; src < NQ; ++src) {
      if (src * 32 >= top) break;
      const int named = min(32, top - src * 32);
      for (int l = 0; l < named; ++l) {
        const int ix = __shfl_sync(0xFFFFFFFFu, index[src], l);
        const float p = __shfl_sync(0xFFFFFFFFu, w[src], l);
        p_label += ix >= 0 && ix == label ? p : 0.f;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {  // places without an entry have p 0
          merged[q] += index[q] == ix ? p : 0.f;
          later[q] |= index[q] == ix && src * 32 + l < q * 32 + lane;
        }
      }
    }
    const bool teach = (flags & kHasTeacher) != 0, lab = (flags & kHasLabel) != 0;
    Entry *out = entries + row * (a.top + 1);
#pragma unroll
    for (int q = 0; q < NQ; ++q) {
      if (q * 32 + lane >= top) continue;
      // the label's place carries its own entry
      const bool dead = !teach || index[q] < 0 || later[q] || (lab && index[q] == label);
      out[q * 32 + lane] = Entry{dead ? -1 : index[q], merged[q]};
    }
    if (lane == 0) {
      const bool in = lab && label < a.classes;
      out[top] = Entry{in ? (int)label : -1, teach ? p_label : 0.f};
      info[row] = RowInfo{plogp, flags};
    }
  }
  if (lane == 0) warp_counts[warp] = counted;
  __syncthreads();
  if (threadIdx.x == 0) {
    int n = 0;
    for (int i = 0; i < kPrepareThreads / 32; ++i) n += warp_counts[i];
    counts[blockIdx.x] = n;
  }
}

// Then the row.  A persistent cluster of 1 to 8 blocks takes one at a time.  A thread holds up to
// NV chunks of 16 bytes of it and their exponentials in registers, both relative to the
// largest of its own elements, so that z is read once and each exponential is computed once:
//   dz = [at e^((m_t - m) / tau)] e^((z - m_t) / tau) + [a1 e^(m_t - m)] e^(z - m_t).
// The next row's part arrives in shared memory meanwhile (bulk copies).  The warps' maxima and sums
// are joined over the cluster: each warp stores its own into every block's shared memory (st.async,
// two sets in turn) and every block waits for all of them on an mbarrier of its own.  A cluster
// barrier in its place also waited for the block's gradient stores.
// An entry is handed to the thread that holds its element (a list a thread in shared memory),
// which writes the corrected value over its own store: no second barrier.
// 8192 rows of 32768 bf16 classes, two temperatures: 294 us with three blocks an SM of 128 threads, 64
// elements a thread (168 registers) and clusters of 4; 317 with four of 32 elements and clusters of
// 8; 315 with six of 64 threads; 341 with one of 256.  What bounds it is the time that a cluster's
// blocks wait for the slowest of them (0.4 instructions a clock and scheduler), at 0.57 of the measured
// HBM rate; the sweep-twice kernel takes 318 us.  Rows of up to 128 x 4 chunks take 4 chunks a thread
// and one block; more take as many blocks of 128 x 8 as hold them, any number up to 8 (2000 x 40000: 5
// blocks 101 us, 8 blocks 158, the other kernel 121).  Rows that 8 do not hold are the other kernel's:
// 2000 x 131000 take 344 us there and took 485 here with 512 threads of 4 chunks.
// Rows that start inside 16 bytes, with the launches around the kernel: 2000 x 40001 137 us (the other
// kernel 148), 2000 x 4097 53 (61), 2000 x 1001 43 (53); 5 to 9 % slower where the last block has
// little to hold (2000 x 32767 136 against 126, 2000 x 50257 186 against 170), which the choice between the
// two does not look at: wherever 8 blocks hold a row it takes this one.
constexpr int kResidentThreads = 128;
constexpr int kResidentParts = 8;

struct Listed {
  int index;
  float p, z;
};
struct HeldRow {
  RowStats stats;
  RowInfo info;
  float in_z;
  bool bad;
  int64_t row;
};

struct ResidentArgs {
  DistillArgs d;
  const Entry *entries;
  const RowInfo *info;
  unsigned *done;
  float *total;  // the reduced loss, or null
  int divide;    // by the count
};

// NT: the block's threads where they are known, else 0.
template <typename T, bool TWO, bool ALIGNED, int NV, int NT>
__global__ void __launch_bounds__(kResidentThreads, NV == 4 ? 4 : 3)
distill_resident_kernel(const ResidentArgs ra) {
  constexpr int VEC = vec_of<T>();
  const DistillArgs &a = ra.d;
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  __shared__ float4 stats[2][kResidentParts * kResidentThreads / 32];  // m, sum tau, sum 1
  // in block 0, of every warp's entries: sum of c (r - z), sum of c, r
  __shared__ float4 shares[2][kResidentParts * kResidentThreads / 32];
  __shared__ uint64_t joined[2], landed[2];
  extern __shared__ __align__(16) uint4 row_smem[];  // two parts of a row, in turn
  __shared__ int head[2][kResidentThreads];   // a thread's first entry, or -1
  __shared__ int next[2][kEntries + 1];
  __shared__ Listed mine[2][kEntries + 1];
  __shared__ HeldRow held_set[32];
  __shared__ double loss_sums[kResidentThreads / 32];
  __shared__ int last;
  const int tid = threadIdx.x, nt = NT ? NT : blockDim.x, lane = tid & 31, warp = tid >> 5, warps = nt >> 5;
  const float kt = kLog2e / a.tau, inv_tau = 1.f / a.tau;
  const T *zb = reinterpret_cast<const T *>(a.z);
  T *db = reinterpret_cast<T *>(a.dz);
  const int classes = (int)a.classes, slots = (int)a.top + 1;
  head[0][tid] = head[1][tid] = -1;
  if (tid < 2) {
    sm100::mbar_init(joined + tid, warps);
    sm100::mbar_init(landed + tid, 1);
  }
  sm100::fence_barrier_init();
  bool failed = false;  // a wait of this thread gave up: NaN from then on

  int count = 0;
  for (int i = lane; i < a.n_counts; i += 32) count += a.counts[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xFFFFFFFFu, count, o);
  float unit = ra.divide ? 1.f / (float)(count > 0 ? count : 1) : 1.f;
  if (a.upstream && !a.upstream_rows) unit *= a.upstream[0];

  // Chunk c of a row covers elements [c VEC - shift, (c + 1) VEC - shift): 16-byte aligned in z
  // (and in dz, which the launch requires); the row's first and last may be cut.
  const int chunk0 = part * nt * NV + tid;
  auto shift_of = [&](int64_t row) {
    return ALIGNED ? 0
                   : (int)((reinterpret_cast<uintptr_t>(zb + row * a.classes) & 15) / sizeof(T));
  };
  // Thread 0 asks for a row's part in whole chunks: a bulk copy's unit is 16 bytes.  A cut chunk brings
  // its neighbours' elements along, or, where those would lie before or after the tensor, stays away.
  auto starts_outside = [&](int64_t row, int shift) { return row * a.classes < shift; };
  auto ends_outside = [&](int64_t row, int shift) {
    const int over = (VEC - (classes + shift) % VEC) % VEC;
    return (a.rows - 1 - row) * a.classes < over;
  };
  auto fetch_row = [&](int64_t row, int buffer) {
    const int shift = shift_of(row);
    const int c0 = part * nt * NV + (part == 0 && starts_outside(row, shift));
    const int c1 = min(part * nt * NV + nt * NV,
                       (classes + shift + VEC - 1) / VEC - ends_outside(row, shift));
    if (c1 > c0) {
      sm100::mbar_arrive_expect_tx(landed + buffer, (uint32_t)(c1 - c0) * 16);
      sm100::bulk_load(sm100::smem_u32(row_smem + buffer * nt * NV + c0 - part * nt * NV),
                       zb + (row * a.classes + c0 * VEC - shift), (uint32_t)(c1 - c0) * 16,
                       landed + buffer);
    } else {
      sm100::mbar_arrive(landed + buffer);
    }
  };
  // A cut chunk, by the thread that holds it: -inf outside the row, and what stayed away.
  auto mend_chunk = [&](int64_t row, int buffer, int shift, int c, bool away) {
    const int at = c - part * nt * NV;
    if (at < 0 || at >= nt * NV || (at & (nt - 1)) != tid) return;
    T *slot = reinterpret_cast<T *>(row_smem + buffer * nt * NV + at);
#pragma unroll 1
    for (int i = 0; i < VEC; ++i) {
      const int e = c * VEC - shift + i;
      if (e < 0 || e >= classes)
        store_f(slot, i, -INFINITY);
      else if (away)
        slot[i] = zb[row * a.classes + e];
    }
    sm100::fence_proxy_async_smem();  // before the copy of a later row into this place
  };
  RowChunk<T, VEC> cur[NV];
  auto load_row = [&](int64_t row, int buffer, int shift, bool whole) {
    if (!ALIGNED && !whole) {
      if (shift) mend_chunk(row, buffer, shift, 0, starts_outside(row, shift));
      if ((classes + shift) % VEC)
        mend_chunk(row, buffer, shift, (classes + shift) / VEC, ends_outside(row, shift));
    }
    const uint4 *part_smem = row_smem + buffer * nt * NV + tid;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (whole || (chunk0 + j * nt) * VEC - shift < classes) {
        const uint4 u = part_smem[j * nt];
        memcpy(&cur[j].raw, &u, 16);
      } else {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[i] = -INFINITY;
        cur[j].put(v);
      }
    }
  };

  if (parts > 1)
    cluster.sync();  // every block of the cluster runs before one writes to it
  else
    __syncthreads();
  const int64_t first = blockIdx.x / parts, step = gridDim.x / parts;
  // Losses wait until warp 0 of the first block has 32 rows, one a lane: their logarithms, taken a
  // row at a time, made the other warps wait.
  int held_rows = 0;
  auto flush = [&]() {
    __syncwarp();
    if (a.loss && part == 0 && warp == 0 && lane < held_rows) {
      const HeldRow held = held_set[lane];
      const RowStats &s = held.stats;
      const float s_one = TWO ? s.s1 : s.st;
      float loss = 0.f;
      if (held.info.flags & kHasTeacher)
        loss = a.alpha * a.tau * a.tau * (held.info.plogp + logf(s.st));
      if (held.info.flags & kHasLabel) loss += (1.f - a.alpha) * logf(s_one);
      loss += held.in_z;
      // nothing left of the row: log q = -inf
      if (s.st == 0.f && (held.info.flags & (kHasTeacher | kHasLabel))) loss = INFINITY;
      a.loss[held.row] = held.bad ? NAN : loss;
    }
    __syncwarp();
    held_rows = 0;
  };
  if (tid == 0 && first < a.rows) fetch_row(first, 0);
  bool coming = true;  // the row was asked for; after a failure no more are, and those that were
                       // are waited for: no block leaves while a copy is on its way to it
  int set = 0;
  uint32_t phase = 0;
  for (int64_t row = first; row < a.rows; row += step, phase ^= set, set ^= 1) {
    T *dz = db + row * a.classes;
    const Entry *entries = ra.entries + row * slots;
    Entry e = tid < slots ? entries[tid] : Entry{-1, 0.f};
    const RowInfo info = ra.info[row];
    const bool wanted = coming;
    coming = !failed && row + step < a.rows;
    if (tid == 0 && coming) fetch_row(row + step, set ^ 1);
    if (wanted && !sm100::mbar_wait_bounded(landed + set, phase, 1000000u)) failed = true;
    // Most parts lie inside their row: without a check a chunk their loads and stores are one
    // instruction each.
    const int shift = shift_of(row);
    const int lo = part * nt * NV * VEC - shift, hi = lo + nt * NV * VEC;
    const bool whole = lo >= 0 && hi <= classes;
    if (whole)
      load_row(row, set, shift, true);
    else
      load_row(row, set, shift, false);

    // ---- exponentials relative to the thread's largest element
    Pair et[NV][VEC / 2], e1[TWO ? NV : 1][VEC / 2];
    RowStats st{kLowest, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j) st.m = fmaxf(st.m, chunk_max(cur[j]));
    const float m_own = st.m;
    {
      const Pair minus = pair(-st.m, -st.m), k2 = pair(kt, kt), l2 = pair(kLog2e, kLog2e);
      Pair sum_t = pair(0.f, 0.f), sum_1 = sum_t;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float v[VEC];
        cur[j].get(v);
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          const Pair d = pair(v[2 * i], v[2 * i + 1]) + minus;
          et[j][i] = exp2_fast(d * k2);
          sum_t = sum_t + et[j][i];
          if (TWO) {
            e1[j][i] = exp2_fast(d * l2);
            sum_1 = sum_1 + e1[j][i];
          }
        }
      }
      float x, y;
      unpair(sum_t, x, y);
      st.st = x + y;
      unpair(sum_1, x, y);
      st.s1 = x + y;
    }

    // ---- entries of this block's classes, to the threads that hold them
    // With sum p = 1 the loss is alpha tau^2 (sum p log p + log S_tau) + (1 - alpha) log S_1
    // + sum c (m - z), c = alpha tau p of an entry and 1 - alpha of the label: the last sum from
    // here, against the largest z of the warp's entries first (masks of the type's lowest value
    // cancel exactly).
    float share_z = 0.f, share_c = 0.f, share_r = kLowest;
    const bool has_l = (info.flags & kHasLabel) != 0;
    for (int j = tid; j < slots; j += nt) {
      if (j != tid) e = entries[j];
      if (e.index >= 0 && e.index >= lo && e.index < hi) {
        const int at_part = e.index - lo, e0 = at_part / VEC * VEC + lo;  // its chunk's first
        const bool held_here = whole || (e0 >= 0 && e0 + VEC <= classes);
        const float zq =
            held_here ? load_f(reinterpret_cast<const T *>(row_smem + set * nt * NV), at_part)
                      : load_f(zb + row * a.classes, e.index);
        const float c =
            a.alpha * a.tau * e.p + (j == slots - 1 && has_l ? 1.f - a.alpha : 0.f);
        if (c != 0.f) {
          const float r = fmaxf(share_r, zq);
          if (share_c != 0.f) share_z = fmaf(share_c, r - share_r, share_z);
          share_z = fmaf(c, r - zq, share_z);
          share_c += c, share_r = r;
        }
        mine[set][j] = Listed{e.index, e.p, zq};
        next[set][j] = atomicExch(&head[set][(at_part / VEC) & (nt - 1)], j);
      }
    }

    // ---- sums joined over warps and blocks
    {
      const float m = warp_max(st.m);
      st.st *= exp2_fast((st.m - m) * kt);
      if (TWO) st.s1 *= exp2_fast((st.m - m) * kLog2e);
      st.m = m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        st.st += __shfl_xor_sync(0xFFFFFFFFu, st.st, o);
        if (TWO) st.s1 += __shfl_xor_sync(0xFFFFFFFFu, st.s1, o);
      }
      if (warp * 32 < slots) {
        const float r = warp_max(share_r);
        if (share_c != 0.f) share_z = fmaf(share_c, r - share_r, share_z);
        share_r = r;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          share_z += __shfl_xor_sync(0xFFFFFFFFu, share_z, o);
          share_c += __shfl_xor_sync(0xFFFFFFFFu, share_c, o);
        }
      }
      if (parts == 1) {
        if (lane == 0) {
          stats[set][warp] = make_float4(st.m, st.st, st.s1, 0.f);
          shares[set][warp] = make_float4(share_z, share_c, share_r, 0.f);
        }
        __syncthreads();
      } else {
        __syncwarp();  // the warp's entries are listed before its arrival
        if (lane < parts)
          sm100::store_async_rank(&stats[set][part * warps + warp], joined + set, lane, st.m,
                                  st.st, st.s1, 0.f);
        if (lane == 0) {
          sm100::store_async_rank(&shares[set][part * warps + warp], joined + set, 0, share_z,
                                  share_c, share_r, 0.f);
          if (warp == 0)
            sm100::mbar_arrive_expect_tx(
                joined + set, (uint32_t)(parts * warps *
                                         (part == 0 ? 2 : 1) * sizeof(float4)));
          else
            sm100::mbar_arrive(joined + set);
        }
        if (!failed) failed = !sm100::mbar_wait_bounded(joined + set, phase, 1000000u);
      }
    }
    {
      const int n = parts * warps;
      RowStats own{kLowest, 0.f, 0.f};
      if (lane < n) {
        const float4 b = stats[set][lane];
        own = RowStats{b.x, b.y, b.z};
      }
      for (int i = lane + 32; i < n; i += 32) {
        const float4 b = stats[set][i];
        stats_join<TWO>(own, RowStats{b.x, b.y, b.z}, kt);
      }
      const float m = warp_max(own.m);
      st.st = own.st * exp2_fast((own.m - m) * kt);
      if (TWO) st.s1 = own.s1 * exp2_fast((own.m - m) * kLog2e);
      st.m = m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        st.st += __shfl_xor_sync(0xFFFFFFFFu, st.st, o);
        if (TWO) st.s1 += __shfl_xor_sync(0xFFFFFFFFu, st.s1, o);
      }
    }
    float in_z = 0.f;
    if (a.loss && part == 0 && warp == 0) {
      for (int i = lane; i < parts * warps; i += 32) {
        const float4 b = shares[set][i];
        if (b.y != 0.f) in_z += fmaf(b.y, st.m - b.z, b.x);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) in_z += __shfl_xor_sync(0xFFFFFFFFu, in_z, o);
    }
    // a row that is -inf throughout: q = 0, log q = -inf
    const float s_one = TWO ? st.s1 : st.st;
    const float inv_t = st.st == 0.f ? 0.f : __fdividef(1.f, st.st);  // sums lie in [1, classes]
    const float inv_1 = s_one == 0.f ? 0.f : __fdividef(1.f, s_one);
    const bool has_t = (info.flags & kHasTeacher) != 0;
    const bool bad = (info.flags & kBad) != 0 || failed;
    if (tid == 0) held_set[held_rows] = HeldRow{st, info, in_z, bad, row};
    if (++held_rows == 32) flush();

    // ---- the gradient
    float scale = a.upstream_rows && a.upstream ? unit * a.upstream[row] : unit;
    if (bad) scale = NAN;
    const float ct = has_t || bad ? a.alpha * a.tau * scale : 0.f;
    const float c1 = has_l ? (1.f - a.alpha) * scale : 0.f;
    float at = ct * inv_t, a1 = c1 * inv_1;
    if (!TWO) at += a1;
    const float ft = at * exp2_fast((m_own - st.m) * kt);
    const float f1 = TWO ? a1 * exp2_fast((m_own - st.m) * kLog2e) : 0.f;
    const Pair ft2 = pair(ft, ft), f12 = pair(f1, f1);
    auto store_row = [&](bool whole_part) {
      T *dpart = dz + chunk0 * VEC - shift;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        float v[VEC];
#pragma unroll
        for (int i = 0; i < VEC / 2; ++i) {
          Pair g = ft2 * et[j][i];
          if (TWO) g = fma(f12, e1[j][i], g);
          unpair(g, v[2 * i], v[2 * i + 1]);
        }
        const int e0 = (chunk0 + j * nt) * VEC - shift;
        if (whole_part || (e0 >= 0 && e0 + VEC <= classes)) {
          RowChunk<T, VEC> k;
          k.put(v);
          k.store(dpart + j * nt * VEC);
        } else if (!ALIGNED && e0 < classes) {
#pragma unroll
          for (int i = 0; i < VEC; ++i)
            if (e0 + i >= 0 && e0 + i < classes) store_f(dz, e0 + i, v[i]);
        }
      }
    };
    if (info.flags == 0 && !bad) {  // no target: 0 whatever the logits are
      for (int64_t i = max(lo, 0) + tid; i < min(hi, classes); i += nt) store_f(dz, i, 0.f);
    } else if (whole) {
      store_row(true);
    } else {
      store_row(false);
    }
    int j = head[set][tid];
    if (j >= 0) {
      head[set][tid] = -1;
      if (!bad)
        for (; j >= 0; j = next[set][j]) {
          const Listed own = mine[set][j];
          const float d = own.z - st.m;
          float g = at * exp2_fast(d * kt);
          if (TWO) g = fmaf(a1, exp2_fast(d * kLog2e), g);
          g -= ct * own.p;
          if (j == slots - 1) g -= c1;
          store_f(dz, own.index, g);
        }
    }
  }

  flush();

  // ---- the last block to finish adds the rows' losses, in a fixed order
  if (ra.total) {
    if (part == 0 && warp == 0) __threadfence();
    __syncthreads();
    if (tid == 0) {
      __threadfence();
      last = atomicAdd(ra.done, 1u) == gridDim.x - 1;
    }
    __syncthreads();
    if (last) {
      __threadfence();
      double s = 0.0;
      for (int64_t i = tid; i < a.rows; i += nt) s += (double)__ldcg(a.loss + i);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
      if (lane == 0) loss_sums[warp] = s;
      __syncthreads();
      if (tid == 0) {
        for (int w = 1; w < warps; ++w) s += loss_sums[w];
        *ra.total = (float)(ra.divide ? s / (double)(count > 0 ? count : 1) : s);
      }
    }
  }
  if (parts > 1) cluster.sync();  // no block leaves while another writes its sums here
}

// How many rows count: those with an entry of the teacher or a label (a warp a row).
__global__ void __launch_bounds__(kCountThreads)
distill_count_kernel(const int64_t *index, const float *teacher, const int64_t *labels,
                     int64_t rows, int64_t top, int *counts) {
  __shared__ int warp_counts[kCountThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int n = 0;
  for (int64_t row = (int64_t)blockIdx.x * (kCountThreads / 32) + warp; row < rows;
       row += (int64_t)gridDim.x * (kCountThreads / 32)) {
    bool any = labels && labels[row] >= 0;
    for (int64_t j = lane; j < top && !any; j += 32)
      any = index[row * top + j] >= 0 && teacher[row * top + j] != -INFINITY;
    n += __any_sync(0xFFFFFFFFu, any) ? 1 : 0;
  }
  if (lane == 0) warp_counts[warp] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    n = 0;
    for (int w = 0; w < kCountThreads / 32; ++w) n += warp_counts[w];
    counts[blockIdx.x] = n;
  }
}

// loss = sum of the rows' losses / count, in a fixed order.
__global__ void __launch_bounds__(kSumThreads)
distill_sum_kernel(const float *row_loss, int64_t rows, const int *counts, int n_counts,
                   float *loss) {
  __shared__ double warp_sums[kSumThreads / 32];
  double s = 0.0;
  for (int64_t i = threadIdx.x; i < rows; i += kSumThreads) s += (double)row_loss[i];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
  if ((threadIdx.x & 31) == 0) warp_sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    s = 0.0;
    for (int w = 0; w < kSumThreads / 32; ++w) s += warp_sums[w];
    if (counts) {
      int n = 0;
      for (int i = 0; i < n_counts; ++i) n += counts[i];
      s /= (double)(n > 0 ? n : 1);
    }
    *loss = (float)s;
  }
}

// values *= scale[0], nothing where the scale is exactly 1.
template <typename T>
__global__ void __launch_bounds__(256) distill_scale_kernel(T *v, int64_t n, const float *scale) {
  const float s = *scale;
  if (s == 1.f) return;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < n;
       i += (int64_t)gridDim.x * blockDim.x)
    store_f(v, i, load_f(v, i) * s);
}

int check_distill(const char *what, const lnet_b200_distill_request *q) {
  if (!q) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: request must not be NULL", what);
  if (q->rows < 0 || q->classes < 1 || q->top < 0)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: rows %lld, classes %lld, top %lld", what,
                (long long)q->rows, (long long)q->classes, (long long)q->top);
  const int64_t wide = std::max(q->classes, q->top);
  if (wide > (int64_t)1 << 30 || q->rows > (int64_t)1 << 27 ||
      (q->rows > 0 && wide > ((int64_t)1 << 46) / q->rows))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: %lld x %lld logits are too many", what,
                (long long)q->rows, (long long)q->classes);
  if (q->dtype != LNET_F32 && q->dtype != LNET_BF16)
    return fail(LNET_ERR_UNSUPPORTED, "%s: logits must be fp32 or bf16", what);
  if (!(q->temperature > 0.f) || !(q->temperature < INFINITY))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: temperature must be positive and finite", what);
  if (!(q->alpha >= 0.f && q->alpha <= 1.f))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: alpha must lie in [0, 1]", what);
  if (q->reduction < 0 || q->reduction > 2)
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: reduction must be 0, 1 or 2", what);
  if (q->rows > 0 && (!q->logits || (q->top > 0 && (!q->teacher_indices || !q->teacher_logits))))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: logits, teacher_indices and teacher_logits must "
                "not be NULL", what);
  return LNET_OK;
}

int count_blocks(int64_t rows) {
  return (int)std::min<int64_t>(cdiv(rows, kCountThreads / 32), 1024);
}

struct DistillWork {
  int *counts;
  unsigned *done;
  float *row_loss;
  Entry *entries;
  RowInfo *info;
};

DistillWork distill_work(Arena &ar, const lnet_b200_distill_request *q) {
  DistillWork w{};
  const int64_t rows = std::max<int64_t>(q->rows, 1);
  w.counts = ar.take<int>(count_blocks(rows));
  w.done = ar.take<unsigned>(1);
  w.row_loss = ar.take<float>(q->reduction == 0 ? 0 : rows);
  if (q->top <= kEntries) {
    w.entries = ar.take<Entry>(rows * (q->top + 1));
    w.info = ar.take<RowInfo>(rows);
  }
  return w;
}

// Where the resident kernel serves a request: threads and blocks of a cluster.
struct ResidentPlan {
  int threads, parts, nv;
  bool aligned;
};

template <typename T>
bool resident_plan(const lnet_b200_distill_request *q, const void *dz, ResidentPlan &p) {
  constexpr int VEC = vec_of<T>();
  const uintptr_t zp = reinterpret_cast<uintptr_t>(q->logits), gp = reinterpret_cast<uintptr_t>(dz);
  if (!dz || ((zp ^ gp) & 15) || q->top > kEntries) return false;
  p.aligned = zp % 16 == 0 && q->classes % VEC == 0;
  // one chunk more where a row may start inside a chunk
  const int64_t chunks = cdiv(q->classes, VEC) + (p.aligned ? 0 : 1);
  // The smallest block that holds the row, 64 or 128 threads of 4 chunks; then 1 to 8 blocks of 128
  // threads of 8.  (A warp a row was slower for 56 and 366 classes.)
  p.threads = 64, p.parts = 1, p.nv = 4;
  auto holds = [&] { return chunks <= (int64_t)p.parts * p.threads * p.nv; };
  while (p.threads < kResidentThreads && !holds()) p.threads *= 2;
  if (!holds()) p.nv = 8;
  while (p.parts < kResidentParts && !holds()) ++p.parts;
  return holds();
}

template <typename T, bool TWO, bool ALIGNED, int NV, int NT>
int launch_resident_typed(const ResidentPlan &p, const ResidentArgs &a, cudaStream_t s) {
  constexpr auto kernel = &distill_resident_kernel<T, TWO, ALIGNED, NV, NT>;
  LNET_TRY(raise_shared_memory<kernel>(2 * kResidentThreads * NV * 16, "distill_resident_kernel"));
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = p.parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cfg.blockDim = dim3(p.threads);
  cfg.gridDim = dim3(p.parts);
  cfg.dynamicSmemBytes = 2 * p.threads * NV * 16;
  // Clusters that run at once: fewer than SMs / parts, since a cluster stays inside one group of
  // SMs.  A waiting cluster would double the time of a persistent grid.
  static std::atomic<int> known[kResidentParts + 1][kResidentThreads / 32 + 1];
  std::atomic<int> &cached = known[p.parts][p.threads / 32];
  int clusters = cached.load();
  if (clusters == 0) {
    if (p.parts == 1) {
      LNET_TRY(cuda_check(cudaOccupancyMaxActiveBlocksPerMultiprocessor(
                              &clusters, kernel, p.threads, cfg.dynamicSmemBytes),
                          "distill_resident_kernel occupancy"));
      clusters *= sm_count();
    } else {
      LNET_TRY(cuda_check(cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg),
                          "distill_resident_kernel occupancy"));
    }
    clusters = std::max(1, clusters);
    cached.store(clusters);
  }
  clusters = (int)std::max<int64_t>(1, std::min<int64_t>(a.d.rows, clusters));
  cfg.gridDim = dim3((unsigned)(clusters * p.parts));
  LNET_TRY(cuda_check(cudaLaunchKernelEx(&cfg, kernel, a), "distill_resident_kernel"));
  return after_launch("distill_resident_kernel");
}

bool two_temperatures(const DistillArgs &a) {
  return a.alpha != 0.f && a.labels && a.alpha != 1.f && a.tau != 1.f;
}

int launch_prepare(const DistillArgs &a, const DistillWork &w, int blocks, cudaStream_t s) {
  if (a.top <= 32)
    distill_prepare_kernel<1><<<blocks, kPrepareThreads, 0, s>>>(a, w.entries, w.info, w.counts,
                                                                    w.done);
  else if (a.top <= 64)
    distill_prepare_kernel<2><<<blocks, kPrepareThreads, 0, s>>>(a, w.entries, w.info, w.counts,
                                                                    w.done);
  else
    distill_prepare_kernel<kEntries / 32><<<blocks, kPrepareThreads, 0, s>>>(
        a, w.entries, w.info, w.counts, w.done);
  return after_launch("distill_prepare_kernel");
}

template <typename T>
int launch_resident(const ResidentPlan &p, const ResidentArgs &a, cudaStream_t s) {
  auto sized = [&](auto two, auto aligned) {
    constexpr bool TWO = decltype(two)::value, ALIGNED = decltype(aligned)::value;
    return p.nv == 4 ? launch_resident_typed<T, TWO, ALIGNED, 4, 0>(p, a, s)
                     : launch_resident_typed<T, TWO, ALIGNED, 8, kResidentThreads>(p, a, s);
  };
  if (two_temperatures(a.d))
    return p.aligned ? sized(std::true_type{}, std::true_type{})
                     : sized(std::true_type{}, std::false_type{});
  return p.aligned ? sized(std::false_type{}, std::true_type{})
                   : sized(std::false_type{}, std::false_type{});
}

template <typename T>
int launch_rows(const lnet_b200_distill_request *q, const DistillArgs &a, cudaStream_t s) {
  // Threads: 4 chunks of 16 bytes each, 64 or more; at most 512 for a row an SM, 256 from there on, 128
  // from 4 rows an SM on, where blocks of other rows fill the waits.  512, 256, 128 and 64 at most, loss
  // alone, fp32: 6263 x 12029 227, 95, 70, 86 us; 2000 x 32768 92, 60, 53, 63; 300 x 100003 47, 33, 47,
  // 77; bf16: 6263 x 12029 116, 82, 64, 79; 600 x 32768 25, 23, 23, 27; 300 x 100003 35, 34, 37, 49.
  const int64_t chunks = cdiv(q->classes, vec_of<T>());
  const int most = q->rows >= 4 * sm_count() ? 128 : q->rows >= sm_count() ? 256 : 512;
  const int threads = (int)std::min<int64_t>(most, std::max<int64_t>(64, cdiv(chunks, 4 * 32) * 32));
  // A cluster where rows alone leave SMs idle and each block keeps 4 chunks a thread (bf16 classes,
  // 4 chunks against 2: 1 x 4096 3.9 us against 4.8, 36 x 100003 10.7 against 13.7,
  // 74 x 32768 6.9 against 10.9; 5 x 100003, the other way, 7.9 against 7.2).
  int parts = 1;
  while (parts < 8 && q->rows * parts * 2 <= 2 * sm_count() && chunks / (parts * 2) >= 4 * threads)
    parts *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.stream = s;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  cfg.gridDim = dim3((unsigned)(q->rows * parts));
  cfg.blockDim = dim3(threads);
  const bool many = a.dz && a.top > kEntries, two = two_temperatures(a);
  if (many) cfg.dynamicSmemBytes = kWindow * sizeof(unsigned long long);
  const auto kernel = many ? (two ? distill_row_kernel<T, true, true> : distill_row_kernel<T, false, true>)
                           : (two ? distill_row_kernel<T, true, false> : distill_row_kernel<T, false, false>);
  const cudaError_t err = cudaLaunchKernelEx(&cfg, kernel, a);
  LNET_TRY(cuda_check(err, "distill_row_kernel"));
  return after_launch("distill_row_kernel");
}

int run_distill(const char *what, const lnet_b200_distill_request *q, void *workspace,
                size_t workspace_bytes, const float *upstream, float *loss, void *dz,
                cudaStream_t stream) {
  LNET_TRY(check_distill(what, q));
  reset_launches();
  Arena ar(workspace, workspace_bytes);
  const DistillWork w = distill_work(ar, q);
  const bool reduce = q->reduction != 0;
  if (!workspace || !ar.ok())
    return fail(LNET_ERR_WORKSPACE, "%s: needs %zu bytes of workspace, got %zu", what, ar.used,
                workspace ? workspace_bytes : 0);
  begin_entry(stream);
  if (q->rows == 0) {
    if (loss && reduce) LNET_TRY(cuda_check(cudaMemsetAsync(loss, 0, sizeof(float), stream), what));
    return LNET_OK;
  }
  // labels without weight still make their rows count
  const bool mean = q->reduction == 2;
  const int n_counts = count_blocks(q->rows);
  DistillArgs a{};
  a.z = q->logits;
  a.index = q->teacher_indices, a.teacher = q->teacher_logits, a.labels = q->labels;
  a.upstream = upstream, a.upstream_rows = reduce ? 0 : 1;
  a.loss = loss ? (reduce ? w.row_loss : loss) : nullptr;
  a.dz = dz;
  a.rows = q->rows, a.classes = q->classes, a.top = q->top;
  a.alpha = q->alpha;
  a.tau = a.alpha == 0.f ? 1.f : q->temperature;  // without the teacher only softmax(z) is needed
  const bool bf16 = q->dtype == LNET_BF16;
  ResidentPlan plan{};
  if (bf16 ? resident_plan<__nv_bfloat16>(q, dz, plan) : resident_plan<float>(q, dz, plan)) {
    LNET_TRY(launch_prepare(a, w, n_counts, stream));
    a.counts = w.counts, a.n_counts = n_counts;
    const ResidentArgs ra{a, w.entries, w.info, w.done, loss && reduce ? loss : nullptr, mean};
    return bf16 ? launch_resident<__nv_bfloat16>(plan, ra, stream)
                : launch_resident<float>(plan, ra, stream);
  }
  if (mean) {
    distill_count_kernel<<<n_counts, kCountThreads, 0, stream>>>(
        q->teacher_indices, q->teacher_logits, q->labels, q->rows, q->top, w.counts);
    LNET_TRY(after_launch("distill_count_kernel"));
    a.counts = w.counts, a.n_counts = n_counts;
  }
  LNET_TRY(bf16 ? launch_rows<__nv_bfloat16>(q, a, stream) : launch_rows<float>(q, a, stream));
  if (loss && reduce) {
    distill_sum_kernel<<<1, kSumThreads, 0, stream>>>(w.row_loss, q->rows, a.counts, a.n_counts,
                                                      loss);
    LNET_TRY(after_launch("distill_sum_kernel"));
  }
  return LNET_OK;
}

}  // namespace
}  // namespace lnet

using namespace lnet;

extern "C" int lnet_b200_distill_workspace_size(const lnet_b200_distill_request *req,
                                                size_t *bytes) {
  const char *what = "distill_workspace_size";
  LNET_TRY(check_distill(what, req));
  if (!bytes) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: bytes must not be NULL", what);
  Arena ar(nullptr, 0);
  distill_work(ar, req);
  *bytes = ar.used;
  return LNET_OK;
}

extern "C" int lnet_b200_distill_forward(const lnet_b200_distill_request *req, void *workspace,
                                         size_t workspace_bytes, float *loss, void *dlogits,
                                         lnet_stream_t stream) {
  const char *what = "distill_forward";
  if (!loss) return fail(LNET_ERR_INVALID_ARGUMENT, "%s: loss must not be NULL", what);
  return run_distill(what, req, workspace, workspace_bytes, nullptr, loss, dlogits, stream);
}

extern "C" int lnet_b200_distill_backward(const lnet_b200_distill_request *req, void *workspace,
                                          size_t workspace_bytes, const float *dloss,
                                          void *dlogits, lnet_stream_t stream) {
  const char *what = "distill_backward";
  LNET_TRY(check_distill(what, req));
  if (req->rows > 0 && (!dloss || !dlogits))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: dloss and dlogits must not be NULL", what);
  return run_distill(what, req, workspace, workspace_bytes, dloss, nullptr, dlogits, stream);
}

extern "C" int lnet_b200_distill_scale(void *dlogits, int32_t dtype, int64_t count,
                                       const float *scale, lnet_stream_t stream) {
  const char *what = "distill_scale";
  if (count < 0 || (count > 0 && (!dlogits || !scale)))
    return fail(LNET_ERR_INVALID_ARGUMENT, "%s: count %lld, or a NULL pointer", what,
                (long long)count);
  if (dtype != LNET_F32 && dtype != LNET_BF16)
    return fail(LNET_ERR_UNSUPPORTED, "%s: dlogits must be fp32 or bf16", what);
  reset_launches();
  if (count == 0) return LNET_OK;
  begin_entry(stream);
  const int blocks = (int)std::min<int64_t>(cdiv(count, 2048), (int64_t)sm_count() * 8);
  if (dtype == LNET_BF16)
    distill_scale_kernel<<<blocks, 256, 0, stream>>>(reinterpret_cast<__nv_bfloat16 *>(dlogits),
                                                     count, scale);
  else
    distill_scale_kernel<<<blocks, 256, 0, stream>>>(reinterpret_cast<float *>(dlogits), count,
                                                     scale);
  return after_launch("distill_scale_kernel");
}

// Distillation from a teacher's top logits, mixed with hard labels.
//
// Row i: entries j with index >= 0 and a teacher logit above -inf,
//   p_j = softmax(t_j / tau) over them,   q = softmax(z / tau) over all classes,
//   KL = sum_j p_j (log p_j - log q_j),   CE = logsumexp(z) - z[label],
//   loss = alpha tau^2 KL [entries] + (1 - alpha) CE [label >= 0],
//   dz = alpha tau (q - p) [entries] + (1 - alpha) (softmax(z) - onehot) [label >= 0].
// A part with weight 0 is left out.  A class at -inf has q = 0 (the loss is +inf
// where the teacher gives it mass); a row that is -inf throughout has q = 0
// everywhere.  An index or label past the classes makes the row's loss NaN and
// touches nothing else.
//
// One sweep reads the row for its running maximum and exponential sums (one sum
// for each of the temperatures tau and 1 that the loss needs), a second one
// writes the gradient from the row in L2 or L1; the few entries of the teacher
// and the label are then corrected in place, each from z again, so that every
// value is rounded once.  A row belongs to a block, or, where there are few
// rows, to a cluster of up to 8 blocks that join their sums through distributed
// shared memory.
#include <cooperative_groups.h>

#include <algorithm>

#include "rows.cuh"

namespace cg = cooperative_groups;

namespace lnet {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLowest = -3.402823466e+38f;
constexpr int kCountThreads = 256;
constexpr int kSumThreads = 1024;

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

// ex2.approx (2 ulp), results below 2^-126 flushed to zero
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
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

template <typename T, bool TWO>
__global__ void distill_row_kernel(const DistillArgs a) {
  constexpr int VEC = vec_of<T>();
  constexpr int U = 4;  // chunks in flight a thread
  cg::cluster_group cluster = cg::this_cluster();
  const int parts = (int)cluster.num_blocks(), part = (int)cluster.block_rank();
  __shared__ RowStats warp_stats[32];
  __shared__ RowStats block_stats;
  __shared__ float scratch[33];
  const int tid = threadIdx.x, nt = blockDim.x;
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
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    RowStats b;
    b.m = __shfl_xor_sync(0xFFFFFFFFu, st.m, o);
    b.st = __shfl_xor_sync(0xFFFFFFFFu, st.st, o);
    b.s1 = TWO ? __shfl_xor_sync(0xFFFFFFFFu, st.s1, o) : 0.f;
    stats_join<TWO>(st, b, kt);
  }
  if ((tid & 31) == 0) warp_stats[tid >> 5] = st;
  __syncthreads();
  st = warp_stats[0];
  for (int w = 1; w < nt / 32; ++w) stats_join<TWO>(st, warp_stats[w], kt);
  if (parts > 1) {
    if (tid == 0) block_stats = st;
    cluster.sync();
    st = *cluster.map_shared_rank(&block_stats, 0);
    for (int p = 1; p < parts; ++p)
      stats_join<TWO>(st, *cluster.map_shared_rank(&block_stats, p), kt);
    cluster.sync();  // no block leaves while another reads its sums
  }
  // a row that is -inf throughout: q = 0, log q = -inf
  const float inv_t = st.st == 0.f ? 0.f : 1.f / st.st;
  const float s_one = TWO ? st.s1 : st.st;  // one temperature: tau = 1, or no label part
  const float inv_1 = s_one == 0.f ? 0.f : 1.f / s_one;

  // ---- the teacher's softmax (every block of a cluster for itself)
  float tmax = kLowest, tsum = 0.f;
  bool has_t = false, bad = false;
  if (use_kl) {
    float m = kLowest;
    int any = 0, out = 0;
    for (int64_t j = tid; j < a.top; j += nt) {
      const int64_t ix = index[j];
      const float t = teacher[j];
      if (ix < 0 || t == -INFINITY) continue;
      any = 1;
      out |= ix >= a.classes;
      m = fmaxf(m, t);
    }
    has_t = __syncthreads_or(any) != 0;
    bad = __syncthreads_or(out) != 0;
    // the largest, by way of order-preserving warp shuffles
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xFFFFFFFFu, m, o));
    if ((tid & 31) == 0) scratch[tid >> 5] = m;
    __syncthreads();
    tmax = scratch[0];
    for (int w = 1; w < nt / 32; ++w) tmax = fmaxf(tmax, scratch[w]);
    float s = 0.f;
    for (int64_t j = tid; j < a.top; j += nt)
      if (index[j] >= 0 && teacher[j] != -INFINITY) s += exp2f((teacher[j] - tmax) * kt);
    tsum = group_reduce<0, SumOp>(s, scratch);
  }
  const int64_t label = use_ce ? a.labels[row] : -1;
  const bool has_l = label >= 0;
  bad |= label >= a.classes;
  const float log_st = logf(st.st), log_tsum = logf(tsum);

  // ---- the loss
  if (a.loss && part == 0) {
    float kl = 0.f;
    if (has_t && !bad) {
      for (int64_t j = tid; j < a.top; j += nt) {
        const int64_t ix = index[j];
        if (ix < 0 || teacher[j] == -INFINITY) continue;
        const float lt = (teacher[j] - tmax) / a.tau;
        const float p = exp2f((teacher[j] - tmax) * kt) / tsum;
        const float zq = load_f(z, ix);
        const float lq = zq == -INFINITY ? -INFINITY : (zq - st.m) / a.tau - log_st;
        if (p != 0.f) kl += p * ((lt - log_tsum) - lq);
      }
    }
    kl = group_reduce<0, SumOp>(kl, scratch);
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
  if (!a.dz) return;

  // ---- the gradient: at * e^((z - m) / tau) + a1 * e^(z - m), then the entries
  float scale = 1.f;
  if (a.counts) {
    int n = 0;
    for (int i = 0; i < a.n_counts; ++i) n += a.counts[i];
    scale = 1.f / (float)(n > 0 ? n : 1);
  }
  if (a.upstream) scale *= a.upstream[a.upstream_rows ? row : 0];
  if (bad) scale = NAN;
  const float ct = has_t ? a.alpha * a.tau * scale : 0.f;
  const float c1s = has_l ? (1.f - a.alpha) * scale : 0.f;
  float at = ct * inv_t, a1 = c1s * inv_1;
  if (!TWO) {
    at += a1;
    a1 = 0.f;
  }
  const float m = st.m;
  auto grad = [&](float v) {
    float g = at * exp2_fast((v - m) * kt);
    if (TWO) g = fmaf(a1, exp2_fast((v - m) * kLog2e), g);
    return g;
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
  if (bad) return;
  __syncthreads();  // the dense part is written
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
}

// How many rows count: those with an entry of the teacher or a label (a warp a row).
__global__ void __launch_bounds__(kCountThreads)
distill_count_kernel(const int64_t *index, const float *teacher, const int64_t *labels,
                     int64_t rows, int64_t top, int use_kl, int *counts) {
  __shared__ int warp_counts[kCountThreads / 32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int n = 0;
  for (int64_t row = (int64_t)blockIdx.x * (kCountThreads / 32) + warp; row < rows;
       row += (int64_t)gridDim.x * (kCountThreads / 32)) {
    bool any = labels && labels[row] >= 0;
    if (use_kl)
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
  return (int)std::min<int64_t>(cdiv(rows, kCountThreads / 32), 128);
}

struct DistillWork {
  int *counts;
  float *row_loss;
};

DistillWork distill_work(Arena &ar, const lnet_b200_distill_request *q) {
  DistillWork w{};
  w.counts = ar.take<int>(count_blocks(std::max<int64_t>(q->rows, 1)));
  w.row_loss = ar.take<float>(q->reduction == 0 ? 0 : q->rows);
  return w;
}

template <typename T>
int launch_rows(const lnet_b200_distill_request *q, const DistillArgs &a, cudaStream_t s) {
  const bool two = a.alpha != 0.f && a.labels && a.alpha != 1.f && a.tau != 1.f;
  // Threads: 4 chunks of 16 bytes each, 64 to 512.
  const int64_t chunks = cdiv(q->classes, vec_of<T>());
  const int threads = (int)std::min<int64_t>(512, std::max<int64_t>(64, cdiv(chunks, 4 * 32) * 32));
  // A cluster where rows alone leave SMs idle and each block keeps 4 chunks a thread.
  int parts = 1;
  while (parts < 8 && q->rows * parts * 2 <= 2 * sm_count() && chunks / (parts * 2) >= 4 * threads)
    parts *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(q->rows * parts));
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  const cudaError_t err = two ? cudaLaunchKernelEx(&cfg, distill_row_kernel<T, true>, a)
                              : cudaLaunchKernelEx(&cfg, distill_row_kernel<T, false>, a);
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
  const int n_counts = mean ? count_blocks(q->rows) : 0;
  if (mean) {
    distill_count_kernel<<<n_counts, kCountThreads, 0, stream>>>(
        q->teacher_indices, q->teacher_logits, q->labels, q->rows, q->top, 1, w.counts);
    LNET_TRY(after_launch("distill_count_kernel"));
  }
  DistillArgs a{};
  a.z = q->logits;
  a.index = q->teacher_indices, a.teacher = q->teacher_logits, a.labels = q->labels;
  a.counts = mean ? w.counts : nullptr, a.n_counts = n_counts;
  a.upstream = upstream, a.upstream_rows = reduce ? 0 : 1;
  a.loss = loss ? (reduce ? w.row_loss : loss) : nullptr;
  a.dz = dz;
  a.rows = q->rows, a.classes = q->classes, a.top = q->top;
  a.alpha = q->alpha;
  a.tau = a.alpha == 0.f ? 1.f : q->temperature;  // without the teacher only softmax(z) is needed
  LNET_TRY(q->dtype == LNET_BF16 ? launch_rows<__nv_bfloat16>(q, a, stream)
                                 : launch_rows<float>(q, a, stream));
  if (loss && reduce) {
    distill_sum_kernel<<<1, kSumThreads, 0, stream>>>(w.row_loss, q->rows, a.counts, n_counts,
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

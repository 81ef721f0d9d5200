// Host path of the feed-forward and distillation operators: a CPython module
// that takes torch tensors, allocates the outputs, calls the C ABI
// (include/lnet_b200.h) on torch's current stream and records the gradient.
//
// Small calls spend their time here and not on the GPU: through
// torch.autograd.Function and ctypes a training call of a few rows took 120 us,
// of which the kernels were 15.  Arguments are checked by the Python callers
// (lnet_b200.norm, linear, distill); this file has no checks of its own beyond
// the C ABI's, but refuses what would pass it by in silence: a forward-mode
// derivative, which would come out as 0, and a trace, which would record the
// outputs' allocation and not the launch.
#define PY_SSIZE_T_CLEAN
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <optional>
#include <string>

#include "lnet_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

// The library that lnet_b200._lib loaded: its entry points, by name, from Python.
#define LNET_ENTRIES(X)                                                                          \
  X(last_error)                                                                                  \
  X(residual_rms_norm)                                                                           \
  X(residual_rms_norm_fp8)                                                                       \
  X(residual_rms_norm_workspace_size)                                                            \
  X(residual_rms_norm_backward)                                                                  \
  X(quantize_rows_fp8)                                                                           \
  X(linear_pack)                                                                                 \
  X(linear_workspace_size)                                                                       \
  X(linear_forward)                                                                              \
  X(linear_backward_workspace_size)                                                              \
  X(linear_backward)                                                                             \
  X(distill_workspace_size)                                                                      \
  X(distill_forward)                                                                             \
  X(distill_backward)                                                                            \
  X(distill_scale)
struct Entries {
#define X(name) decltype(&lnet_b200_##name) name = nullptr;
  LNET_ENTRIES(X)
#undef X
} lib;

void check(int status, const char *what) {
  if (status == LNET_OK) return;
  const std::string msg = std::string("lnet_b200_") + what + ": " + lib.last_error();
  if (status == LNET_ERR_INVALID_ARGUMENT) TORCH_CHECK_VALUE(false, msg);
  if (status == LNET_ERR_UNSUPPORTED) TORCH_CHECK_TYPE(false, msg);
  TORCH_CHECK(false, msg);
}

int dtype_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kBFloat16: return LNET_BF16;
    case at::kFloat: return LNET_F32;
    case at::kFloat8_e4m3fn: return LNET_E4M3;
    default: TORCH_CHECK_TYPE(false, "unexpected dtype ", t.scalar_type());
  }
}
lnet_stream_t stream_of(const Tensor &t) {
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}
// Null where there is no tensor, and only there: a wrapper without memory of its own (fake, functional,
// distributed) would read as an argument that was left out.
void *ptr(const Tensor &t) {
  if (!t.defined()) return nullptr;
  void *p = t.data_ptr();
  TORCH_CHECK(p || t.numel() == 0, "a tensor without memory of its own (a fake, functional or "
                                   "distributed wrapper) cannot be used here");
  return p;
}
Tensor dense(const Tensor &t) { return t.defined() ? t.contiguous() : t; }
Tensor dense(const OptTensor &t) { return t.has_value() ? dense(*t) : Tensor(); }
Tensor workspace(size_t bytes, const Tensor &like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}
int64_t rows_of(const Tensor &t) { return t.size(-1) ? t.numel() / t.size(-1) : 0; }
bool tracked(std::initializer_list<const Tensor *> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor *t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
void refuse(const char *what, std::initializer_list<const Tensor *> ts) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what,
              " cannot be traced: use the torch.ops.lnet_b200 operator");
  for (const Tensor *t : ts)
    TORCH_CHECK(!t->defined() || !t->_fw_grad(0).defined(), what,
                " has no forward-mode derivative");
}
// A backward pass run with create_graph: its results raise where they are differentiated.
variable_list once(variable_list grads, const char *what) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list some;
  for (auto &g : grads)
    if (g.defined()) some.push_back(g.detach().requires_grad_(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(
      std::string(what) + " can be differentiated once only", (int)some.size());
  some = (*node)(std::move(some));
  size_t k = 0;
  for (auto &g : grads)
    if (g.defined()) g = some[k++];
  return grads;
}

// ---------------------------------------------------------------- norm
struct NormOut {
  Tensor y, stream, rstd;
};
NormOut norm_forward(const Tensor &x, const Tensor &w, const Tensor &r, double eps, bool keep) {
  NormOut o;
  o.y = at::empty_like(x);
  if (r.defined()) o.stream = at::empty_like(x);
  if (keep) o.rstd = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
  check(lib.residual_rms_norm(ptr(x), ptr(r), ptr(w), dtype_of(x), dtype_of(w), rows_of(x),
                              x.size(-1), (float)eps, ptr(o.y), ptr(o.stream), (float *)ptr(o.rstd),
                              stream_of(x)),
        "residual_rms_norm");
  return o;
}
std::pair<Tensor, Tensor> norm_backward(const Tensor &stream, const Tensor &rstd, const Tensor &w,
                                        const Tensor &dy, const Tensor &dstream, bool want_w) {
  Tensor dx = at::empty_like(stream), dw, ws;
  size_t bytes = 0;
  if (want_w) {
    dw = at::empty_like(w);
    check(lib.residual_rms_norm_workspace_size(dtype_of(stream), rows_of(stream), stream.size(-1),
                                               &bytes),
          "residual_rms_norm_workspace_size");
    ws = workspace(bytes, stream);
  }
  check(lib.residual_rms_norm_backward(ptr(stream), (const float *)ptr(rstd), ptr(w), ptr(dy),
                                       ptr(dstream), dtype_of(stream), dtype_of(w),
                                       rows_of(stream), stream.size(-1), ptr(dx), ptr(dw), ptr(ws),
                                       bytes, stream_of(stream)),
        "residual_rms_norm_backward");
  return {dx, dw};
}

struct NormFunction : torch::autograd::Function<NormFunction> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &w,
                               const OptTensor &r, double eps) {
    ctx->saved_data["need"] = (int64_t)((x.requires_grad() ? 1 : 0) | (w.requires_grad() ? 2 : 0) |
                                        (r.has_value() && r->requires_grad() ? 4 : 0));
    const Tensor xc = dense(x), wc = dense(w);
    NormOut o = norm_forward(xc, wc, dense(r), eps, true);
    ctx->save_for_backward({r.has_value() ? o.stream : xc, wc, o.rstd});
    ctx->set_materialize_grads(false);
    // without a residual the stream is x itself
    return {o.y, r.has_value() ? o.stream : x};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const int64_t need = ctx->saved_data["need"].toInt();
    const auto saved = ctx->get_saved_variables();
    const Tensor &dy = grads[0], dstream = grads[1];
    refuse("residual_rms_norm's gradient", {&dy, &dstream});
    Tensor dx, dw;
    if (!dy.defined()) {
      dx = dstream;
      if (need & 2) dw = at::zeros_like(saved[1]);
    } else {
      c10::cuda::CUDAGuard guard(saved[0].device());
      std::tie(dx, dw) =
          norm_backward(saved[0], saved[2], saved[1], dense(dy), dense(dstream), (need & 2) != 0);
    }
    return once({need & 1 ? dx : Tensor(), dw, need & 4 ? dx : Tensor(), Tensor()},
                "residual_rms_norm");
  }
};

// ---------------------------------------------------------------- linear
// A product's operand as [rows, K] with unit column stride.  Where the product runs on tiles (more
// rows than kFewRows) its rows start on 16-byte boundaries: as they lie, or in a padded copy, made
// once for the forward and the backward pass.
constexpr int64_t kFewRows = 8;
Tensor operand(const Tensor &t, bool tiles) {
  const int64_t k = t.size(-1), elem = (int64_t)t.element_size();
  Tensor m = t;
  if (t.dim() != 2 || t.stride(1) != 1 || (t.size(0) > 1 && t.stride(0) < k))
    m = t.contiguous().view({rows_of(t), k});
  const int64_t pitch = m.size(0) > 1 ? m.stride(0) : k;
  const bool aligned = (uintptr_t)ptr(m) % 16 == 0 && (m.size(0) <= 1 || pitch * elem % 16 == 0);
  if (!tiles || aligned || m.size(0) == 0) return m;
  const int64_t wide = (k * elem + 15) / 16 * 16 / elem;
  Tensor copy = at::empty({m.size(0), wide}, m.options());
  check(lib.linear_pack(ptr(m), dtype_of(m), m.size(0), k, pitch, ptr(copy), wide, stream_of(m)),
        "linear_pack");
  return copy.narrow(1, 0, k);
}
lnet_b200_linear_request linear_request(const Tensor &x, const Tensor &w, const Tensor &b,
                                        const Tensor &r, int64_t act, const Tensor &xs,
                                        const Tensor &ws) {
  lnet_b200_linear_request q{};
  q.rows = x.size(0), q.inner = x.size(1), q.outer = w.size(0);
  q.dtype = dtype_of(x), q.activation = (int32_t)act;
  q.x = ptr(x), q.weight = ptr(w), q.bias = ptr(b), q.residual = ptr(r);
  q.x_scale = (const float *)ptr(xs), q.weight_scale = (const float *)ptr(ws);
  // one row has no pitch; its bytes, up to the next 16, may not be there: no tile reads them
  q.x_pitch = q.rows > 1 ? x.stride(0) : 0, q.weight_pitch = q.outer > 1 ? w.stride(0) : 0;
  return q;
}
struct LinearOut {
  Tensor y, pre, x, w;  // x, w: the operands as they were used
};
LinearOut linear_forward(const Tensor &x, const Tensor &w, const Tensor &b, const Tensor &r,
                         int64_t act, const Tensor &xs, const Tensor &ws, bool keep) {
  const bool tiles = rows_of(x) > kFewRows;
  LinearOut o;
  o.x = operand(x, tiles), o.w = operand(w, tiles);
  const Tensor bc = dense(b), rc = dense(r), xsc = dense(xs), wsc = dense(ws);
  const auto q = linear_request(o.x, o.w, bc, rc, act, xsc, wsc);
  size_t bytes = 0;
  check(lib.linear_workspace_size(&q, &bytes), "linear_workspace_size");
  if (x.dim() == 2) {
    o.y = at::empty({q.rows, q.outer}, x.options().dtype(at::kBFloat16));
  } else {
    auto shape = x.sizes().vec();
    shape.back() = q.outer;
    o.y = at::empty(shape, x.options().dtype(at::kBFloat16));
  }
  if (keep) o.pre = at::empty_like(o.y);
  Tensor space = workspace(bytes, x);
  check(lib.linear_forward(&q, ptr(space), bytes, ptr(o.y), ptr(o.pre), stream_of(x)),
        "linear_forward");
  return o;
}
// x and w as linear_forward left them; dx in `x_sizes`.
variable_list linear_backward(const Tensor &x, const Tensor &w, int64_t act, const Tensor &pre,
                              const Tensor &dy, int64_t need, at::IntArrayRef x_sizes) {
  const auto q = linear_request(x, w, Tensor(), Tensor(), act, Tensor(), Tensor());
  size_t bytes = 0;
  check(lib.linear_backward_workspace_size(&q, ptr(pre), ptr(dy), need & 1, need & 2, need & 4,
                                           &bytes),
        "linear_backward_workspace_size");
  Tensor dx, dw, db, ws = workspace(bytes, x);
  if (need & 1) dx = at::empty(x_sizes, x.options());
  if (need & 2) dw = at::empty({q.outer, q.inner}, x.options());
  if (need & 4) db = at::empty({q.outer}, x.options());
  check(lib.linear_backward(&q, ptr(pre), ptr(dy), ptr(ws), bytes, ptr(dx), ptr(dw), ptr(db),
                            stream_of(x)),
        "linear_backward");
  return {dx, dw, db};
}

struct LinearFunction : torch::autograd::Function<LinearFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &w, const OptTensor &b,
                        const OptTensor &r, int64_t act) {
    const int64_t need = (x.requires_grad() ? 1 : 0) | (w.requires_grad() ? 2 : 0) |
                         (b.has_value() && b->requires_grad() ? 4 : 0) |
                         (r.has_value() && r->requires_grad() ? 8 : 0);
    LinearOut o = linear_forward(x, w, b.value_or(Tensor()), r.value_or(Tensor()), act, Tensor(),
                                 Tensor(), act != 0 && (need & 7));
    ctx->saved_data["need"] = need;
    ctx->saved_data["act"] = act;
    if (x.dim() != 2) ctx->saved_data["sizes"] = x.sizes().vec();
    ctx->save_for_backward({o.x, o.w, o.pre});
    return o.y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const int64_t need = ctx->saved_data["need"].toInt(), act = ctx->saved_data["act"].toInt();
    variable_list g(3);
    refuse("linear_act's gradient", {&grads[0]});
    if (need & 7) {
      const auto saved = ctx->get_saved_variables();
      c10::cuda::CUDAGuard guard(saved[0].device());
      const auto sizes = ctx->saved_data.find("sizes");
      const auto shape = sizes == ctx->saved_data.end() ? saved[0].sizes().vec()
                                                        : sizes->second.toIntVector();
      g = linear_backward(saved[0], saved[1], act, saved[2], dense(grads[0]), need, shape);
    }
    return once({g[0], g[1], g[2], need & 8 ? grads[0] : Tensor(), Tensor()}, "linear_act");
  }
};

// ---------------------------------------------------------------- distillation
struct DistillCall {
  lnet_b200_distill_request q{};
  Tensor ws;
  size_t bytes = 0;
  DistillCall(const Tensor &z, const Tensor &index, const Tensor &teacher, const Tensor &labels,
              double tau, double alpha, int64_t reduction) {
    q.rows = rows_of(z), q.classes = z.size(-1), q.top = index.size(-1);
    q.dtype = dtype_of(z), q.reduction = (int32_t)reduction;
    q.logits = ptr(z), q.teacher_indices = (const int64_t *)ptr(index);
    q.teacher_logits = (const float *)ptr(teacher), q.labels = (const int64_t *)ptr(labels);
    q.temperature = (float)tau, q.alpha = (float)alpha;
    check(lib.distill_workspace_size(&q, &bytes), "distill_workspace_size");
    ws = workspace(bytes, z);
  }
};
std::pair<Tensor, Tensor> distill_forward(const Tensor &z, const Tensor &index,
                                          const Tensor &teacher, const Tensor &labels, double tau,
                                          double alpha, int64_t reduction, bool want_grad) {
  DistillCall c(z, index, teacher, labels, tau, alpha, reduction);
  const auto shape = reduction == 0 ? z.sizes().slice(0, z.dim() - 1) : at::IntArrayRef();
  Tensor loss = at::empty(shape, z.options().dtype(at::kFloat)), dz;
  if (want_grad) dz = at::empty_like(z);
  check(lib.distill_forward(&c.q, ptr(c.ws), c.bytes, (float *)ptr(loss), ptr(dz), stream_of(z)),
        "distill_forward");
  return {loss, dz};
}
Tensor distill_backward(const Tensor &z, const Tensor &index, const Tensor &teacher,
                        const Tensor &labels, double tau, double alpha, int64_t reduction,
                        const Tensor &dloss) {
  DistillCall c(z, index, teacher, labels, tau, alpha, reduction);
  Tensor dz = at::empty_like(z);
  check(lib.distill_backward(&c.q, ptr(c.ws), c.bytes, (const float *)ptr(dloss), ptr(dz),
                             stream_of(z)),
        "distill_backward");
  return dz;
}

// A reduced loss takes its gradient in the forward pass, while the row is on chip; the backward
// pass scales it in place by the loss's gradient (a launch that reads one value where that is 1;
// for another value a bf16 gradient is rounded twice, half a unit in the last place each time).
// The rows' losses (no reduction), and a second backward pass, take it from the logits again.
struct DistillFunction : torch::autograd::Function<DistillFunction> {
  static Tensor forward(AutogradContext *ctx, const Tensor &logits, const Tensor &indices,
                        const Tensor &teacher_logits, const OptTensor &label_opt, double tau,
                        double alpha, int64_t reduction) {
    const Tensor z = dense(logits), index = dense(indices);
    const Tensor teacher = dense(teacher_logits.to(at::kFloat)), labels = dense(label_opt);
    auto [loss, dz] =
        distill_forward(z, index, teacher, labels, tau, alpha, reduction, reduction != 0);
    ctx->save_for_backward({z, index, teacher, labels});
    ctx->saved_data["tau"] = tau;
    ctx->saved_data["alpha"] = alpha;
    ctx->saved_data["reduction"] = reduction;
    if (dz.defined()) ctx->saved_data["ready"] = dz;
    return loss;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &z = saved[0];
    refuse("distillation_loss's gradient", {&grads[0]});
    c10::cuda::CUDAGuard guard(z.device());
    const Tensor dloss = dense(grads[0].to(at::kFloat));
    Tensor dz;
    const auto ready = ctx->saved_data.find("ready");
    if (ready != ctx->saved_data.end()) {
      dz = ready->second.toTensor();
      ctx->saved_data.erase(ready);
      check(lib.distill_scale(ptr(dz), dtype_of(z), dz.numel(), (const float *)ptr(dloss),
                              stream_of(z)),
            "distill_scale");
    } else {
      dz = distill_backward(z, saved[1], saved[2], saved[3], ctx->saved_data["tau"].toDouble(),
                            ctx->saved_data["alpha"].toDouble(),
                            ctx->saved_data["reduction"].toInt(), dloss);
    }
    return once({dz, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()},
                "distillation_loss");
  }
};

// ---------------------------------------------------------------- module
Tensor tensor_arg(PyObject *o) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), "expected a tensor");
  return THPVariable_Unpack(o);
}
Tensor optional_arg(PyObject *o) { return o == Py_None ? Tensor() : tensor_arg(o); }
OptTensor opt(const Tensor &t) { return t.defined() ? OptTensor(t) : OptTensor(); }
int64_t int_arg(PyObject *o) {
  const int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
double float_arg(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
void want_args(Py_ssize_t n, Py_ssize_t want) {
  TORCH_CHECK_TYPE(n == want, "expected ", want, " arguments, got ", n);
}
PyObject *wrap(const Tensor &t) {
  if (!t.defined()) Py_RETURN_NONE;
  return THPVariable_Wrap(t);
}
PyObject *wrap_tuple(std::initializer_list<Tensor> ts) {
  PyObject *out = PyTuple_New((Py_ssize_t)ts.size());
  if (!out) throw python_error();
  Py_ssize_t i = 0;
  for (const Tensor &t : ts) PyTuple_SET_ITEM(out, i++, wrap(t));
  return out;
}
// Without the GIL: a launch may wait for room in the stream's queue.
struct NoGil {
  PyThreadState *state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

PyObject *py_bind(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Py_ssize_t i = 0;
#define X(name) ++i;
  LNET_ENTRIES(X)
#undef X
  want_args(n, i);
  i = 0;
#define X(name) lib.name = reinterpret_cast<decltype(lib.name)>((uintptr_t)int_arg(args[i++]));
  LNET_ENTRIES(X)
#undef X
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

PyObject *py_entries(PyObject *, PyObject *) {
  const char *names[] = {
#define X(name) "lnet_b200_" #name,
      LNET_ENTRIES(X)
#undef X
  };
  const Py_ssize_t n = (Py_ssize_t)(sizeof(names) / sizeof(names[0]));
  PyObject *out = PyTuple_New(n);
  if (!out) return nullptr;
  for (Py_ssize_t i = 0; i < n; ++i) PyTuple_SET_ITEM(out, i, PyUnicode_FromString(names[i]));
  return out;
}

// (x, weight, residual | None, eps) -> (y, stream)
PyObject *py_norm(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 4);
  const Tensor x = tensor_arg(args[0]), w = tensor_arg(args[1]), r = optional_arg(args[2]);
  const double eps = float_arg(args[3]);
  refuse("residual_rms_norm", {&x, &w, &r});
  Tensor y, stream;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(x.device());
    if (tracked({&x, &w, &r})) {
      auto out = NormFunction::apply(x, w, opt(r), eps);
      y = out[0], stream = out[1];
    } else {
      NormOut o = norm_forward(dense(x), dense(w), dense(r), eps, false);
      y = o.y, stream = r.defined() ? o.stream : x;
    }
  }
  return wrap_tuple({y, stream});
  END_HANDLE_TH_ERRORS
}

// (x, weight, residual | None, eps) -> (y, stream | None, rstd), without autograd
PyObject *py_norm_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 4);
  const Tensor x = tensor_arg(args[0]), w = tensor_arg(args[1]), r = optional_arg(args[2]);
  const double eps = float_arg(args[3]);
  refuse("residual_rms_norm", {&x, &w, &r});
  NormOut o;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(x.device());
    o = norm_forward(dense(x), dense(w), dense(r), eps, true);
  }
  return wrap_tuple({o.y, o.stream, o.rstd});
  END_HANDLE_TH_ERRORS
}

// (stream, rstd, weight, dy, dstream | None) -> (dx, dweight), without autograd
PyObject *py_norm_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 5);
  const Tensor h = tensor_arg(args[0]), rstd = tensor_arg(args[1]), w = tensor_arg(args[2]);
  const Tensor dy = tensor_arg(args[3]), dh = optional_arg(args[4]);
  refuse("residual_rms_norm", {&h, &rstd, &w, &dy, &dh});
  Tensor dx, dw;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(h.device());
    std::tie(dx, dw) = norm_backward(dense(h), dense(rstd), dense(w), dense(dy), dense(dh), true);
  }
  return wrap_tuple({dx, dw});
  END_HANDLE_TH_ERRORS
}

// (x, weight, residual | None, eps) -> (values, scales, stream)
PyObject *py_norm_fp8(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 4);
  const Tensor x0 = tensor_arg(args[0]), w0 = tensor_arg(args[1]), r0 = optional_arg(args[2]);
  const double eps = float_arg(args[3]);
  refuse("residual_rms_norm_fp8", {&x0, &w0, &r0});
  Tensor q, s, stream;
  {
    NoGil gil;
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x0.device());
    const Tensor x = dense(x0), w = dense(w0), r = dense(r0);
    q = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
    s = at::empty(x.sizes().slice(0, x.dim() - 1), x.options().dtype(at::kFloat));
    stream = r.defined() ? at::empty_like(x) : x0;
    check(lib.residual_rms_norm_fp8(ptr(x), ptr(r), ptr(w), dtype_of(x), dtype_of(w), rows_of(x),
                                    x.size(-1), (float)eps, (uint8_t *)ptr(q), (float *)ptr(s),
                                    r.defined() ? ptr(stream) : nullptr, stream_of(x)),
          "residual_rms_norm_fp8");
  }
  return wrap_tuple({q, s, stream});
  END_HANDLE_TH_ERRORS
}

// (t) -> (values, scales)
PyObject *py_quantize(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 1);
  const Tensor t0 = tensor_arg(args[0]);
  refuse("quantize_rows_fp8", {&t0});
  Tensor q, s;
  {
    NoGil gil;
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(t0.device());
    const Tensor t = dense(t0);
    q = at::empty(t.sizes(), t.options().dtype(at::kFloat8_e4m3fn));
    s = at::empty(t.sizes().slice(0, t.dim() - 1), t.options().dtype(at::kFloat));
    check(lib.quantize_rows_fp8(ptr(t), dtype_of(t), rows_of(t), t.size(-1), (uint8_t *)ptr(q),
                                (float *)ptr(s), stream_of(t)),
          "quantize_rows_fp8");
  }
  return wrap_tuple({q, s});
  END_HANDLE_TH_ERRORS
}

// (x, weight, bias | None, residual | None, activation) -> y
PyObject *py_linear(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 5);
  const Tensor x = tensor_arg(args[0]), w = tensor_arg(args[1]);
  const Tensor b = optional_arg(args[2]), r = optional_arg(args[3]);
  const int64_t act = int_arg(args[4]);
  refuse("linear_act", {&x, &w, &b, &r});
  Tensor y;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(x.device());
    if (tracked({&x, &w, &b, &r})) {
      y = LinearFunction::apply(x, w, opt(b), opt(r), act);
    } else {
      y = linear_forward(x, w, b, r, act, Tensor(), Tensor(), false).y;
    }
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

// (x, weight, activation, preact | None, dy) -> (dx, dweight, dbias), without autograd
PyObject *py_linear_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 5);
  const Tensor x = tensor_arg(args[0]), w = tensor_arg(args[1]);
  const int64_t act = int_arg(args[2]);
  const Tensor pre = optional_arg(args[3]), dy = tensor_arg(args[4]);
  refuse("linear_act", {&x, &w, &pre, &dy});
  variable_list g;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(x.device());
    g = linear_backward(operand(x, true), operand(w, true), act, dense(pre), dense(dy), 7,
                        x.sizes());
  }
  return wrap_tuple({g[0], g[1], g[2]});
  END_HANDLE_TH_ERRORS
}

// (x, weight, bias | None, residual | None, activation) -> (y, preact), without autograd
PyObject *py_linear_forward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 5);
  const Tensor x = tensor_arg(args[0]), w = tensor_arg(args[1]);
  const Tensor b = optional_arg(args[2]), r = optional_arg(args[3]);
  const int64_t act = int_arg(args[4]);
  refuse("linear_act", {&x, &w, &b, &r});
  LinearOut out;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(x.device());
    out = linear_forward(x, w, b, r, act, Tensor(), Tensor(), act != 0);
  }
  return wrap_tuple({out.y, out.pre});
  END_HANDLE_TH_ERRORS
}

// (x, x_scale, weight, weight_scale, bias | None, residual | None, activation) -> y
PyObject *py_linear_fp8(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 7);
  const Tensor x = tensor_arg(args[0]), xs = tensor_arg(args[1]), w = tensor_arg(args[2]);
  const Tensor ws = tensor_arg(args[3]), b = optional_arg(args[4]), r = optional_arg(args[5]);
  const int64_t act = int_arg(args[6]);
  refuse("linear_act_fp8", {&x, &xs, &w, &ws, &b, &r});
  Tensor y;
  {
    NoGil gil;
    at::NoGradGuard no_grad;
    c10::cuda::CUDAGuard guard(x.device());
    y = linear_forward(x, w, b, r, act, xs, ws, false).y;
  }
  return wrap(y);
  END_HANDLE_TH_ERRORS
}

struct DistillArgs {
  Tensor z, index, teacher, labels;
  double tau, alpha;
  int64_t reduction;
  explicit DistillArgs(PyObject *const *args)
      : z(tensor_arg(args[0])),
        index(tensor_arg(args[1])),
        teacher(tensor_arg(args[2])),
        labels(optional_arg(args[3])),
        tau(float_arg(args[4])),
        alpha(float_arg(args[5])),
        reduction(int_arg(args[6])) {}
};

// (logits, indices, teacher logits, labels | None, temperature, alpha, reduction) -> loss
PyObject *py_distill(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 7);
  const DistillArgs a(args);
  refuse("distillation_loss", {&a.z, &a.teacher});
  Tensor loss;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(a.z.device());
    if (tracked({&a.z}))
      loss = DistillFunction::apply(a.z, a.index, a.teacher, opt(a.labels), a.tau, a.alpha,
                                    a.reduction);
    else
      loss = distill_forward(dense(a.z), dense(a.index), dense(a.teacher.to(at::kFloat)),
                             dense(a.labels), a.tau, a.alpha, a.reduction, false)
                 .first;
  }
  return wrap(loss);
  END_HANDLE_TH_ERRORS
}

// py_distill's arguments and dloss -> dlogits, without autograd
PyObject *py_distill_backward(PyObject *, PyObject *const *args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  want_args(n, 8);
  const DistillArgs a(args);
  const Tensor dloss = tensor_arg(args[7]);
  refuse("distillation_loss", {&a.z, &a.teacher, &dloss});
  Tensor dz;
  {
    NoGil gil;
    c10::cuda::CUDAGuard guard(a.z.device());
    dz = distill_backward(dense(a.z), dense(a.index), dense(a.teacher.to(at::kFloat)),
                          dense(a.labels), a.tau, a.alpha, a.reduction,
                          dense(dloss.to(at::kFloat)));
  }
  return wrap(dz);
  END_HANDLE_TH_ERRORS
}

#define FAST(name) reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(name)), METH_FASTCALL
PyMethodDef methods[] = {
    {"entries", py_entries, METH_NOARGS, "C ABI symbols that bind() takes the addresses of"},
    {"bind", FAST(py_bind), "addresses of the loaded library's entry points"},
    {"norm", FAST(py_norm), nullptr},
    {"norm_forward", FAST(py_norm_forward), nullptr},
    {"norm_backward", FAST(py_norm_backward), nullptr},
    {"norm_fp8", FAST(py_norm_fp8), nullptr},
    {"quantize", FAST(py_quantize), nullptr},
    {"linear", FAST(py_linear), nullptr},
    {"linear_forward", FAST(py_linear_forward), nullptr},
    {"linear_backward", FAST(py_linear_backward), nullptr},
    {"linear_fp8", FAST(py_linear_fp8), nullptr},
    {"distill", FAST(py_distill), nullptr},
    {"distill_backward", FAST(py_distill_backward), nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_torch_ops", nullptr, -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_ops(void) { return PyModule_Create(&module); }

// Python binding of the training and serving operators: checks PyTorch tensors,
// fills the C ABI's parameter blocks (include/avey_b200.h) and calls the library
// on the tensors' device and its current stream. Host code only; the library's
// entry points are handed over by bind() (avey_kernel_b200/_binding.py), so that
// there is one loaded library in a process. Bad arguments raise ValueError;
// a non-OK AveyStatus is returned and raised by the Python side.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <cmath>
#include <vector>

#include "avey_b200.h"

namespace {

using at::Tensor;

struct Library {
  int (*adamw)(const AveyAdamWParams*, void*) = nullptr;
  int (*linear_fwd)(const AveyLinearParams*, void*) = nullptr;
  int (*linear_bwd)(const AveyLinearParams*, void*) = nullptr;
  int (*linear_workspace)(const AveyLinearParams*, int, uint64_t*) = nullptr;
  int (*loss_fwd)(const AveyLossParams*, void*) = nullptr;
  int (*loss_bwd)(const AveyLossParams*, void*) = nullptr;
  int (*loss_workspace)(const AveyLossParams*, int, uint64_t*) = nullptr;
  int (*route_fwd)(const AveyRouteParams*, void*) = nullptr;
  int (*route_bwd)(const AveyRouteParams*, void*) = nullptr;
  int (*arrange)(const AveyArrangeParams*, void*) = nullptr;
  int (*arrange_workspace)(const AveyArrangeParams*, uint64_t*) = nullptr;
  int (*dispatch)(const AveyRowsParams*, void*) = nullptr;
  int (*combine)(const AveyRowsParams*, void*) = nullptr;
  int (*combine_bwd)(const AveyRowsParams*, void*) = nullptr;
  int (*rows_workspace)(const AveyRowsParams*, uint64_t*) = nullptr;
  int (*embedding_fwd)(const AveyEmbeddingParams*, void*) = nullptr;
  int (*embedding_bwd)(const AveyEmbeddingParams*, void*) = nullptr;
  int (*embedding_workspace)(const AveyEmbeddingParams*, uint64_t*) = nullptr;
  const char* (*last_error)() = nullptr;
};
Library lib;

int dtype_id(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return AVEY_F32;
    case at::kHalf: return AVEY_F16;
    case at::kBFloat16: return AVEY_BF16;
    default: return -1;
  }
}

// The operators work on the memory of their tensors, which torch does not see: a
// forward-mode derivative would be lost and a trace would hold their outputs as
// they were allocated, so both are refused. `visit(f)` calls f for each tensor.
template <typename Visit>
void refuse_unseen(Visit visit) {
  const bool traced =
      torch::jit::tracer::isTracing() || c10::impl::tls_is_dispatch_key_included(c10::DispatchKey::PreDispatch) ||
      (c10::impl::TorchDispatchModeTLS::any_modes_set() &&
       c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY).has_value());
  TORCH_CHECK(!traced, "the native operators cannot be traced (torch.jit.trace, make_fx)");
  // Tangents exist within a level of forward-mode differentiation only; there is one at most.
  if (!torch::autograd::ForwardADLevel::try_get_by_idx(0)) return;
  visit([](const Tensor& t) {
    TORCH_CHECK(!t.defined() || !t._fw_grad(0).defined(),
                "the native operators have no forward-mode derivative (a tensor has a tangent)");
  });
}

// ------------------------------------------------------------------- AdamW

// A list or tuple of tensors, read without copying them.
class TensorList {
 public:
  TensorList(const py::object& o, const char* name) : name_(name) {
    if (o.is_none()) return;
    given_ = true;
    seq_ = py::reinterpret_steal<py::object>(PySequence_Fast(o.ptr(), "a list of tensors is expected"));
    if (!seq_) throw py::error_already_set();
    n_ = PySequence_Fast_GET_SIZE(seq_.ptr());
    items_ = PySequence_Fast_ITEMS(seq_.ptr());
    for (Py_ssize_t i = 0; i < n_; ++i)
      TORCH_CHECK_VALUE(THPVariable_Check(items_[i]), name, "[", i, "] is not a tensor");
  }
  bool given() const { return given_; }
  Py_ssize_t size() const { return n_; }
  const Tensor& operator[](Py_ssize_t i) const { return THPVariable_Unpack(items_[i]); }
  void need(Py_ssize_t n) const {
    TORCH_CHECK_VALUE(given_ && n_ == n, name_, " must hold one tensor for each parameter");
  }

 private:
  const char* name_;
  bool given_ = false;
  py::object seq_;
  Py_ssize_t n_ = 0;
  PyObject** items_ = nullptr;
};

void same_layout(const Tensor& t, const Tensor& p, const char* name, Py_ssize_t i) {
  TORCH_CHECK_VALUE(t.sizes() == p.sizes() && (t.strides() == p.strides() || p.numel() <= 1), name, "[", i,
                    "] must have the shape and strides of its parameter");
}

int adamw_step(const py::object& params, const py::object& grads, const py::object& exp_avgs,
               const py::object& exp_avg_sqs, const py::object& masters, const py::object& avg_scales,
               const py::object& sq_scales, int64_t step, double lr, double beta1, double beta2, double eps,
               double weight_decay, uint64_t seed, const std::optional<Tensor>& grad_scale) {
  const TensorList p(params, "params"), g(grads, "grads"), m(exp_avgs, "exp_avgs"), v(exp_avg_sqs, "exp_avg_sqs"),
      w(masters, "masters"), ms(avg_scales, "exp_avg_scales"), vs(sq_scales, "exp_avg_sq_scales");
  const Py_ssize_t n = p.size();
  g.need(n);
  m.need(n);
  v.need(n);
  if (w.given()) w.need(n);
  if (n == 0) return AVEY_OK;
  refuse_unseen([&](auto f) {
    for (const TensorList* l : {&p, &g, &m, &v, &w, &ms, &vs})
      for (Py_ssize_t i = 0; i < l->size(); ++i) f((*l)[i]);
    if (grad_scale) f(*grad_scale);
  });
  const auto device = p[0].device();
  const auto dt = p[0].scalar_type();
  const auto state_type = m[0].scalar_type();
  const bool q8 = state_type == at::kFloat8_e4m3fn;
  TORCH_CHECK_VALUE(device.is_cuda(), "the native AdamW step needs CUDA tensors");
  TORCH_CHECK_VALUE(dtype_id(p[0]) >= 0, "parameters must be float32, float16 or bfloat16");
  TORCH_CHECK_VALUE(q8 || state_type == at::kFloat, "states must be float32 or float8_e4m3fn");
  TORCH_CHECK_VALUE(ms.given() == q8 && vs.given() == q8,
                    "exp_avg_scales and exp_avg_sq_scales go with float8_e4m3fn states, and only with them");
  if (q8) {
    ms.need(n);
    vs.need(n);
  }
  std::vector<AveyAdamWTensor> table(n);
  std::vector<Tensor> keep;  // gradients laid out like their parameters
  for (Py_ssize_t i = 0; i < n; ++i) {
    const Tensor &pi = p[i], &gi = g[i], &mi = m[i], &vi = v[i];
    TORCH_CHECK_VALUE(pi.device() == device && gi.device() == device && mi.device() == device &&
                          vi.device() == device,
                      "all tensors of a step must be on one device (number ", i, " is not)");
    TORCH_CHECK_VALUE(pi.scalar_type() == dt && gi.scalar_type() == dt,
                      "parameters and gradients of a step must have one type (number ", i, " has not)");
    TORCH_CHECK_VALUE(mi.scalar_type() == state_type && vi.scalar_type() == state_type,
                      "the states of a step must have one type (number ", i, " has not)");
    TORCH_CHECK_VALUE(gi.layout() == at::kStrided && pi.layout() == at::kStrided, "sparse tensors are not supported");
    TORCH_CHECK_VALUE(pi.is_non_overlapping_and_dense(), "params[", i, "] must be dense in memory");
    TORCH_CHECK_VALUE(gi.sizes() == pi.sizes(), "grads[", i, "] must have the shape of its parameter");
    same_layout(mi, pi, "exp_avgs", i);
    same_layout(vi, pi, "exp_avg_sqs", i);
    AveyAdamWTensor& t = table[i];
    t.numel = pi.numel();
    t.param = pi.data_ptr();
    if (gi.strides() == pi.strides() || t.numel <= 1) {
      t.grad = gi.const_data_ptr();
    } else {
      keep.push_back(at::empty_like(pi).copy_(gi));
      t.grad = keep.back().const_data_ptr();
    }
    t.exp_avg = mi.data_ptr();
    t.exp_avg_sq = vi.data_ptr();
    if (w.given()) {
      const Tensor& wi = w[i];
      TORCH_CHECK_VALUE(wi.device() == device && wi.scalar_type() == at::kFloat, "masters[", i,
                        "] must be float32 on the parameters' device");
      same_layout(wi, pi, "masters", i);
      t.master = static_cast<float*>(wi.data_ptr());
    }
    if (q8) {
      const int64_t blocks = (t.numel + AVEY_ADAMW_BLOCK - 1) / AVEY_ADAMW_BLOCK;
      for (const Tensor* s : {&ms[i], &vs[i]})
        TORCH_CHECK_VALUE(s->device() == device && s->scalar_type() == at::kFloat && s->is_contiguous() &&
                              s->numel() == blocks,
                          "scales of parameter ", i, " must be ", blocks, " contiguous float32 values");
      t.exp_avg_scale = static_cast<float*>(ms[i].data_ptr());
      t.exp_avg_sq_scale = static_cast<float*>(vs[i].data_ptr());
    }
  }
  std::vector<const void*> starts;
  starts.reserve(n);
  for (const auto& t : table)
    if (t.numel) starts.push_back(t.param);
  std::sort(starts.begin(), starts.end());
  TORCH_CHECK_VALUE(std::adjacent_find(starts.begin(), starts.end()) == starts.end(),
                    "a parameter is listed more than once");
  AveyAdamWParams a{};
  a.struct_size = sizeof(a);
  a.dtype = dtype_id(p[0]);
  a.state_bits = q8 ? 8 : 32;
  a.count = static_cast<int32_t>(n);
  a.tensors = table.data();
  a.lr = lr;
  a.beta1 = beta1;
  a.beta2 = beta2;
  a.eps = eps;
  a.weight_decay = weight_decay;
  a.step = step;
  a.seed = seed;
  if (grad_scale) {
    TORCH_CHECK_VALUE(grad_scale->device() == device && grad_scale->scalar_type() == at::kFloat &&
                          grad_scale->numel() == 1,
                      "grad_scale must be one float32 value on the parameters' device");
    a.grad_scale = static_cast<const float*>(grad_scale->const_data_ptr());
  }
  const c10::cuda::CUDAGuard guard(device);
  const int status = lib.adamw(&a, at::cuda::getCurrentCUDAStream().stream());
  // Autograd sees that the parameters changed, as after any in-place operation.
  if (status == AVEY_OK)
    for (Py_ssize_t i = 0; i < n; ++i) torch::autograd::impl::bump_version(p[i]);
  return status;
}

// ------------------------------------------------------------ linear layers

void check_status(int status) { TORCH_CHECK(status == AVEY_OK, "status ", status, ": ", lib.last_error()); }

// t as rows of `cols` values with unit stride (a copy only where no view has that form).
Tensor as_rows(const Tensor& t, int64_t cols) {
  Tensor r = t.dim() == 2 ? t : t.reshape({-1, cols});
  if ((cols > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < cols)) r = r.contiguous();
  return r;
}
// Row stride; a single row may claim any.
int64_t row_ld(const Tensor& r, int64_t cols) { return r.size(0) > 1 ? r.stride(0) : (cols + 7) / 8 * 8; }

// The weights [d_out, d_in] or [groups, d_out, d_in] with unit stride along d_in.
Tensor as_weight(const Tensor& w) {
  const int64_t n = w.size(-2), k = w.size(-1);
  const bool ok = (k == 1 || w.stride(-1) == 1) && (n == 1 || w.stride(-2) >= k) &&
                  (w.dim() == 2 || w.size(0) == 1 || w.stride(0) >= (n > 1 ? (n - 1) * w.stride(-2) : 0) + k);
  return ok ? w : w.contiguous();
}

// The parameter block but for the operands, from the shapes of x and the weights;
// `like` has their type.
AveyLinearParams linear_params(at::IntArrayRef x, at::IntArrayRef w, const Tensor* offsets, const Tensor& like,
                               int64_t act) {
  AveyLinearParams p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_id(like);
  p.activation = static_cast<int32_t>(act);
  p.d_in = w[w.size() - 1];
  p.d_out = w[w.size() - 2];
  p.rows = 1;
  for (size_t i = 0; i + 1 < x.size(); ++i) p.rows *= x[i];
  p.groups = offsets ? w[0] : 1;
  if (offsets) p.offsets = static_cast<const int32_t*>(offsets->const_data_ptr());
  p.x_ld = p.weight_ld = p.d_in;
  if (p.groups > 1) p.weight_group_stride = p.d_out * p.d_in;
  return p;
}
void set_x(AveyLinearParams& p, const Tensor& x) {
  p.x = x.const_data_ptr();
  p.x_ld = row_ld(x, p.d_in);
}
void set_weight(AveyLinearParams& p, const Tensor& w) {
  p.weight = w.const_data_ptr();
  p.weight_ld = p.d_out > 1 ? w.stride(-2) : (p.d_in + 7) / 8 * 8;
  if (p.groups > 1) p.weight_group_stride = w.stride(0);
}

Tensor workspace(AveyLinearParams& p, int backward, const Tensor& like) {
  uint64_t bytes = 0;
  check_status(lib.linear_workspace(&p, backward, &bytes));
  if (bytes == 0) return {};
  Tensor ws = at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
  p.workspace = ws.data_ptr();
  p.workspace_bytes = bytes;
  return ws;
}

// y and, with want_deriv, the codes of act'.
std::pair<Tensor, Tensor> linear_forward(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
                                         const std::optional<Tensor>& residual, const std::optional<Tensor>& offsets,
                                         int64_t act, int64_t kernel, bool want_deriv) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor w = as_weight(weight), xr = as_rows(x, weight.size(-1));
  AveyLinearParams p = linear_params(x.sizes(), w.sizes(), offsets ? &*offsets : nullptr, x, act);
  set_x(p, xr);
  set_weight(p, w);
  p.kernel = static_cast<int32_t>(kernel);
  Tensor b, r, deriv;
  if (bias) {
    b = bias->contiguous();
    p.bias = b.const_data_ptr();
    p.bias_group_stride = p.d_out;
  }
  if (residual) {
    r = as_rows(*residual, p.d_out);
    p.residual = r.const_data_ptr();
    p.residual_ld = row_ld(r, p.d_out);
  }
  auto shape = x.sizes().vec();
  shape.back() = p.d_out;
  Tensor y = at::empty(shape, x.options());
  p.y = y.data_ptr();
  p.y_ld = p.d_out;
  if (want_deriv && act != AVEY_ACT_IDENTITY && p.rows > 0) {
    deriv = at::empty({p.rows, (p.d_out + 15) / 16 * 16}, x.options().dtype(at::kShort));
    p.deriv = deriv.data_ptr();
  }
  const Tensor ws = workspace(p, 0, x);
  check_status(lib.linear_fwd(&p, at::cuda::getCurrentCUDAStream().stream()));
  return {y, deriv};
}

class LinearFunction : public torch::autograd::Function<LinearFunction> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const std::optional<Tensor>& bias, const std::optional<Tensor>& residual,
                        const std::optional<Tensor>& offsets, int64_t act, int64_t kernel) {
    const bool want = x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad());
    auto [y, deriv] = linear_forward(x, weight, bias, residual, offsets, act, kernel, want);
    // x goes into dW and the weights into dx only: what is not needed is neither
    // held nor has to stay as it is.
    ctx->save_for_backward({weight.requires_grad() ? x : Tensor(), x.requires_grad() ? weight : Tensor(),
                            offsets ? *offsets : Tensor(), deriv});
    // The call's numbers: activation, the bias's dimensions, whether there is a
    // residual, the dimensions of x, and the sizes of x and the weights.
    std::vector<int64_t> call{act, bias ? bias->dim() : 0, residual.has_value(), x.dim()};
    call.insert(call.end(), x.sizes().begin(), x.sizes().end());
    call.insert(call.end(), weight.sizes().begin(), weight.sizes().end());
    ctx->saved_data["call"] = std::move(call);
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "the gradients of the native linear layers cannot be differentiated again (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1], &offs = saved[2], &deriv = saved[3];
    const std::vector<int64_t> call = ctx->saved_data["call"].toIntVector();
    const at::IntArrayRef sizes = at::IntArrayRef(call).slice(4), x_sizes = sizes.slice(0, call[3]),
                          w_sizes = sizes.slice(call[3]);
    const int64_t has_bias = call[1];
    torch::autograd::variable_list out(7);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    refuse_unseen([&](auto f) { f(dy); });
    // needs_input_grad counts the tensors that were given.
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1),
               need_b = has_bias && ctx->needs_input_grad(2);
    if (call[2] && ctx->needs_input_grad(has_bias ? 3 : 2)) out[3] = dy;
    if (!need_x && !need_w && !need_b) return out;
    const c10::cuda::CUDAGuard guard(dy.device());
    AveyLinearParams p = linear_params(x_sizes, w_sizes, offs.defined() ? &offs : nullptr, dy, call[0]);
    Tensor w, xr;
    if (need_x) set_weight(p, w = as_weight(weight));
    if (need_w) set_x(p, xr = as_rows(x, p.d_in));
    const Tensor g = as_rows(dy, p.d_out);
    p.dy = g.const_data_ptr();
    p.dy_ld = row_ld(g, p.d_out);
    if (deriv.defined()) p.deriv = deriv.data_ptr();
    if (need_x) {
      out[0] = at::empty(x_sizes, dy.options());
      p.dx = out[0].data_ptr();
      p.dx_ld = p.d_in;
    }
    if (need_w) {
      out[1] = at::empty(w_sizes, dy.options());
      p.dweight = out[1].data_ptr();
    }
    if (need_b) {
      out[2] = has_bias == 2 ? at::empty({p.groups, p.d_out}, dy.options()) : at::empty({p.d_out}, dy.options());
      p.dbias = out[2].data_ptr();
    }
    const Tensor ws = workspace(p, 1, dy);
    check_status(lib.linear_bwd(&p, at::cuda::getCurrentCUDAStream().stream()));
    return out;
  }
};

Tensor linear(const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias,
              const std::optional<Tensor>& residual, const std::optional<Tensor>& offsets, int64_t act,
              int64_t kernel) {
  refuse_unseen([&](auto f) {
    f(x);
    f(weight);
    for (const std::optional<Tensor>* t : {&bias, &residual})
      if (*t) f(**t);
  });
  const auto dt = x.scalar_type();
  const auto device = x.device();
  TORCH_CHECK_VALUE(device.is_cuda() && (dt == at::kBFloat16 || dt == at::kHalf),
                    "the native linear layers take bf16 / f16 CUDA tensors of one dtype");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == (offsets ? 3 : 2) && weight.size(-1) == x.size(-1) &&
                        weight.size(-1) > 0 && weight.size(-2) > 0,
                    "x must be [..., d_in] and weight ", offsets ? "[experts, d_out, d_in]" : "[d_out, d_in]");
  for (const std::optional<Tensor>& t : {std::optional<Tensor>(weight), bias, residual})
    TORCH_CHECK_VALUE(!t || (t->scalar_type() == dt && t->device() == device),
                      "the native linear layers take bf16 / f16 CUDA tensors of one dtype");
  if (bias) {
    auto want = weight.sizes().vec();
    want.pop_back();
    TORCH_CHECK_VALUE(bias->sizes() == at::IntArrayRef(want), "bias must have shape ", at::IntArrayRef(want));
  }
  if (residual) {
    auto want = x.sizes().vec();
    want.back() = weight.size(-2);
    TORCH_CHECK_VALUE(residual->sizes() == at::IntArrayRef(want), "residual must have shape ", at::IntArrayRef(want));
  }
  if (offsets) {
    TORCH_CHECK_VALUE(x.dim() == 2, "x must be [rows, d_in]");
    TORCH_CHECK_VALUE(weight.size(0) > 0, "weight must hold at least one expert");
    TORCH_CHECK_VALUE(offsets->dim() == 1 && offsets->size(0) == weight.size(0) + 1 &&
                          offsets->scalar_type() == at::kInt && offsets->device() == device &&
                          offsets->is_contiguous(),
                      "offsets must be ", weight.size(0) + 1, " contiguous int32 values on x's device");
  }
  if (at::GradMode::is_enabled() &&
      (x.requires_grad() || weight.requires_grad() || (bias && bias->requires_grad()) ||
       (residual && residual->requires_grad())))
    return LinearFunction::apply(x, weight, bias, residual, offsets, act, kernel);
  return linear_forward(x, weight, bias, residual, offsets, act, kernel, false).first;
}

// ------------------------------------------------------------ cross entropy

void check_integers(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt || t.scalar_type() == at::kLong, name, " must be int32 or int64");
}

// The parameter block but for the operands, and for `targets` [rows].
AveyLossParams loss_params(const Tensor& like, int64_t rows, int64_t width, int64_t vocab, const Tensor& targets,
                           int64_t ignore, int64_t reduction, double z_loss) {
  AveyLossParams p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_id(like);
  p.target_bits = targets.scalar_type() == at::kLong ? 64 : 32;
  p.reduction = static_cast<int32_t>(reduction);
  p.rows = rows;
  p.width = width;
  p.vocab = vocab;
  p.targets = targets.const_data_ptr();
  p.target_stride = rows > 1 ? targets.stride(0) : 1;
  p.ignore_index = ignore;
  p.z_loss = z_loss;
  return p;
}

Tensor loss_workspace(AveyLossParams& p, int backward, const Tensor& like) {
  uint64_t bytes = 0;
  check_status(lib.loss_workspace(&p, backward, &bytes));
  if (bytes == 0) return {};
  Tensor ws = at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
  p.workspace = ws.data_ptr();
  p.workspace_bytes = bytes;
  return ws;
}

// The operands of a call, as the library takes them: rows with unit stride.
struct LossRows {
  Tensor x, w, t;
  LossRows(AveyLossParams& p, const Tensor& x_, const Tensor& w_) : x(as_rows(x_, p.width)), w(as_weight(w_)) {
    p.x = x.const_data_ptr();
    p.x_ld = row_ld(x, p.width);
    p.weight = w.const_data_ptr();
    p.weight_ld = p.vocab > 1 ? w.stride(0) : (p.width + 7) / 8 * 8;
  }
};

void set_saved(AveyLossParams& p, const Tensor& saved) {
  p.saved = saved.data_ptr<float>();
  p.saved_low = p.saved + p.rows + 1;
}

// The loss and, with keep, what the backward pass needs of it.
std::pair<Tensor, Tensor> loss_forward(const Tensor& x, const Tensor& weight, const Tensor& targets, int64_t ignore,
                                       int64_t reduction, double z_loss, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor t = targets.reshape({-1});
  AveyLossParams p = loss_params(x, t.size(0), weight.size(1), weight.size(0), t, ignore, reduction, z_loss);
  const LossRows rows(p, x, weight);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor loss = reduction == AVEY_LOSS_NONE ? at::empty(targets.sizes(), f32) : at::empty({}, f32), saved;
  p.loss = loss.data_ptr<float>();
  if (keep) {
    saved = at::empty({2 * p.rows + 1}, f32);
    set_saved(p, saved);
  }
  const Tensor ws = loss_workspace(p, 0, x);
  check_status(lib.loss_fwd(&p, at::cuda::getCurrentCUDAStream().stream()));
  return {loss, saved};
}

class LossFunction : public torch::autograd::Function<LossFunction> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const Tensor& targets, int64_t ignore, int64_t reduction, double z_loss) {
    auto [loss, saved] = loss_forward(x, weight, targets, ignore, reduction, z_loss, true);
    ctx->save_for_backward({x, weight, targets, saved});
    ctx->saved_data["call"] = std::vector<int64_t>{ignore, reduction};
    ctx->saved_data["z_loss"] = z_loss;
    return loss;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "the gradients of the native cross entropy cannot be differentiated again (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &weight = saved[1];
    const std::vector<int64_t> call = ctx->saved_data["call"].toIntVector();
    torch::autograd::variable_list out(6);
    if (!grads[0].defined()) return out;
    refuse_unseen([&](auto f) { f(grads[0]); });
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    if (!need_x && !need_w) return out;
    const c10::cuda::CUDAGuard guard(x.device());
    const Tensor t = saved[2].reshape({-1}), g = grads[0].reshape({-1});
    AveyLossParams p = loss_params(x, t.size(0), weight.size(1), weight.size(0), t, call[0], call[1],
                                   ctx->saved_data["z_loss"].toDouble());
    const LossRows rows(p, x, weight);
    set_saved(p, saved[3]);
    p.dloss = g.const_data_ptr<float>();
    p.dloss_stride = g.size(0) > 1 ? g.stride(0) : 1;
    if (need_x) {
      out[0] = at::empty(x.sizes(), x.options());
      p.dx = out[0].data_ptr();
      p.dx_ld = p.width;
    }
    if (need_w) {
      out[1] = at::empty(weight.sizes(), weight.options());
      p.dweight = out[1].data_ptr();
    }
    const Tensor ws = loss_workspace(p, 1, x);
    check_status(lib.loss_bwd(&p, at::cuda::getCurrentCUDAStream().stream()));
    return out;
  }
};

Tensor cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& targets, int64_t ignore, int64_t reduction,
                     double z_loss) {
  refuse_unseen([&](auto f) {
    f(x);
    f(weight);
  });
  const auto dt = x.scalar_type();
  TORCH_CHECK_VALUE(x.is_cuda() && (dt == at::kBFloat16 || dt == at::kHalf) && weight.scalar_type() == dt &&
                        weight.device() == x.device(),
                    "the native cross entropy takes bf16 / f16 CUDA tensors of one dtype");
  TORCH_CHECK_VALUE(x.dim() >= 1 && weight.dim() == 2 && weight.numel() > 0 && weight.size(1) == x.size(-1),
                    "x must be [..., width] and weight [vocab, width]");
  check_integers(targets, "targets");
  TORCH_CHECK_VALUE(targets.device() == x.device() && targets.sizes() == x.sizes().slice(0, x.dim() - 1),
                    "targets must have shape ", x.sizes().slice(0, x.dim() - 1), " on x's device");
  TORCH_CHECK_VALUE(std::isfinite(z_loss), "z_loss must be finite");
  if (at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad()))
    return LossFunction::apply(x, weight, targets, ignore, reduction, z_loss);
  return loss_forward(x, weight, targets, ignore, reduction, z_loss, false).first;
}

// ------------------------------------------------------------ routing

constexpr int64_t kMaxExperts = 1024, kMaxChoices = 32, kMaxGroups = 32;
void check_floating(const Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && dtype_id(t) >= 0, name, " must be a CUDA tensor of float32, float16 or bfloat16");
}
Tensor byte_workspace(uint64_t bytes, const Tensor& like) {
  return bytes ? at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte)) : Tensor();
}
void* stream_of() { return at::cuda::getCurrentCUDAStream().stream(); }

// The numbers of a call, as they are kept for the backward pass.
struct RouteCall {
  int64_t k, score, groups, top_groups, group_best, renormalize;
  double scale;
};
AveyRouteParams route_params(const Tensor& rows, const RouteCall& call) {
  AveyRouteParams p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_id(rows);
  p.score = static_cast<int32_t>(call.score);
  p.renormalize = static_cast<int32_t>(call.renormalize);
  p.k = static_cast<int32_t>(call.k);
  p.groups = static_cast<int32_t>(call.groups);
  p.top_groups = static_cast<int32_t>(call.top_groups);
  p.group_best = static_cast<int32_t>(call.group_best);
  p.tokens = rows.size(0);
  p.experts = rows.size(1);
  p.scale = call.scale;
  p.logits = rows.const_data_ptr();
  p.logits_ld = row_ld(rows, p.experts);
  return p;
}

std::pair<Tensor, Tensor> route_forward(const Tensor& logits, const std::optional<Tensor>& bias, const RouteCall& call) {
  const c10::cuda::CUDAGuard guard(logits.device());
  const Tensor rows = as_rows(logits, logits.size(-1));
  AveyRouteParams p = route_params(rows, call);
  auto shape = logits.sizes().vec();
  shape.back() = call.k;
  Tensor weights = at::empty(shape, logits.options().dtype(at::kFloat));
  Tensor chosen = at::empty(shape, logits.options().dtype(at::kInt));
  Tensor b;
  if (bias) {
    b = bias->contiguous();
    p.bias = b.const_data_ptr<float>();
  }
  p.weights = weights.data_ptr<float>();
  p.chosen = chosen.data_ptr<int32_t>();
  check_status(lib.route_fwd(&p, stream_of()));
  return {weights, chosen};
}

class RouteFunction : public torch::autograd::Function<RouteFunction> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits,
                                                const std::optional<Tensor>& bias, int64_t k, int64_t score,
                                                int64_t groups, int64_t top_groups, int64_t group_best,
                                                int64_t renormalize, double scale) {
    const RouteCall call{k, score, groups, top_groups, group_best, renormalize, scale};
    auto [weights, chosen] = route_forward(logits, bias, call);
    ctx->save_for_backward({logits, weights, chosen});
    ctx->mark_non_differentiable({chosen});
    ctx->set_materialize_grads(false);
    ctx->saved_data["call"] = std::vector<int64_t>{k, score, groups, top_groups, group_best, renormalize};
    ctx->saved_data["scale"] = scale;
    return {weights, chosen};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "the gradients of the native routing cannot be differentiated again (create_graph)");
    const auto saved = ctx->get_saved_variables();
    torch::autograd::variable_list out(9);
    const Tensor &logits = saved[0], &dw = grads[0];
    if (!dw.defined()) return out;
    refuse_unseen([&](auto f) { f(dw); });
    const std::vector<int64_t> c = ctx->saved_data["call"].toIntVector();
    const RouteCall call{c[0], c[1], c[2], c[3], c[4], c[5], ctx->saved_data["scale"].toDouble()};
    const c10::cuda::CUDAGuard guard(logits.device());
    const Tensor rows = as_rows(logits, logits.size(-1)), g = dw.contiguous();
    AveyRouteParams p = route_params(rows, call);
    p.weights = saved[1].data_ptr<float>();
    p.chosen = saved[2].data_ptr<int32_t>();
    p.dweights = g.const_data_ptr<float>();
    out[0] = at::empty(logits.sizes(), logits.options());
    p.dlogits = out[0].data_ptr();
    check_status(lib.route_bwd(&p, stream_of()));
    return out;
  }
};

std::pair<Tensor, Tensor> route(const Tensor& logits, const std::optional<Tensor>& bias, int64_t k, int64_t score,
                                int64_t groups, int64_t top_groups, int64_t group_best, bool renormalize,
                                double scale) {
  refuse_unseen([&](auto f) {
    f(logits);
    if (bias) f(*bias);
  });
  check_floating(logits, "logits");
  TORCH_CHECK_VALUE(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= kMaxExperts,
                    "logits must be [..., experts] with 1 to ", kMaxExperts, " experts");
  const int64_t experts = logits.size(-1);
  TORCH_CHECK_VALUE(groups >= 1 && groups <= kMaxGroups && experts % groups == 0 && top_groups >= 1 &&
                        top_groups <= groups,
                    "groups must divide the experts and be 1 to ", kMaxGroups, ", top_groups 1 to groups");
  TORCH_CHECK_VALUE(group_best == 1 || group_best == 2, "group_best must be 1 or 2");
  TORCH_CHECK_VALUE(k >= 1 && k <= kMaxChoices && k <= experts / groups * top_groups, "k must be 1 to ", kMaxChoices,
                    " and no more than the experts to choose from");
  TORCH_CHECK_VALUE(std::isfinite(scale), "scale must be finite");
  if (bias)
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat && bias->device() == logits.device() && bias->dim() == 1 &&
                          bias->size(0) == experts,
                      "bias must be float32 of shape [experts] on the logits' device");
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    auto out = RouteFunction::apply(logits, bias, k, score, groups, top_groups, group_best,
                                    static_cast<int64_t>(renormalize), scale);
    return {out[0], out[1]};
  }
  return route_forward(logits, bias, {k, score, groups, top_groups, group_best, renormalize, scale});
}

std::pair<Tensor, Tensor> arrange(const Tensor& chosen, int64_t experts) {
  refuse_unseen([](auto) {});
  check_integers(chosen, "chosen");
  TORCH_CHECK_VALUE(experts >= 1 && experts <= kMaxExperts, "num_experts must be 1 to ", kMaxExperts);
  const c10::cuda::CUDAGuard guard(chosen.device());
  const Tensor c = chosen.contiguous();
  const auto i32 = chosen.options().dtype(at::kInt);
  Tensor slots = at::empty(chosen.sizes(), i32), offsets = at::empty({experts + 1}, i32);
  AveyArrangeParams p{};
  p.struct_size = sizeof(p);
  p.index_bits = c.scalar_type() == at::kLong ? 64 : 32;
  p.count = c.numel();
  p.experts = experts;
  p.chosen = c.const_data_ptr();
  p.slots = slots.data_ptr<int32_t>();
  p.offsets = offsets.data_ptr<int32_t>();
  uint64_t bytes = 0;
  check_status(lib.arrange_workspace(&p, &bytes));
  const Tensor ws = byte_workspace(bytes, c);
  if (bytes) p.workspace = ws.data_ptr();
  p.workspace_bytes = bytes;
  check_status(lib.arrange(&p, stream_of()));
  return {slots, offsets};
}

// ------------------------------------------------------------ rows of tokens

AveyRowsParams rows_params(const Tensor& like, const Tensor& slots, int64_t width) {
  AveyRowsParams p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_id(like);
  p.tokens = slots.size(0);
  p.k = static_cast<int32_t>(slots.size(1));
  p.width = width;
  p.slots = slots.const_data_ptr<int32_t>();
  return p;
}
void set_rows(AveyRowsParams& p, const Tensor& rows) {
  p.rows = const_cast<void*>(rows.const_data_ptr());
  p.rows_ld = row_ld(rows, p.width);
}
void set_tokens(AveyRowsParams& p, const Tensor& x) {
  p.x = x.const_data_ptr();
  p.x_ld = row_ld(x, p.width);
}

// Places that no slot names get zeros: what a tensor held before never comes out.
Tensor clear_places(AveyRowsParams& p, const Tensor& like) {
  p.clear = 1;
  uint64_t bytes = 0;
  check_status(lib.rows_workspace(&p, &bytes));
  const Tensor ws = byte_workspace(bytes, like);
  if (bytes) p.workspace = ws.data_ptr();
  p.workspace_bytes = bytes;
  return ws;
}

Tensor dispatch_rows(const Tensor& x, const Tensor& slots) {
  const c10::cuda::CUDAGuard guard(x.device());
  const Tensor xr = as_rows(x, x.size(1)), s = slots.contiguous();
  AveyRowsParams p = rows_params(x, s, x.size(1));
  Tensor rows = at::empty({slots.numel(), x.size(1)}, x.options());
  set_tokens(p, xr);
  p.rows = rows.data_ptr();
  p.rows_ld = p.width;
  const Tensor ws = clear_places(p, x);
  check_status(lib.dispatch(&p, stream_of()));
  return rows;
}

Tensor combine_rows(const Tensor& rows, const Tensor& slots, const std::optional<Tensor>& weights,
                    const std::optional<Tensor>& residual) {
  const c10::cuda::CUDAGuard guard(rows.device());
  const Tensor r = as_rows(rows, rows.size(1)), s = slots.contiguous();
  AveyRowsParams p = rows_params(rows, s, rows.size(1));
  set_rows(p, r);
  Tensor w, res, out = at::empty({slots.size(0), rows.size(1)}, rows.options());
  if (weights) {
    w = weights->contiguous();
    p.weights = w.const_data_ptr<float>();
  }
  if (residual) set_tokens(p, res = as_rows(*residual, p.width));
  p.out = out.data_ptr();
  check_status(lib.combine(&p, stream_of()));
  return out;
}

class DispatchFunction : public torch::autograd::Function<DispatchFunction> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& slots) {
    ctx->save_for_backward({slots});
    return dispatch_rows(x, slots);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "the gradients of the native dispatch cannot be differentiated again (create_graph)");
    if (!grads[0].defined()) return {Tensor(), Tensor()};
    refuse_unseen([&](auto f) { f(grads[0]); });
    return {combine_rows(grads[0], ctx->get_saved_variables()[0], std::nullopt, std::nullopt), Tensor()};
  }
};

class CombineFunction : public torch::autograd::Function<CombineFunction> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& rows, const Tensor& slots,
                        const Tensor& weights, const std::optional<Tensor>& residual) {
    // The rows go into the weights' gradient only.
    ctx->save_for_backward({weights.requires_grad() ? rows : Tensor(), slots, weights});
    ctx->saved_data["residual"] = residual.has_value();
    return combine_rows(rows, slots, weights, residual);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "the gradients of the native combine cannot be differentiated again (create_graph)");
    torch::autograd::variable_list out(4);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    refuse_unseen([&](auto f) { f(dy); });
    const auto saved = ctx->get_saved_variables();
    // needs_input_grad counts the tensors that were given: rows, slots, weights, residual.
    const bool need_rows = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(2);
    if (ctx->saved_data["residual"].toBool() && ctx->needs_input_grad(3)) out[3] = dy;
    if (!need_rows && !need_w) return out;
    const c10::cuda::CUDAGuard guard(dy.device());
    const Tensor g = as_rows(dy, dy.size(1)), s = saved[1].contiguous(), w = saved[2].contiguous();
    AveyRowsParams p = rows_params(dy, s, dy.size(1));
    set_tokens(p, g);
    p.weights = w.const_data_ptr<float>();
    Tensor rows;
    if (need_w) {
      set_rows(p, rows = as_rows(saved[0], p.width));
      out[2] = at::empty(s.sizes(), w.options());
      p.dweights = out[2].data_ptr<float>();
    }
    Tensor ws;
    if (need_rows) {
      out[0] = at::empty({s.numel(), p.width}, dy.options());
      p.drows = out[0].data_ptr();
      ws = clear_places(p, dy);
    }
    check_status(lib.combine_bwd(&p, stream_of()));
    return out;
  }
};

void check_slots(const Tensor& slots, const Tensor& like) {
  TORCH_CHECK_VALUE(slots.dim() == 2 && slots.scalar_type() == at::kInt && slots.device() == like.device() &&
                        slots.size(1) >= 1 && slots.size(1) <= kMaxChoices,
                    "slots must be [tokens, k] in int32 on the rows' device, with k from 1 to ", kMaxChoices);
  TORCH_CHECK_VALUE(like.dim() == 2 && like.size(1) > 0, "x and rows must be [rows, width]");
}

Tensor dispatch(const Tensor& x, const Tensor& slots) {
  refuse_unseen([&](auto f) { f(x); });
  check_floating(x, "x");
  check_slots(slots, x);
  TORCH_CHECK_VALUE(slots.size(0) == x.size(0), "slots must have ", x.size(0), " rows");
  if (at::GradMode::is_enabled() && x.requires_grad()) return DispatchFunction::apply(x, slots);
  return dispatch_rows(x, slots);
}

Tensor combine(const Tensor& rows, const Tensor& slots, const Tensor& weights, const std::optional<Tensor>& residual) {
  refuse_unseen([&](auto f) {
    f(rows);
    f(weights);
    if (residual) f(*residual);
  });
  check_floating(rows, "rows");
  check_slots(slots, rows);
  TORCH_CHECK_VALUE(rows.size(0) == slots.numel(), "rows must be [", slots.numel(), ", width]");
  TORCH_CHECK_VALUE(weights.scalar_type() == at::kFloat && weights.device() == rows.device() &&
                        weights.sizes() == slots.sizes(),
                    "weights must be float32 of shape ", slots.sizes(), " on the rows' device");
  if (residual)
    TORCH_CHECK_VALUE(residual->scalar_type() == rows.scalar_type() && residual->device() == rows.device() &&
                          residual->dim() == 2 && residual->size(0) == slots.size(0) &&
                          residual->size(1) == rows.size(1),
                      "residual must have the rows' type and device and shape [", slots.size(0), ", ", rows.size(1), "]");
  if (at::GradMode::is_enabled() &&
      (rows.requires_grad() || weights.requires_grad() || (residual && residual->requires_grad())))
    return CombineFunction::apply(rows, slots, weights, residual);
  return combine_rows(rows, slots, weights, residual);
}

// ------------------------------------------------------------ embedding

AveyEmbeddingParams embedding_params(const Tensor& like, const Tensor& tokens, int64_t vocab, int64_t width,
                                     double scale, int64_t padding) {
  AveyEmbeddingParams p{};
  p.struct_size = sizeof(p);
  p.dtype = dtype_id(like);
  p.index_bits = tokens.scalar_type() == at::kLong ? 64 : 32;
  p.count = tokens.numel();
  p.width = width;
  p.vocab = vocab;
  p.padding = padding;
  p.scale = scale;
  p.tokens = tokens.const_data_ptr();
  return p;
}

Tensor embedding_forward(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding) {
  const c10::cuda::CUDAGuard guard(weight.device());
  const Tensor t = tokens.contiguous(), w = as_weight(weight);
  AveyEmbeddingParams p = embedding_params(weight, t, weight.size(0), weight.size(1), scale, padding);
  auto shape = tokens.sizes().vec();
  shape.push_back(p.width);
  Tensor out = at::empty(shape, weight.options());
  p.table = w.const_data_ptr();
  p.table_ld = p.vocab > 1 ? w.stride(0) : p.width;
  p.out = out.data_ptr();
  check_status(lib.embedding_fwd(&p, stream_of()));
  return out;
}

class EmbeddingFunction : public torch::autograd::Function<EmbeddingFunction> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& tokens, const Tensor& weight, double scale,
                        int64_t padding) {
    ctx->save_for_backward({tokens});
    ctx->saved_data["call"] = std::vector<int64_t>{weight.size(0), weight.size(1), padding};
    ctx->saved_data["scale"] = scale;
    return embedding_forward(tokens, weight, scale, padding);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "the gradient of the native embedding cannot be differentiated again (create_graph)");
    torch::autograd::variable_list out(4);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    refuse_unseen([&](auto f) { f(dy); });
    const std::vector<int64_t> call = ctx->saved_data["call"].toIntVector();
    const c10::cuda::CUDAGuard guard(dy.device());
    const Tensor t = ctx->get_saved_variables()[0].contiguous(), g = as_rows(dy, call[1]);
    AveyEmbeddingParams p = embedding_params(dy, t, call[0], call[1], ctx->saved_data["scale"].toDouble(), call[2]);
    p.dy = g.const_data_ptr();
    p.dy_ld = row_ld(g, p.width);
    out[1] = at::empty({p.vocab, p.width}, dy.options());
    p.dtable = out[1].data_ptr();
    uint64_t bytes = 0;
    check_status(lib.embedding_workspace(&p, &bytes));
    const Tensor ws = byte_workspace(bytes, dy);
    if (bytes) p.workspace = ws.data_ptr();
    p.workspace_bytes = bytes;
    check_status(lib.embedding_bwd(&p, stream_of()));
    return out;
  }
};

Tensor embedding(const Tensor& tokens, const Tensor& weight, double scale, int64_t padding) {
  refuse_unseen([&](auto f) { f(weight); });
  check_floating(weight, "weight");
  TORCH_CHECK_VALUE(weight.dim() == 2 && weight.numel() > 0, "weight must be [vocab, width]");
  check_integers(tokens, "tokens");
  TORCH_CHECK_VALUE(tokens.device() == weight.device(), "tokens must be on the weight's device");
  TORCH_CHECK_VALUE(padding >= -1 && padding < weight.size(0), "padding_idx must be a token of the vocabulary");
  TORCH_CHECK_VALUE(std::isfinite(scale), "scale must be finite");
  if (at::GradMode::is_enabled() && weight.requires_grad())
    return EmbeddingFunction::apply(tokens, weight, scale, padding);
  return embedding_forward(tokens, weight, scale, padding);
}

// Entry points of the loaded library, by name.
void bind(const py::dict& addresses) {
  auto at = [&](const char* name) { return addresses[name].cast<uintptr_t>(); };
  lib.adamw = reinterpret_cast<decltype(lib.adamw)>(at("avey_adamw_v1"));
  lib.linear_fwd = reinterpret_cast<decltype(lib.linear_fwd)>(at("avey_linear_fwd_v1"));
  lib.linear_bwd = reinterpret_cast<decltype(lib.linear_bwd)>(at("avey_linear_bwd_v1"));
  lib.linear_workspace = reinterpret_cast<decltype(lib.linear_workspace)>(at("avey_linear_workspace_size"));
  lib.loss_fwd = reinterpret_cast<decltype(lib.loss_fwd)>(at("avey_loss_fwd_v1"));
  lib.loss_bwd = reinterpret_cast<decltype(lib.loss_bwd)>(at("avey_loss_bwd_v1"));
  lib.loss_workspace = reinterpret_cast<decltype(lib.loss_workspace)>(at("avey_loss_workspace_size"));
  lib.route_fwd = reinterpret_cast<decltype(lib.route_fwd)>(at("avey_route_fwd_v1"));
  lib.route_bwd = reinterpret_cast<decltype(lib.route_bwd)>(at("avey_route_bwd_v1"));
  lib.arrange = reinterpret_cast<decltype(lib.arrange)>(at("avey_arrange_v1"));
  lib.arrange_workspace = reinterpret_cast<decltype(lib.arrange_workspace)>(at("avey_arrange_workspace_size"));
  lib.dispatch = reinterpret_cast<decltype(lib.dispatch)>(at("avey_dispatch_v1"));
  lib.combine = reinterpret_cast<decltype(lib.combine)>(at("avey_combine_v1"));
  lib.combine_bwd = reinterpret_cast<decltype(lib.combine_bwd)>(at("avey_combine_bwd_v1"));
  lib.rows_workspace = reinterpret_cast<decltype(lib.rows_workspace)>(at("avey_rows_workspace_size"));
  lib.embedding_fwd = reinterpret_cast<decltype(lib.embedding_fwd)>(at("avey_embedding_fwd_v1"));
  lib.embedding_bwd = reinterpret_cast<decltype(lib.embedding_bwd)>(at("avey_embedding_bwd_v1"));
  lib.embedding_workspace = reinterpret_cast<decltype(lib.embedding_workspace)>(at("avey_embedding_workspace_size"));
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at("avey_last_error"));
}

}  // namespace

PYBIND11_MODULE(_torch_binding, m) {
  m.def("bind", &bind);
  m.def("adamw_step", &adamw_step);
  m.def("linear", &linear);
  m.def("cross_entropy", &cross_entropy);
  m.def("route", &route);
  m.def("arrange", &arrange);
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("embedding", &embedding);
}

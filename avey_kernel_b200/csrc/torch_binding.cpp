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
#include <vector>

#include "avey_b200.h"

namespace {

using at::Tensor;

struct Library {
  int (*adamw)(const AveyAdamWParams*, void*) = nullptr;
  int (*linear_fwd)(const AveyLinearParams*, void*) = nullptr;
  int (*linear_bwd)(const AveyLinearParams*, void*) = nullptr;
  int (*linear_workspace)(const AveyLinearParams*, int, uint64_t*) = nullptr;
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

// Entry points of the loaded library, by name.
void bind(const py::dict& addresses) {
  auto at = [&](const char* name) { return addresses[name].cast<uintptr_t>(); };
  lib.adamw = reinterpret_cast<decltype(lib.adamw)>(at("avey_adamw_v1"));
  lib.linear_fwd = reinterpret_cast<decltype(lib.linear_fwd)>(at("avey_linear_fwd_v1"));
  lib.linear_bwd = reinterpret_cast<decltype(lib.linear_bwd)>(at("avey_linear_bwd_v1"));
  lib.linear_workspace = reinterpret_cast<decltype(lib.linear_workspace)>(at("avey_linear_workspace_size"));
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at("avey_last_error"));
}

}  // namespace

PYBIND11_MODULE(_torch_binding, m) {
  m.def("bind", &bind);
  m.def("adamw_step", &adamw_step);
  m.def("linear", &linear);
}

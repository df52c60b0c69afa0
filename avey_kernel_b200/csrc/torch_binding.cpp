// Python binding of the training and serving operators: checks PyTorch tensors,
// fills the C ABI's parameter blocks (include/avey_b200.h) and calls the library
// on the tensors' device and its current stream. Host code only; the library's
// entry points are handed over by bind() (avey_kernel_b200/_binding.py), so that
// there is one loaded library in a process. Bad arguments raise ValueError;
// a non-OK AveyStatus is returned and raised by the Python side.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/extension.h>

#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <vector>

#include "avey_b200.h"

namespace {

using at::Tensor;

struct Library {
  int (*adamw)(const AveyAdamWParams*, void*) = nullptr;
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
  return lib.adamw(&a, at::cuda::getCurrentCUDAStream().stream());
}

// Entry points of the loaded library, by name.
void bind(const py::dict& addresses) {
  auto at = [&](const char* name) { return addresses[name].cast<uintptr_t>(); };
  lib.adamw = reinterpret_cast<decltype(lib.adamw)>(at("avey_adamw_v1"));
}

}  // namespace

PYBIND11_MODULE(_torch_binding, m) {
  m.def("bind", &bind);
  m.def("adamw_step", &adamw_step);
}

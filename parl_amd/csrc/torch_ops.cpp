// torch_ops.cpp — the operators over logits and gradients as torch functions (module parl_amd._torch_ops).
//
// What ops.py does for most entries of the C ABI in Python — check the arguments, allocate the results, hand out pointers —
// costs tens of microseconds a call where there is an autograd node to build (a Python backward pass takes the
// interpreter in the engine's thread) or a few hundred tensors to look at: more than the kernels behind it.  Here it is
// C++: no computation, only the same checks and the same entries of libparl_hip.so, whose addresses bind() is given (so
// that PARL_HIP_LIB goes for these too).  Every refusal of a call is a ParlHipError; what fails in a backward pass is the
// RuntimeError that the autograd engine makes of it.
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <ATen/ops/zeros.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <sstream>
#include <vector>

#include "../../include/parl_hip.h"

namespace py = pybind11;
using at::Tensor;

namespace {

struct Entries {
  decltype(&parlhip_strerror) strerror;
  decltype(&parlhip_last_hip_error) last_hip_error;
  decltype(&parlhip_logits_sample_workspace_bytes) sample_workspace;
  decltype(&parlhip_logits_sample) sample;
  decltype(&parlhip_logits_log_prob_workspace_bytes) log_prob_workspace;
  decltype(&parlhip_logits_log_prob) log_prob;
  decltype(&parlhip_logits_log_prob_backward) log_prob_backward;
  decltype(&parlhip_grad_norm_workspace_bytes) norm_workspace;
  decltype(&parlhip_grad_norm) norm;
  decltype(&parlhip_clip_grad_norm) clip;
} lib;

PyObject* error_type = nullptr;   // parl_amd._native.ParlHipError

struct Refused : std::runtime_error {
  using std::runtime_error::runtime_error;
};

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw Refused(s.str());
}

void check(int code, const char* what) {
  if (code < 0)
    refuse(what, " failed: ", lib.strerror(code), " (code ", code, ", hip error ", lib.last_hip_error(), ")");
}

int type_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PARLHIP_F32;
    case at::kBFloat16: return PARLHIP_BF16;
    case at::kHalf: return PARLHIP_F16;
    default: return -1;
  }
}

// torch's current stream of the device
void* stream_of(const c10::Device& d) {
  const c10::Stream s = c10::impl::VirtualGuardImpl(d.type()).getStream(d);
  return (void*)c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, s).stream();
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void check_logits(const Tensor& t, const char* name) {
  if (type_code(t) < 0 || t.layout() != at::kStrided)
    refuse(name, ": logits must be float32, bfloat16 or float16, got ", t.scalar_type());
  if (t.dim() < 1 || t.size(-1) < 1) refuse(name, ": logits must be [..., A] with at least one action, got ", t.sizes());
  if (!t.is_cuda())
    refuse(name, " needs device (HIP) tensors; got a ", t.device(), " tensor. There is no CPU fallback.");
}

struct Rows {
  Tensor x;   // [n, a], elements of a row adjacent
  int64_t n, a, stride;
};

// Rows of a wider buffer (a padded action set) are read in place, anything else is laid out first.
Rows rows_of(const Tensor& logits) {
  Rows r;
  r.a = logits.size(-1);
  r.n = logits.numel() / r.a;
  r.x = logits.detach().resolve_neg();
  if (r.x.dim() != 2) r.x = r.x.reshape({r.n, r.a});
  r.stride = r.n > 1 ? r.x.stride(0) : r.a;
  if (r.stride < r.a || (r.a > 1 && r.x.stride(1) != 1)) {
    r.x = r.x.contiguous();
    r.stride = r.a;
  }
  return r;
}

Tensor per_row(const Tensor& t, at::ScalarType dtype, const Tensor& logits, const char* what, const char* name) {
  if (t.scalar_type() != dtype) refuse(name, ": ", what, " must be ", dtype, ", got ", t.scalar_type());
  if (t.device() != logits.device()) refuse(name, ": ", what, " is on ", t.device(), ", logits on ", logits.device());
  const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
  if (t.sizes() != lead) refuse(name, ": ", what, " must have the shape ", lead, ", got ", t.sizes());
  return t.detach().resolve_neg().contiguous();
}

Tensor unpack(const py::handle& h, const char* what, const char* name) {
  if (!THPVariable_Check(h.ptr())) refuse(name, ": ", what, " must be a tensor, got ", Py_TYPE(h.ptr())->tp_name);
  return THPVariable_Unpack(h.ptr());
}

double number(const py::handle& h, const char* what, const char* name) {
  const double v = PyFloat_AsDouble(h.ptr());
  if (v == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    refuse(name, ": ", what, " must be a number or a tensor, got ", Py_TYPE(h.ptr())->tp_name);
  }
  return v;
}

py::tuple logits_sample(const py::handle& logits_, const py::handle& uniforms_, const py::handle& temperature,
                        const py::handle& top_k, const py::handle& top_p, const py::handle& min_p) {
  const char* name = "logits_sample";
  const Tensor logits = unpack(logits_, "logits", name);
  check_logits(logits, name);
  const Tensor u = per_row(unpack(uniforms_, "uniforms", name), at::kDouble, logits, "uniforms", name);
  Tensor t, k, p, m;
  double tv = 1.0, pv = 1.0, mv = 0.0;
  Py_ssize_t kv = 0;
  if (THPVariable_Check(temperature.ptr())) {
    t = per_row(THPVariable_Unpack(temperature.ptr()), at::kFloat, logits, "temperature", name);
  } else if (tv = number(temperature, "temperature", name); !(tv >= 0.0) || std::isinf((float)tv)) {
    refuse(name, ": temperature must be a finite float32 >= 0, got ", tv);
  }
  if (THPVariable_Check(top_k.ptr())) {
    k = per_row(THPVariable_Unpack(top_k.ptr()), at::kInt, logits, "top_k", name);
  } else {
    kv = PyIndex_Check(top_k.ptr()) ? PyNumber_AsSsize_t(top_k.ptr(), PyExc_OverflowError) : -2;
    const bool wrong = PyErr_Occurred() || !PyIndex_Check(top_k.ptr()) || kv < INT32_MIN || kv > INT32_MAX;
    PyErr_Clear();
    if (wrong) refuse(name, ": top_k must be a whole number of 32 bits or a tensor");
  }
  if (THPVariable_Check(top_p.ptr())) {
    p = per_row(THPVariable_Unpack(top_p.ptr()), at::kFloat, logits, "top_p", name);
  } else if (pv = number(top_p, "top_p", name); !(pv >= 0.0)) {
    refuse(name, ": top_p must be >= 0, got ", pv);
  }
  if (THPVariable_Check(min_p.ptr())) {
    m = per_row(THPVariable_Unpack(min_p.ptr()), at::kFloat, logits, "min_p", name);
  } else if (mv = number(min_p, "min_p", name); !(mv >= 0.0 && mv <= 1.0)) {
    refuse(name, ": min_p must be in [0, 1], got ", mv);
  }
  Tensor actions, log_probs;
  {
    py::gil_scoped_release free;
    const c10::DeviceGuard guard(logits.device());
    const Rows r = rows_of(logits);
    const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
    const auto opt = at::TensorOptions().device(logits.device());
    actions = at::empty(lead, opt.dtype(at::kLong));
    log_probs = at::empty(lead, opt.dtype(at::kFloat));
    const size_t bytes = lib.sample_workspace(r.n, r.a);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)(bytes + 7) / 8}, opt.dtype(at::kDouble));
    check(lib.sample(data(r.x), type_code(logits), r.stride, (const double*)data(u), (const float*)data(t),
                     (const int32_t*)data(k), (const float*)data(p), (const float*)data(m), (float)tv, (int32_t)kv, (float)pv,
                     (float)mv, (int64_t*)data(actions), (float*)data(log_probs), r.n, r.a, data(ws), bytes,
                     stream_of(logits.device())),
          "parlhip_logits_sample");
  }
  return py::make_tuple(actions, log_probs);
}

struct LogProbFn : torch::autograd::Function<LogProbFn> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& logits,
                                                const Tensor& actions, double temperature) {
    const c10::DeviceGuard guard(logits.device());
    const Rows r = rows_of(logits);
    const at::IntArrayRef lead = logits.sizes().slice(0, logits.dim() - 1);
    const auto opt = at::TensorOptions().device(logits.device()).dtype(at::kFloat);
    const Tensor log_probs = at::empty(lead, opt), entropies = at::empty(lead, opt);
    const Tensor stats = at::empty({r.n, 2}, opt);
    const size_t bytes = lib.log_prob_workspace(r.n, r.a);
    Tensor ws;
    if (bytes) ws = at::empty({(int64_t)(bytes + 3) / 4}, opt);
    check(lib.log_prob(data(r.x), type_code(logits), r.stride, (const int64_t*)data(actions), (float*)data(log_probs),
                       (float*)data(entropies), (float*)data(stats), r.n, r.a, (float)temperature, data(ws), bytes,
                       stream_of(logits.device())),
          "parlhip_logits_log_prob");
    ctx->save_for_backward({logits, actions, stats, entropies});
    ctx->saved_data["temperature"] = temperature;
    ctx->set_materialize_grads(false);
    return {log_probs, entropies};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list g) {
    if (!g[0].defined() && !g[1].defined()) return {Tensor(), Tensor(), Tensor()};
    TORCH_CHECK(!at::GradMode::is_enabled(), "logits_log_prob: the gradient is not differentiable again");
    const auto saved = ctx->get_saved_variables();
    const Tensor &logits = saved[0], &actions = saved[1], &stats = saved[2], &entropies = saved[3];
    const c10::DeviceGuard guard(logits.device());
    const Rows r = rows_of(logits);
    for (Tensor& t : g)
      if (t.defined()) t = t.to(at::kFloat).resolve_neg().contiguous();
    const Tensor grad = at::empty(logits.sizes(), logits.options());
    check(lib.log_prob_backward(data(r.x), type_code(logits), r.stride, (const int64_t*)data(actions),
                                (const float*)data(stats), (const float*)data(entropies), (const float*)data(g[0]),
                                (const float*)data(g[1]), data(grad), r.n, r.a,
                                (float)ctx->saved_data["temperature"].toDouble(), stream_of(logits.device())),
          "parlhip_logits_log_prob_backward");
    return {grad, Tensor(), Tensor()};
  }
};

py::tuple logits_log_prob(const py::handle& logits_, const py::handle& actions_, const py::handle& temperature) {
  const char* name = "logits_log_prob";
  const Tensor logits = unpack(logits_, "logits", name);
  check_logits(logits, name);
  const Tensor actions = per_row(unpack(actions_, "actions", name), at::kLong, logits, "actions", name);
  if (THPVariable_Check(temperature.ptr()) && THPVariable_Unpack(temperature.ptr()).numel() != 1)
    refuse(name, ": temperature must be one number for all rows; for one of each row's own divide the logits by it first");
  const double t = number(temperature, "temperature", name);
  if (!(t > 0.0) || std::isinf((float)t)) refuse(name, ": temperature must be a finite float32 > 0, got ", t);
  torch::autograd::variable_list out;
  {
    py::gil_scoped_release free;
    out = LogProbFn::apply(logits, actions, t);
  }
  return py::make_tuple(out[0], out[1]);
}

struct Table {
  std::vector<Tensor> keep;
  std::vector<void*> at;
  std::vector<int64_t> numel;
  std::vector<int32_t> types;
  c10::optional<c10::Device> device;

  void add(const Tensor& t, const char* name) {
    const int code = t.layout() == at::kStrided ? type_code(t) : -1;
    if (code < 0)
      refuse(name, ": needs dense float32, bfloat16 or float16 tensors, got ", t.layout(), " ", t.scalar_type());
    if (!t.is_cuda() || (device && t.device() != *device))
      refuse(name, ": the tensors must be on one HIP device, got ", t.device());
    if (t.is_neg()) refuse(name, ": a lazily negated view has no values in memory to read or write");
    if (!t.is_non_overlapping_and_dense())
      refuse(name, ": a tensor of shape ", t.sizes(), " and strides ", t.strides(), " does not fill its memory");
    device = t.device();
    keep.push_back(t);
    at.push_back(t.data_ptr());
    numel.push_back(t.numel());
    types.push_back(code);
  }
  int n() const { return (int)keep.size(); }
  c10::Device where() const {
    return device ? *device : c10::impl::VirtualGuardImpl(c10::DeviceType::CUDA).getDevice();
  }
};

template <typename F>
void each_tensor(const py::handle& h, const char* what, const char* name, F&& f) {
  if (THPVariable_Check(h.ptr())) return f(THPVariable_Unpack(h.ptr()));
  for (const py::handle& item : py::reinterpret_borrow<py::object>(h)) f(unpack(item, what, name));
}

Tensor run_norm(const Table& g) {
  const c10::DeviceGuard guard(g.where());
  const auto opt = at::TensorOptions().device(g.where());
  const Tensor norm = at::empty({}, opt.dtype(at::kFloat));
  const size_t bytes = lib.norm_workspace(g.n(), g.numel.data());
  const Tensor ws = at::empty({(int64_t)(bytes + 7) / 8}, opt.dtype(at::kDouble));
  check(lib.norm(g.n(), g.at.data(), g.numel.data(), g.types.data(), data(ws), bytes, (float*)data(norm),
                 stream_of(g.where())),
        "parlhip_grad_norm");
  return norm;
}

Tensor grad_norm(const py::handle& tensors) {
  Table g;
  each_tensor(tensors, "an element of tensors", "grad_norm", [&](const Tensor& t) { g.add(t, "grad_norm"); });
  return run_norm(g);
}

void written(const Tensor& t) {   // through a raw pointer: what autograd saved of it is no longer there
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

Tensor clip_grad_norm(const py::handle& parameters, double max_norm, bool error_if_nonfinite, const py::handle& out_) {
  const char* name = "clip_grad_norm_";
  if (!(max_norm >= 0.0)) refuse(name, ": max_norm must be >= 0, got ", max_norm);
  Table g, out;
  each_tensor(parameters, "a parameter", name, [&](const Tensor& p) {
    const Tensor& grad = p.grad();
    if (grad.defined()) g.add(grad, name);
  });
  const bool apart = !out_.is_none();
  if (apart) {
    each_tensor(out_, "an element of out", name, [&](const Tensor& t) { out.add(t, name); });
    if (out.n() != g.n()) refuse(name, ": out has ", out.n(), " tensors for ", g.n(), " gradients");
    for (int i = 0; i < g.n(); ++i) {
      const Tensor &a = g.keep[i], &b = out.keep[i];
      if (a.device() != b.device() || a.sizes() != b.sizes() ||
          !(a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous())))
        refuse(name, ": an out of shape ", b.sizes(), ", strides ", b.strides(), " on ", b.device(),
               " for a gradient of shape ", a.sizes(), ", strides ", a.strides(), " on ", a.device());
    }
  }
  if (error_if_nonfinite) {
    double norm;
    {
      py::gil_scoped_release free;   // waits for the device
      norm = run_norm(g).item<double>();
    }
    if (!std::isfinite(norm)) {
      std::ostringstream s;
      s << name << ": the global norm of the gradients is " << norm << "; they are unchanged";
      throw std::runtime_error(s.str());
    }
  }
  const c10::DeviceGuard guard(g.where());
  const auto opt = at::TensorOptions().device(g.where());
  const Tensor norm = at::empty({}, opt.dtype(at::kFloat));
  const size_t bytes = lib.norm_workspace(g.n(), g.numel.data());
  const Tensor ws = at::empty({(int64_t)(bytes + 7) / 8}, opt.dtype(at::kDouble));
  check(lib.clip(g.n(), g.at.data(), apart ? out.at.data() : nullptr, g.numel.data(), g.types.data(),
                 apart ? out.types.data() : nullptr, max_norm, data(ws), bytes, (float*)data(norm), stream_of(g.where())),
        "parlhip_clip_grad_norm");
  for (const Tensor& t : apart ? out.keep : g.keep) written(t);
  return norm;
}

void bind(const py::object& error, const py::dict& address) {
  error_type = error.ptr();
  Py_INCREF(error_type);
  const auto set = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(address[name].cast<uintptr_t>());
  };
  set(lib.strerror, "parlhip_strerror");
  set(lib.last_hip_error, "parlhip_last_hip_error");
  set(lib.sample_workspace, "parlhip_logits_sample_workspace_bytes");
  set(lib.sample, "parlhip_logits_sample");
  set(lib.log_prob_workspace, "parlhip_logits_log_prob_workspace_bytes");
  set(lib.log_prob, "parlhip_logits_log_prob");
  set(lib.log_prob_backward, "parlhip_logits_log_prob_backward");
  set(lib.norm_workspace, "parlhip_grad_norm_workspace_bytes");
  set(lib.norm, "parlhip_grad_norm");
  set(lib.clip, "parlhip_clip_grad_norm");
}

// torch's own errors (out of memory) keep their types; refusals are ParlHipErrors
template <typename F, typename... A>
py::object guarded(F f, const A&... a) {
  try {
    if constexpr (std::is_same_v<decltype(f(a...)), Tensor>) return py::cast(f(a...));
    else return f(a...);
  } catch (const Refused& e) {
    PyErr_SetString(error_type, e.what());
    throw py::error_already_set();
  } catch (const py::error_already_set&) {
    throw;
  } catch (const c10::Error& e) {
    torch::PyWarningHandler handler;
    torch::translate_exception_to_python(std::current_exception());
    throw py::error_already_set();
  }
}

}  // namespace

PYBIND11_MODULE(_torch_ops, m) {
  m.def("bind", &bind);
  m.def("source_hash", [] { return PARL_SOURCE_HASH; });   // of what it was built from (srchash.py)
  m.def("logits_sample", [](py::handle a, py::handle b, py::handle c, py::handle d, py::handle e, py::handle f) {
    return guarded(logits_sample, a, b, c, d, e, f);
  });
  m.def("logits_log_prob", [](py::handle a, py::handle b, py::handle c) { return guarded(logits_log_prob, a, b, c); });
  m.def("grad_norm", [](py::handle a) { return guarded(grad_norm, a); });
  m.def("clip_grad_norm", [](py::handle a, double b, bool c, py::handle d) { return guarded(clip_grad_norm, a, b, c, d); });
}

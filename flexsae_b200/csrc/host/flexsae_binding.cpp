// Python binding of the optimizer entry points: checks the tensor lists of a call, collects their
// addresses and calls the C ABI, in C++ because a step over a small model is shorter than the
// interpreter needs for that (20 tensors: 100 us in Python for 40 us on the GPU).
//
// The C ABI itself lives in the library that flexsae_b200/_native.py loads; init() is handed its entry
// points, so that whichever library was loaded is the one that is called.
#include <torch/csrc/python_headers.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <ATen/ops/empty_like.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/util/SmallVector.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/object_ptr.h>

#include <cmath>
#include <limits>
#include <sstream>

#include "../../../include/flexsae_b200.h"

namespace {

struct Entries {
  decltype(&flexsae_adamw_step) adamw = nullptr;
  decltype(&flexsae_adamw_unit_rows_step) unit_rows = nullptr;
  decltype(&flexsae_grad_norm) grad_norm = nullptr;
  decltype(&flexsae_grad_norm_workspace_bytes) grad_norm_workspace = nullptr;
  decltype(&flexsae_last_error) last_error = nullptr;
  decltype(&flexsae_last_launch_count) launches = nullptr;
  PyObject* error = nullptr;      // the exception for calls that the library refuses
} g;

constexpr int64_t kBlock = 256;   // elements that share a scale

// An exception to be raised in Python.
struct Refusal {
  PyObject* type;
  std::string text;
};

template <typename... Args>
[[noreturn]] void refuse(PyObject* type, const Args&... args) {
  std::ostringstream s;
  (s << ... << args);
  throw Refusal{type, s.str()};
}

// A list, tuple or other sequence of tensors (None allowed where asked for: an undefined tensor).  It holds
// references of its own, since another thread may change the sequence while a call has let go of the interpreter.
struct List {
  c10::SmallVector<at::Tensor, 24> t;

  void read(PyObject* o, const char* name, bool may_be_none = false) {
    const THPObjectPtr fast(PySequence_Fast(o, "expected a sequence of tensors"));
    if (!fast) throw Refusal{nullptr, {}};
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(fast.get());
    t.reserve(n);
    for (Py_ssize_t i = 0; i < n; i++) {
      PyObject* x = PySequence_Fast_GET_ITEM(fast.get(), i);
      if (may_be_none && x == Py_None) {
        t.emplace_back();
      } else {
        if (!THPVariable_Check(x)) refuse(PyExc_TypeError, name, " must hold tensors, got ", Py_TYPE(x)->tp_name);
        t.push_back(THPVariable_Unpack(x));
      }
    }
  }
  size_t size() const { return t.size(); }
  const at::Tensor& operator[](size_t i) const { return t[i]; }
};

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? FLEXSAE_F32 : t == at::kBFloat16 ? FLEXSAE_BF16 : t == at::kHalf ? FLEXSAE_F16 : -1;
}

bool same_layout(const at::Tensor& a, const at::Tensor& b) {
  if (a.numel() == 0) return true;
  for (int64_t d = 0; d < a.dim(); d++)
    if (a.size(d) != 1 && a.stride(d) != b.stride(d)) return false;
  return true;
}

bool dense(const at::Tensor& t) { return t.numel() == 0 || t.is_contiguous() || t.unsafeGetTensorImpl()->is_non_overlapping_and_dense(); }

// A view that stands for the negated values of its memory is not what a kernel would read.
void check_as_stored(const char* name, const at::Tensor& t) {
  if (t.is_neg()) refuse(PyExc_ValueError, name, " must not be a lazily negated view");
}

void check_one(const char* name, const at::Tensor& t, const at::Tensor& p, at::ScalarType type) {
  if (t.scalar_type() != type) refuse(PyExc_TypeError, name, " must be ", type, ", got ", t.scalar_type());
  if (t.device() != p.device()) refuse(PyExc_RuntimeError, "a tensor in ", name, " is on ", t.device(), ", the parameters are on ", p.device());
  if (!t.sizes().equals(p.sizes()) || !same_layout(t, p))
    refuse(PyExc_ValueError, "a tensor in ", name, " has shape ", t.sizes(), " and strides ", t.strides(), ", its parameter ", p.sizes(), " and ", p.strides());
  check_as_stored(name, t);
}

void check_count(const char* name, const List& list, const List& params) {
  if (list.size() != params.size()) refuse(PyExc_ValueError, list.size(), " tensors in ", name, ", ", params.size(), " parameters");
}

void check_scales(const char* name, const at::Tensor& t, const at::Tensor& p) {
  const int64_t blocks = (p.numel() + kBlock - 1) / kBlock;
  if (t.scalar_type() != at::kFloat) refuse(PyExc_TypeError, name, " must be Float, got ", t.scalar_type());
  if (t.device() != p.device()) refuse(PyExc_RuntimeError, "a tensor in ", name, " is on ", t.device(), ", the parameters are on ", p.device());
  if (t.dim() != 1 || t.size(0) != blocks || !t.is_contiguous())
    refuse(PyExc_ValueError, name, " of ", p.numel(), " elements is contiguous float32 [", blocks, "], got ", t.sizes());
  check_as_stored(name, t);
}

// A number on the device.
const at::Tensor& word(const char* name, PyObject* o, at::ScalarType type, const at::Device& dev) {
  if (!THPVariable_Check(o) || THPVariable_Unpack(o).numel() != 1) refuse(PyExc_ValueError, name, " must be a tensor of one element");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (t.scalar_type() != type) refuse(PyExc_TypeError, name, " must be ", type, ", got ", t.scalar_type());
  if (t.device() != dev) refuse(PyExc_RuntimeError, name, " is on ", t.device(), ", the parameters are on ", dev);
  check_as_stored(name, t);
  return t;
}

double number(const char* name, PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw Refusal{nullptr, {}};
  return x;
}

void at_least(const char* name, double x, double least) {
  if (!(std::isfinite(x) && x >= least)) refuse(PyExc_ValueError, name, " must be a finite number >= ", least, ", got ", x);
}

// Autograd's saved copies of a tensor that was written are out of date.
void written(const at::Tensor& t) {
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

enum Kind { kAdamw = 0, kAdamw8 = 1, kUnitRows = 2 };

// step(kind, params, grads, exp_avgs, exp_avg_scales, exp_avg_sqs, exp_avg_sq_scales, masters, step, lr, betas, eps,
//      weight_decay, norm, max_norm, seed) -> launches
long run_step(PyObject* const* a) {
  const long kind = PyLong_AsLong(a[0]);
  List params, grads, m, ms, v, vs, masters;
  params.read(a[1], "params");
  grads.read(a[2], "grads");
  m.read(a[3], "exp_avgs");
  v.read(a[5], "exp_avg_sqs");
  const size_t n = params.size();
  if (n == 0) refuse(PyExc_ValueError, "no parameters");
  if (grads.size() != n) refuse(PyExc_ValueError, grads.size(), " gradients, ", n, " parameters");
  const at::Device dev = params[0].device();
  if (!dev.is_cuda()) refuse(PyExc_RuntimeError, "flexsae_b200.optim needs CUDA tensors: there is no CPU path");
  check_count("exp_avgs", m, params);
  check_count("exp_avg_sqs", v, params);
  if (kind == kAdamw8) {
    ms.read(a[4], "exp_avg_scales");
    vs.read(a[6], "exp_avg_sq_scales");
    check_count("exp_avg_scales", ms, params);
    check_count("exp_avg_sq_scales", vs, params);
  }
  const bool with_masters = a[7] != Py_None;
  if (with_masters) {
    masters.read(a[7], "masters", true);
    if (masters.size() != n) refuse(PyExc_ValueError, masters.size(), " masters, ", n, " parameters");
  }
  const c10::cuda::CUDAGuard guard(dev);
  const at::ScalarType type_m = kind == kAdamw8 ? at::kFloat8_e4m3fn : at::kFloat, type_v = kind == kAdamw8 ? at::kFloat8_e5m2 : at::kFloat;
  c10::SmallVector<flexsae_optim_tensor, 24> table(n);
  c10::SmallVector<at::Tensor, 4> copies;     // gradients brought into their parameters' layout
  for (size_t i = 0; i < n; i++) {
    const at::Tensor &p = params[i], &grad = grads[i];
    if (dtype_code(p.scalar_type()) < 0) refuse(PyExc_TypeError, "parameters must be float32, bfloat16 or float16, got ", p.scalar_type());
    if (grad.layout() != at::kStrided) refuse(PyExc_TypeError, "gradients must be dense tensors, got ", grad.layout());
    if (p.layout() != at::kStrided) refuse(PyExc_TypeError, "parameters must be dense tensors, got ", p.layout());
    if (grad.scalar_type() != p.scalar_type() && grad.scalar_type() != at::kFloat)
      refuse(PyExc_TypeError, "the gradient of a ", p.scalar_type(), " parameter must have its type or be Float, got ", grad.scalar_type());
    if (p.device() != dev || grad.device() != dev)
      refuse(PyExc_RuntimeError, "parameters and gradients must be on one device, got ", p.device(), " and ", grad.device(), " beside ", dev);
    if (!grad.sizes().equals(p.sizes())) refuse(PyExc_ValueError, "a gradient has shape ", grad.sizes(), ", its parameter ", p.sizes());
    if (!dense(p)) refuse(PyExc_ValueError, "a parameter of shape ", p.sizes(), " with strides ", p.strides(), " does not fill its memory");
    check_as_stored("params", p);
    if (kind == kUnitRows && (p.dim() != 2 || !p.is_contiguous()))
      refuse(PyExc_ValueError, "unit rows need a contiguous [F, D] parameter, got ", p.sizes(), " with strides ", p.strides());
    check_one("exp_avgs", m[i], p, type_m);
    check_one("exp_avg_sqs", v[i], p, type_v);
    if (kind == kAdamw8) {
      check_scales("exp_avg_scales", ms[i], p);
      check_scales("exp_avg_sq_scales", vs[i], p);
    }
    if (with_masters && masters[i].defined()) {
      if (p.scalar_type() == at::kFloat) refuse(PyExc_ValueError, "masters go with 16-bit parameters only");
      check_one("masters", masters[i], p, at::kFloat);
    }
  }
  const at::Tensor& step = word("step", a[8], at::kLong, dev);
  const bool lr_on_device = THPVariable_Check(a[9]);
  const float* lr_device = lr_on_device ? word("lr", a[9], at::kFloat, dev).const_data_ptr<float>() : nullptr;
  const double lr = lr_on_device ? 0.0 : number("lr", a[9]);
  at_least("lr", lr, 0.0);
  if (!PyTuple_Check(a[10]) || PyTuple_GET_SIZE(a[10]) != 2) refuse(PyExc_ValueError, "betas must be a pair of numbers");
  const double b1 = number("betas", PyTuple_GET_ITEM(a[10], 0)), b2 = number("betas", PyTuple_GET_ITEM(a[10], 1));
  if (!(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1)) refuse(PyExc_ValueError, "betas must be in [0, 1), got ", b1, ", ", b2);
  const double eps = number("eps", a[11]), decay = number("weight_decay", a[12]);
  at_least("eps", eps, std::numeric_limits<float>::min());
  at_least("weight_decay", decay, 0.0);
  const float* norm = a[13] == Py_None ? nullptr : word("norm", a[13], at::kFloat, dev).const_data_ptr<float>();
  double max_norm = std::numeric_limits<double>::infinity();
  if (a[14] != Py_None) {
    max_norm = number("max_norm", a[14]);
    if (!norm || !(max_norm > 0)) refuse(PyExc_ValueError, "max_norm must be positive and goes with norm");
  }
  const long long seed = PyLong_AsLongLong(a[15]);
  if (PyErr_Occurred()) PyErr_Clear(), refuse(PyExc_ValueError, "seed must be a whole number in [0, 2**32)");
  if (seed < 0 || seed >= (1ll << 32)) refuse(PyExc_ValueError, "seed must be in [0, 2**32), got ", seed);
  // Everything is checked; from here on memory is touched.
  for (size_t i = 0; i < n; i++) {
    const at::Tensor& p = params[i];
    const at::Tensor* grad = &grads[i];
    if (!same_layout(*grad, p) || grad->is_neg()) {
      copies.push_back(at::empty_like(p, p.options().dtype(grad->scalar_type()).requires_grad(false)).copy_(grad->detach()));
      grad = &copies.back();
    }
    flexsae_optim_tensor& d = table[i];
    d.param = p.mutable_data_ptr();
    d.grad = grad->const_data_ptr();
    d.exp_avg = m[i].mutable_data_ptr();
    d.exp_avg_sq = v[i].mutable_data_ptr();
    d.exp_avg_scale = kind == kAdamw8 ? ms[i].mutable_data_ptr<float>() : nullptr;
    d.exp_avg_sq_scale = kind == kAdamw8 ? vs[i].mutable_data_ptr<float>() : nullptr;
    d.master = with_masters && masters[i].defined() ? masters[i].mutable_data_ptr<float>() : nullptr;
    d.numel = p.numel();
    d.cols = kind == kUnitRows ? p.size(1) : 0;
    d.param_dtype = dtype_code(p.scalar_type());
    d.grad_dtype = dtype_code(grad->scalar_type());
  }
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  int64_t* count = step.mutable_data_ptr<int64_t>();
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = kind == kUnitRows ? g.unit_rows(table.data(), (int64_t)n, count, lr, lr_device, b1, b2, eps, decay, norm, max_norm, stream)
                         : g.adamw(table.data(), (int64_t)n, kind == kAdamw8 ? 8 : 32, count, lr, lr_device, b1, b2, eps, decay, norm, max_norm,
                                   (uint32_t)seed, stream);
  Py_END_ALLOW_THREADS
  if (rc) refuse(g.error, kind == kUnitRows ? "flexsae_adamw_unit_rows_step" : "flexsae_adamw_step", " failed (code ", rc, "): ", g.last_error());
  for (size_t i = 0; i < n; i++) {
    written(params[i]);
    written(m[i]);
    written(v[i]);
    if (kind == kAdamw8) written(ms[i]), written(vs[i]);
    if (with_masters && masters[i].defined()) written(masters[i]);
  }
  written(step);
  return g.launches();
}

// grad_norm(grads) -> (norm, launches)
at::Tensor run_norm(PyObject* o, long* launches) {
  List grads;
  grads.read(o, "grads");
  const size_t n = grads.size();
  if (n == 0) refuse(PyExc_ValueError, "no gradients");
  const at::Device dev = grads[0].device();
  if (!dev.is_cuda()) refuse(PyExc_RuntimeError, "flexsae_b200.optim needs CUDA tensors: there is no CPU path");
  c10::SmallVector<const void*, 24> at_(n);
  c10::SmallVector<int64_t, 24> numel(n);
  c10::SmallVector<int32_t, 24> types(n);
  c10::SmallVector<at::Tensor, 4> copies;
  const c10::cuda::CUDAGuard guard(dev);
  for (size_t i = 0; i < n; i++) {
    const at::Tensor& x = grads[i];
    if (x.layout() != at::kStrided) refuse(PyExc_TypeError, "gradients must be dense tensors, got ", x.layout());
    types[i] = dtype_code(x.scalar_type());
    if (types[i] < 0) refuse(PyExc_TypeError, "gradients must be float32, bfloat16 or float16, got ", x.scalar_type());
    if (x.device() != dev) refuse(PyExc_RuntimeError, "gradients must be on one device, got ", x.device(), " beside ", dev);
  }
  int64_t elements = 0;
  for (size_t i = 0; i < n; i++) {
    const at::Tensor* x = &grads[i];
    if (!dense(*x)) {
      copies.push_back(x->detach().contiguous());
      x = &copies.back();
    }
    at_[i] = x->const_data_ptr();
    numel[i] = x->numel();
    elements += numel[i];
  }
  const at::TensorOptions options = at::TensorOptions().device(dev);
  at::Tensor norm = at::empty({}, options.dtype(at::kFloat));
  size_t need = 0;
  if (const int rc = g.grad_norm_workspace((int64_t)n, elements, &need))
    refuse(g.error, "flexsae_grad_norm failed (code ", rc, "): ", g.last_error());
  at::Tensor ws;
  if (need) ws = at::empty({(int64_t)need}, options.dtype(at::kByte));
  void* stream = c10::cuda::getCurrentCUDAStream(dev.index()).stream();
  float* out = norm.mutable_data_ptr<float>();
  void* scratch = need ? ws.mutable_data_ptr() : nullptr;
  int rc = 0;
  Py_BEGIN_ALLOW_THREADS
  rc = g.grad_norm(at_.data(), numel.data(), types.data(), (int64_t)n, out, scratch, need, stream);
  Py_END_ALLOW_THREADS
  if (rc) refuse(g.error, "flexsae_grad_norm failed (code ", rc, "): ", g.last_error());
  *launches = g.launches();
  return norm;
}

PyObject* raise(const Refusal& r) {
  if (r.type) PyErr_SetString(r.type, r.text.c_str());      // without one, Python's own error is set
  return nullptr;
}

PyObject* py_step(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 16) return PyErr_Format(PyExc_TypeError, "step takes 16 arguments, got %zd", n);
  try {
    return PyLong_FromLong(run_step(args));
  } catch (const Refusal& r) {
    return raise(r);
  }
  END_HANDLE_TH_ERRORS
}

PyObject* py_norm(PyObject*, PyObject* grads) {
  HANDLE_TH_ERRORS
  try {
    long launches = 0;
    at::Tensor norm = run_norm(grads, &launches);
    PyObject* t = THPVariable_Wrap(std::move(norm));
    return t ? Py_BuildValue("(Nl)", t, launches) : nullptr;
  } catch (const Refusal& r) {
    return raise(r);
  }
  END_HANDLE_TH_ERRORS
}

// init(error class, addresses of the six entry points)
PyObject* py_init(PyObject*, PyObject* args) {
  PyObject* error;
  unsigned long long a, b, c, d, e, f;
  if (!PyArg_ParseTuple(args, "OKKKKKK", &error, &a, &b, &c, &d, &e, &f)) return nullptr;
  Py_INCREF(error);
  Py_XDECREF(g.error);
  g.error = error;
  g.adamw = reinterpret_cast<decltype(g.adamw)>(a);
  g.unit_rows = reinterpret_cast<decltype(g.unit_rows)>(b);
  g.grad_norm = reinterpret_cast<decltype(g.grad_norm)>(c);
  g.grad_norm_workspace = reinterpret_cast<decltype(g.grad_norm_workspace)>(d);
  g.last_error = reinterpret_cast<decltype(g.last_error)>(e);
  g.launches = reinterpret_cast<decltype(g.launches)>(f);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"init", py_init, METH_VARARGS, nullptr},
    {"step", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_step)), METH_FASTCALL, nullptr},
    {"grad_norm", py_norm, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "flexsae_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_flexsae_binding() { return PyModule_Create(&module); }

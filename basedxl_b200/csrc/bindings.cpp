// Native side of the training operators' wrappers (layernorm_fwd / _bwd, linear_act / _bwd in ops.py): checks of the arguments, results,
// workspaces and the call of the C ABI.  In Python these took 5 to 10 us a call on top of 2.5 us a launch, more than the
// kernels themselves at one row (layernorm_fwd of 1 x 1280: 9.5 us, 1.8 of them on the device).  The other operators stay on
// ctypes; the library behind both knows no torch types.
//
// Every function takes its arguments by position (ops.py has the signatures), raises ValueError for arguments that the kernels
// would misread, before any CUDA call, and BxlError for what the library reports.
#include <Python.h>

#include <string>

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/basedxl_b200.h"

namespace {

using at::Tensor;

PyObject* g_lib_module = nullptr;   // basedxl_b200._lib: lib() initialises a device, `launches` counts kernels, BxlError

const Tensor& tensor_arg(PyObject* o, const char* who, const char* what) {
  TORCH_CHECK_TYPE(THPVariable_Check(o), who, ": ", what, " must be a tensor");
  return THPVariable_Unpack(o);
}
// None, or a tensor
struct Optional {
  const Tensor* t;
  explicit operator bool() const { return t != nullptr; }
  const Tensor* operator->() const { return t; }
  const void* ptr() const { return t ? t->const_data_ptr() : nullptr; }
};
Optional optional_arg(PyObject* o, const char* who, const char* what) { return o == Py_None ? Optional{nullptr} : Optional{&tensor_arg(o, who, what)}; }

// Messages are put together from strings: numbers do not go through a stream here, whose locale may be that of another copy of the
// C++ library than the one that formats them (PyTorch brings its own).
std::string text(at::IntArrayRef sizes) {
  std::string r = "[";
  for (size_t i = 0; i < sizes.size(); ++i) r += (i ? ", " : "") + std::to_string(sizes[i]);
  return r + "]";
}
const char* text(at::ScalarType t) { return c10::toString(t); }
std::string text(const at::Device& d) { return std::string(d.is_cuda() ? "cuda:" : d.is_cpu() ? "cpu" : "another device") + (d.is_cuda() ? std::to_string(d.index()) : ""); }

int type_of(at::ScalarType t) { return t == at::kHalf ? BXL_F16 : t == at::kBFloat16 ? BXL_BF16 : t == at::kFloat ? BXL_F32 : -1; }

// A tensor as rows of its last axis, one stride apart: a view where its strides allow one, else a copy.
struct Rows {
  Tensor copy;
  const void* p = nullptr;
  int64_t ld = 0;
  explicit Rows(const Tensor& t) {
    const auto sizes = t.sizes(), strides = t.strides();
    const int64_t n = t.dim(), cols = sizes[n - 1];
    bool view = cols == 1 || strides[n - 1] == 1;
    ld = cols;
    int64_t last = -1;   // the innermost axis of several rows met so far ...
    for (int64_t i = n - 2; i >= 0 && view; --i) {
      if (sizes[i] == 1) continue;
      if (last < 0) ld = strides[i];
      else view = strides[i] == strides[last] * sizes[last];   // ... which the next one has to continue
      last = i;
    }
    if (view && ld >= 0) {
      p = t.const_data_ptr();
    } else {
      copy = t.contiguous();
      p = copy.const_data_ptr(), ld = cols;
    }
  }
};

Tensor empty(at::IntArrayRef sizes, at::ScalarType type, at::Device dev) { return Tensor(at::detail::empty_cuda(sizes, type, dev, std::nullopt)); }

void same(const char* who, const char* what, const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  TORCH_CHECK_VALUE(t.sizes() == sizes && t.scalar_type() == type, who, ": ", what, " must be ", text(sizes), " of type ", text(type), ", got ", text(t.sizes()), " of type ", text(t.scalar_type()));
}
void same_device(const char* who, std::initializer_list<const Tensor*> others, const Tensor& x) {
  TORCH_CHECK_VALUE(x.is_cuda() && x.device().index() == c10::cuda::current_device(), who, ": expected tensors of the current CUDA device, got ", text(x.device()));
  for (const Tensor* t : others) TORCH_CHECK_VALUE(!t || t->device() == x.device(), who, ": expected all tensors on ", text(x.device()), ", got ", text(t->device()));
}

// `out` is written while other rows of the inputs are still being read: it may be one of them from end to end where that is said, and
// otherwise shares no memory with them.
void apart(const char* who, const Tensor& out, const char* what, const Tensor* other, bool may_be_it) {
  if (!other || !out.numel() || !other->numel()) return;
  auto behind = [](const Tensor& t) {
    int64_t last = 0;
    for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
    return static_cast<const char*>(t.const_data_ptr()) + (last + 1) * t.element_size();
  };
  const char *a = static_cast<const char*>(out.const_data_ptr()), *b = static_cast<const char*>(other->const_data_ptr());
  if (a >= behind(*other) || b >= behind(out)) return;
  TORCH_CHECK_VALUE(may_be_it && a == b && other->is_contiguous(), who, ": out overlaps ", what);
}

// As PyTorch's own functions: what is written to it would be missing from the graph that autograd records.
void writable(const char* who, const Tensor& out) {
  TORCH_CHECK_VALUE(out.is_contiguous(), who, ": out must be contiguous");
  TORCH_CHECK_VALUE(!(out.requires_grad() && at::GradMode::is_enabled()), who, ": out requires a gradient, which is not recorded here");
}
// A tensor that has been written to counts as changed: its new version is by what autograd and this package's caches (K/V of the
// conditioning, packed weights) see it.
void written(const Tensor& out) {
  if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
}

// The library, set up for the current device (through _lib.lib(), once per device).
void ensure_device(int dev) {
  static bool ready[64] = {};
  if (dev >= 0 && dev < 64 && ready[dev]) return;
  PyObject* r = PyObject_CallMethod(g_lib_module, "lib", nullptr);
  if (!r) throw python_error();
  Py_DECREF(r);
  if (dev >= 0 && dev < 64) ready[dev] = true;
}
void raise_failure(int rc) {
  PyObject* error = PyObject_GetAttrString(g_lib_module, "BxlError");
  if (error) {
    PyErr_Format(error, "libbasedxl_b200 error %d: %s", rc, bxl_last_error());
    Py_DECREF(error);
  }
  throw python_error();
}
void finish(int rc, long kernels) {
  if (rc != 0) raise_failure(rc);
  PyObject* dict = PyModule_GetDict(g_lib_module);   // borrowed
  PyObject* now = PyDict_GetItemString(dict, "launches");
  PyObject* then = now ? PyLong_FromLong(PyLong_AsLong(now) + kernels) : nullptr;
  if (!then || PyDict_SetItemString(dict, "launches", then) != 0) {
    Py_XDECREF(then);
    throw python_error();
  }
  Py_DECREF(then);
}

PyObject* wrap(const Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}
PyObject* wrap3(const Tensor& a, const Tensor& b, const Tensor& c) {
  PyObject* r = PyTuple_New(3);
  if (!r) throw python_error();
  const Tensor* t[3] = {&a, &b, &c};
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(r, i, wrap(*t[i]));
  return r;
}
void arguments(Py_ssize_t got, Py_ssize_t want) { TORCH_CHECK_TYPE(got == want, "expected ", std::to_string(want), " arguments, got ", std::to_string(got)); }

// ---- LayerNorm -----------------------------------------------------------------------------------
at::ScalarType norm_input(const char* who, const Tensor& x) {
  TORCH_CHECK_VALUE(type_of(x.scalar_type()) >= 0 && x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= (1 << 30), who,
                    ": expected fp16, bf16 or fp32 rows of at least one element, got ", text(x.scalar_type()), " ", text(x.sizes()));
  return x.scalar_type();
}
void norm_param(const char* who, const Tensor& t, const Tensor& x) {
  TORCH_CHECK_VALUE(t.dim() == 1 && t.size(0) == x.size(-1) && t.is_contiguous() && (t.scalar_type() == x.scalar_type() || t.scalar_type() == at::kFloat), who,
                    ": weight and bias must be contiguous [", std::to_string(x.size(-1)), "] vectors in the type of x or in fp32");
}

PyObject* layernorm_fwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const char* who = "layernorm_fwd";
  arguments(nargs, 6);
  const Tensor& x = tensor_arg(args[0], who, "x");
  const Optional w = optional_arg(args[1], who, "weight"), b = optional_arg(args[2], who, "bias"), into = optional_arg(args[4], who, "out");
  const double eps = PyFloat_AsDouble(args[3]);
  if (PyErr_Occurred()) throw python_error();
  const bool stats = args[5] == Py_True;
  const at::ScalarType type = norm_input(who, x);
  if (w) norm_param(who, *w.t, x);
  if (b) norm_param(who, *b.t, x);
  TORCH_CHECK_VALUE(!w || !b || w->scalar_type() == b->scalar_type(), who, ": weight and bias must share a type");
  if (into) {
    same(who, "out", *into.t, x.sizes(), type);
    writable(who, *into.t);
    apart(who, *into.t, "x", &x, true), apart(who, *into.t, "weight", w.t, false), apart(who, *into.t, "bias", b.t, false);
  }
  same_device(who, {w.t, b.t, into.t}, x);
  const int64_t c = x.size(-1), rows = x.numel() / c;
  Tensor y = into ? *into.t : empty(x.sizes(), type, x.device()), mean, rstd;
  if (stats) {
    mean = empty(x.sizes().slice(0, x.dim() - 1), at::kFloat, x.device());
    rstd = empty(mean.sizes(), at::kFloat, x.device());
  }
  if (rows) {
    ensure_device(x.device().index());
    const Rows r(x);
    const int dt = type_of(type), pt = w ? type_of(w->scalar_type()) : b ? type_of(b->scalar_type()) : dt;
    finish(bxl_layernorm_fwd(r.p, r.ld, w.ptr(), b.ptr(), y.mutable_data_ptr(), c, stats ? mean.mutable_data_ptr<float>() : nullptr,
                             stats ? rstd.mutable_data_ptr<float>() : nullptr, rows, (int)c, dt, pt, (float)eps, c10::cuda::getCurrentCUDAStream().stream()),
           1);
    if (into) written(y);
  }
  return stats ? wrap3(y, mean, rstd) : wrap(y);
  END_HANDLE_TH_ERRORS
}

PyObject* layernorm_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const char* who = "layernorm_bwd";
  arguments(nargs, 7);
  const Tensor &dy = tensor_arg(args[0], who, "dy"), &x = tensor_arg(args[1], who, "x"), &mean = tensor_arg(args[2], who, "mean"), &rstd = tensor_arg(args[3], who, "rstd");
  const Optional w = optional_arg(args[4], who, "weight");
  const bool want_dw = args[5] == Py_True && w, want_db = args[6] == Py_True;
  const at::ScalarType type = norm_input(who, x);
  same(who, "dy", dy, x.sizes(), type);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  same(who, "mean", mean, lead, at::kFloat);
  same(who, "rstd", rstd, lead, at::kFloat);
  TORCH_CHECK_VALUE(mean.is_contiguous() && rstd.is_contiguous(), who, ": mean and rstd must be contiguous");
  if (w) norm_param(who, *w.t, x);
  same_device(who, {&dy, &mean, &rstd, w.t}, x);
  const int64_t c = x.size(-1), rows = x.numel() / c;
  const at::ScalarType param = w ? w->scalar_type() : type;
  Tensor dx = empty(x.sizes(), type, x.device()), dw, db;
  if (want_dw) dw = empty({c}, param, x.device());
  if (want_db) db = empty({c}, param, x.device());
  if (rows) {
    ensure_device(x.device().index());
    const Rows rd(dy), rx(x);
    const int64_t bytes = want_dw || want_db ? bxl_layernorm_bwd_workspace_bytes(rows, (int)c) : 0;
    const Tensor ws = bytes ? empty({bytes}, at::kByte, x.device()) : Tensor();
    const int rc = bxl_layernorm_bwd(rd.p, rd.ld, rx.p, rx.ld, mean.const_data_ptr<float>(), rstd.const_data_ptr<float>(), w.ptr(), dx.mutable_data_ptr(), c,
                                     want_dw ? dw.mutable_data_ptr() : nullptr, want_db ? db.mutable_data_ptr() : nullptr, rows, (int)c, type_of(type), type_of(param),
                                     bytes ? ws.mutable_data_ptr() : nullptr, bytes, c10::cuda::getCurrentCUDAStream().stream());
    finish(rc, bxl_layernorm_bwd_launches());
  } else {
    if (want_dw) dw.zero_();
    if (want_db) db.zero_();
  }
  return wrap3(dx, dw, db);
  END_HANDLE_TH_ERRORS
}

// ---- linear layers with an activation -------------------------------------------------------------
// x [..., K], weight [N, K]; returns the sizes of the result
c10::SmallVector<int64_t, 6> linear_input(const char* who, const Tensor& x, const Tensor& w) {
  const at::ScalarType t = x.scalar_type();
  TORCH_CHECK_VALUE((t == at::kHalf || t == at::kBFloat16) && x.dim() >= 1 && w.dim() == 2 && w.scalar_type() == t && w.size(1) == x.size(-1) && w.size(0) >= 1 && w.size(1) >= 1,
                    who, ": expected fp16 or bf16 x [..., K] and weight [N, K], got ", text(t), " ", text(x.sizes()), " and ", text(w.scalar_type()), " ", text(w.sizes()));
  TORCH_CHECK_VALUE(x.numel() / x.size(-1) <= (1 << 30) && w.size(0) <= (1 << 30) && w.size(1) <= (1 << 30), who, ": extents of at most 2^30");
  c10::SmallVector<int64_t, 6> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = w.size(0);
  return sizes;
}

PyObject* linear_act(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const char* who = "linear_act";
  arguments(nargs, 7);
  const Tensor &x = tensor_arg(args[0], who, "x"), &w = tensor_arg(args[1], who, "weight");
  const Optional b = optional_arg(args[2], who, "bias"), res = optional_arg(args[4], who, "residual"), into = optional_arg(args[5], who, "out");
  const long act = PyLong_AsLong(args[3]);
  if (PyErr_Occurred()) throw python_error();
  const bool want_pre = args[6] == Py_True;
  const auto sizes = linear_input(who, x, w);
  const at::ScalarType type = x.scalar_type();
  const int64_t k = w.size(1), n = w.size(0), m = x.numel() / k;
  if (b) {
    same(who, "bias", *b.t, {n}, type);
    TORCH_CHECK_VALUE(b->is_contiguous(), who, ": bias must be contiguous");
  }
  if (res) same(who, "residual", *res.t, sizes, type);
  if (into) {
    same(who, "out", *into.t, sizes, type);
    writable(who, *into.t);
    apart(who, *into.t, "x", &x, false), apart(who, *into.t, "weight", &w, false), apart(who, *into.t, "bias", b.t, false), apart(who, *into.t, "residual", res.t, true);
  }
  same_device(who, {&w, b.t, res.t, into.t}, x);
  Tensor y = into ? *into.t : empty(sizes, type, x.device()), pre;
  if (want_pre) pre = empty(sizes, type, x.device());
  if (m) {
    ensure_device(x.device().index());
    const Rows rx(x), rw(w);
    bxl_linear_args a = {};
    a.x = rx.p, a.ldx = rx.ld, a.weight = rw.p, a.ldw = rw.ld, a.bias = b.ptr();
    Tensor keep;
    if (res) {
      const Rows rr(*res.t);
      keep = rr.copy, a.residual = rr.p, a.ldr = rr.ld;
    }
    a.y = y.mutable_data_ptr(), a.ldy = n;
    if (want_pre) a.pre = pre.mutable_data_ptr(), a.ldp = n;
    a.M = (int)m, a.N = (int)n, a.K = (int)k, a.dtype = type_of(type), a.act = (int)act;
    a.workspace_bytes = bxl_linear_act_fwd_workspace_bytes(&a);
    const Tensor ws = a.workspace_bytes ? empty({a.workspace_bytes}, at::kByte, x.device()) : Tensor();
    if (ws.defined()) a.workspace = ws.mutable_data_ptr();
    int launches = 0;
    const int rc = bxl_linear_act_fwd(&a, &launches, c10::cuda::getCurrentCUDAStream().stream());
    finish(rc, launches);
    if (into) written(y);
  }
  if (!want_pre) return wrap(y);
  PyObject* r = PyTuple_New(2);
  if (!r) throw python_error();
  PyTuple_SET_ITEM(r, 0, wrap(y));
  PyTuple_SET_ITEM(r, 1, wrap(pre));
  return r;
  END_HANDLE_TH_ERRORS
}

PyObject* linear_act_bwd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  const char* who = "linear_act_bwd";
  arguments(nargs, 8);
  const Tensor &dy = tensor_arg(args[0], who, "dy"), &x = tensor_arg(args[1], who, "x"), &w = tensor_arg(args[2], who, "weight");
  const Optional pre = optional_arg(args[3], who, "pre");
  const long act = PyLong_AsLong(args[4]);
  if (PyErr_Occurred()) throw python_error();
  const bool want_dx = args[5] == Py_True, want_dw = args[6] == Py_True, want_db = args[7] == Py_True;
  const auto sizes = linear_input(who, x, w);
  const at::ScalarType type = x.scalar_type();
  const int64_t k = w.size(1), n = w.size(0), m = x.numel() / k;
  same(who, "dy", dy, sizes, type);
  if (pre) same(who, "pre", *pre.t, sizes, type);
  TORCH_CHECK_VALUE(act == BXL_ACT_NONE || pre, who, ": an activation needs the value before it (pre)");
  same_device(who, {&dy, &w, pre.t}, x);
  Tensor dx, dw, db;
  if (want_dx) dx = empty(x.sizes(), type, x.device());
  if (want_dw) dw = empty({n, k}, type, x.device());
  if (want_db) db = empty({n}, type, x.device());
  if (!m) {
    if (want_dw) dw.zero_();
    if (want_db) db.zero_();
  } else if (want_dx || want_dw || want_db) {
    ensure_device(x.device().index());
    const Rows rx(x), rw(w), rd(dy);
    bxl_linear_args a = {};
    a.x = rx.p, a.ldx = rx.ld, a.weight = rw.p, a.ldw = rw.ld, a.dy = rd.p, a.lddy = rd.ld;
    Tensor keep;
    if (pre) {
      const Rows rp(*pre.t);
      keep = rp.copy, a.pre = const_cast<void*>(rp.p), a.ldp = rp.ld;
    }
    if (want_dx) a.dx = dx.mutable_data_ptr(), a.lddx = k;
    if (want_dw) a.dweight = dw.mutable_data_ptr(), a.lddw = k;
    if (want_db) a.dbias = db.mutable_data_ptr();
    a.M = (int)m, a.N = (int)n, a.K = (int)k, a.dtype = type_of(type), a.act = (int)act;
    a.workspace_bytes = bxl_linear_act_bwd_workspace_bytes(&a);
    const Tensor ws = a.workspace_bytes ? empty({a.workspace_bytes}, at::kByte, x.device()) : Tensor();
    if (ws.defined()) a.workspace = ws.mutable_data_ptr();
    int launches = 0;
    const int rc = bxl_linear_act_bwd(&a, &launches, c10::cuda::getCurrentCUDAStream().stream());
    finish(rc, launches);
  }
  return wrap3(dx, dw, db);
  END_HANDLE_TH_ERRORS
}

// The module that _lib.py is: called once, before the first operator.
PyObject* connect(PyObject*, PyObject* module) {
  Py_XINCREF(module);
  Py_XDECREF(g_lib_module);
  g_lib_module = module;
  Py_RETURN_NONE;
}

PyCFunction fast(_PyCFunctionFast f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }
PyMethodDef g_methods[] = {
    {"connect", connect, METH_O, nullptr},
    {"layernorm_fwd", fast(layernorm_fwd), METH_FASTCALL, nullptr},
    {"layernorm_bwd", fast(layernorm_bwd), METH_FASTCALL, nullptr},
    {"linear_act", fast(linear_act), METH_FASTCALL, nullptr},
    {"linear_act_bwd", fast(linear_act_bwd), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_native", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__native() { return PyModule_Create(&g_module); }

// torch_int8.cc -- the calls of kaldi_amd/int8.py on torch tensors, as a Python extension module (kaldi_amd/lib/_torch_int8.*.so).
//
// A call on one frame takes the GPU 2 to 3 us; looked at from Python (attribute reads of four tensors, two allocations, sixteen
// converted arguments) it took 9.  Here the same checks read the tensors themselves.  The work is the C-ABI's: the module is handed
// the entry points of the library that is loaded (init), and links to torch alone.
#define PY_SSIZE_T_CLEAN
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/ops/empty_strided.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>

#include <algorithm>
#include <string>

#include "../../include/kaldi_amd.h"

namespace {

PyObject *g_error = NULL, *g_stream = NULL;       // KamdError; device index -> stream of torch's current one, as a number
decltype(&kamd_rms_norm_device) g_norm = NULL;
decltype(&kamd_quantize_rows_device) g_quantize = NULL;
decltype(&kamd_component_i8_propagate) g_propagate = NULL;
decltype(&kamd_last_error) g_last_error = NULL;

struct Refused {};                                // the Python error is set
[[noreturn]] void Refuse(const std::string &what) {
  PyErr_SetString(g_error, what.c_str());
  throw Refused();
}
std::string Name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kBFloat16: return "torch.bfloat16";
    case at::kHalf: return "torch.float16";
    case at::kDouble: return "torch.float64";
    case at::kChar: return "torch.int8";
    default: return c10::toString(t);
  }
}
std::string Shape(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); i++) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}
int Type(at::ScalarType t, const char *what) {
  if (t == at::kFloat) return KAMD_F32;
  if (t == at::kBFloat16) return KAMD_BF16;
  if (t == at::kHalf) return KAMD_F16;
  Refuse(std::string(what) + ": float32, bfloat16 or float16 expected, got " + Name(t));
}

struct Matrix {
  at::Tensor t;
  int64_t rows = 0, cols = 0, ld = 0;
  bool given() const { return t.defined(); }
  void *data() const { return t.defined() ? t.data_ptr() : NULL; }
  PyObject *wrap() const { return THPVariable_Wrap(t); }
};

// While torch records what is computed, these calls, no operators of torch's, would be left out and their results kept as constants.
void RefuseTracing() {
  using Modes = c10::impl::TorchDispatchModeTLS;
  using Key = c10::impl::TorchDispatchModeKey;
  if (torch::jit::tracer::isTracing() || Modes::get_mode(Key::PROXY) || Modes::get_mode(Key::FAKE) || Modes::get_mode(Key::FUNCTIONAL))
    Refuse("kaldi_amd.int8: these calls cannot be traced (torch.jit.trace, make_fx, FakeTensorMode)");
}
void RefuseGradient(const at::Tensor &t, const char *what) {
  if (t.requires_grad() && at::GradMode::is_enabled())
    Refuse(std::string(what) + ": has a gradient to keep track of, and these calls have none (torch.no_grad or detach)");
  if (t._fw_grad(0).defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode())
    Refuse(std::string(what) + ": has a tangent (forward-mode gradient) to carry on, and these calls have none (detach)");
}
// a tensor whose values are not what its memory holds, or that has none: fake, wrapped (by a subclass or by functionalization,
// whose null pointer would read as an argument that is not given) or lazily negated ones
void RefuseHollow(const at::Tensor &t, const char *what) {
  if (t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize})) || !t.has_storage() || t.is_neg() || t._is_zerotensor())
    Refuse(std::string(what) + ": a plain tensor with memory of its own is expected");
  // the memory can be shorter than what the shape spans: untyped_storage().resize_() leaves the tensors on it as they were
  int64_t span = t.numel() == 0 ? 0 : 1;
  for (int64_t d = 0; span > 0 && d < t.dim(); d++) span += (t.size(d) - 1) * t.stride(d);
  if (span > 0 && static_cast<int64_t>(t.storage().nbytes()) < (t.storage_offset() + span) * static_cast<int64_t>(t.itemsize()))
    Refuse(std::string(what) + ": its storage is shorter than the tensor");
}
// a given output is about to be written: autograd is told, as after torch's own in-place operators
void Written(const at::Tensor &t) {
  if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
Matrix Take(PyObject *o, const char *what) {
  if (!THPVariable_Check(o) || !THPVariable_Unpack(o).is_cuda()) Refuse(std::string(what) + ": a tensor on the GPU is expected");
  Matrix m;
  m.t = THPVariable_Unpack(o);
  RefuseHollow(m.t, what);
  if (m.t.dim() != 2) Refuse(std::string(what) + ": a matrix is expected, got shape " + Shape(m.t.sizes()));
  RefuseGradient(m.t, what);
  m.rows = m.t.size(0); m.cols = m.t.size(1); m.ld = m.t.stride(0);
  if (m.t.stride(1) != 1 && m.cols > 1) Refuse(std::string(what) + ": the values of a row have to be contiguous (strides " + Shape(m.t.strides()) + ")");
  if (m.rows <= 1 && m.ld < m.cols) m.ld = m.cols;             // (one row: whatever torch calls its distance)
  return m;
}
// another argument of a call whose first is on `device`
Matrix TakeLike(PyObject *o, const char *what, at::ScalarType type, int64_t rows, int64_t cols, c10::Device device) {
  Matrix m = Take(o, what);
  if (m.t.scalar_type() != type) Refuse(std::string(what) + ": " + Name(type) + " expected, got " + Name(m.t.scalar_type()));
  if (m.rows != rows || m.cols != cols) Refuse(std::string(what) + ": shape " + Shape({rows, cols}) + " expected, got " + Shape(m.t.sizes()));
  if (m.t.device() != device) Refuse(std::string(what) + ": on " + m.t.device().str() + ", the other arguments on " + device.str());
  return m;
}
float *TakeVector(PyObject *o, const char *what, int64_t n, c10::Device device) {
  if (THPVariable_Check(o)) {
    const at::Tensor &t = THPVariable_Unpack(o);
    RefuseGradient(t, what);
    RefuseHollow(t, what);
    if (t.device() == device && t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == n && t.is_contiguous()) return static_cast<float *>(t.data_ptr());
  }
  Refuse(std::string(what) + ": a contiguous float32 vector of " + std::to_string(n) + " on " + device.str() + " is expected");
}
Matrix Make(int64_t rows, int64_t cols, at::ScalarType type, c10::Device device) {
  Matrix m;
  m.t = at::empty_strided({rows, cols}, {cols, 1}, at::TensorOptions().dtype(type).device(device));
  m.rows = rows; m.cols = cols; m.ld = cols;
  return m;
}
// rows of codes as the product takes them: each begins on a multiple of 16 bytes
Matrix MakeCodes(int64_t rows, int64_t cols, c10::Device device) {
  const int64_t ld = (cols + 15) / 16 * 16;
  Matrix m = Make(rows, ld, at::kChar, device);
  if (ld != cols) m.t = m.t.narrow(1, 0, cols);
  m.cols = cols;
  return m;
}
void *Stream(c10::Device device) {
  PyObject *index = PyLong_FromLong(device.index()), *s = index ? PyObject_CallFunctionObjArgs(g_stream, index, NULL) : NULL;
  Py_XDECREF(index);
  if (!s) throw Refused();
  void *p = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  if (!p && PyErr_Occurred()) throw Refused();
  return p;
}
void Check(int rc) { if (rc < 0) Refuse(g_last_error()); }
bool None(PyObject *o) { return o == Py_None; }

template <typename F>
PyObject *Guarded(F f) {
  HANDLE_TH_ERRORS
  try {
    return f();
  } catch (const Refused &) {
    return NULL;
  }
  END_HANDLE_TH_ERRORS
}
PyObject *Pack(PyObject *a, PyObject *b, PyObject *c) {
  PyObject *t = a && b && (c || !PyErr_Occurred()) ? PyTuple_New(c ? 3 : 2) : NULL;
  if (!t) { Py_XDECREF(a); Py_XDECREF(b); Py_XDECREF(c); return NULL; }
  PyTuple_SET_ITEM(t, 0, a); PyTuple_SET_ITEM(t, 1, b);
  if (c) PyTuple_SET_ITEM(t, 2, c);
  return t;
}

// codes and scales of a call's output: given as a pair, or made
struct Codes { Matrix q; at::Tensor scale; };
Codes TakeCodes(PyObject *out, int64_t rows, int64_t cols, c10::Device device) {
  Codes c;
  if (None(out)) {
    c.q = MakeCodes(rows, cols, device);
    c.scale = at::empty_strided({rows}, {1}, at::TensorOptions().dtype(at::kFloat).device(device));
    return c;
  }
  if (!PyTuple_Check(out) || PyTuple_GET_SIZE(out) != 2) Refuse("out: a pair (codes, scale) is expected");
  c.q = TakeLike(PyTuple_GET_ITEM(out, 0), "codes", at::kChar, rows, cols, device);
  (void)TakeVector(PyTuple_GET_ITEM(out, 1), "scale", rows, device);
  c.scale = THPVariable_Unpack(PyTuple_GET_ITEM(out, 1));
  return c;
}

// (x, gain, eps, residual, sum_out, out, int8) -> y | (y, h) | (codes, scale) | (codes, scale, h)
PyObject *RmsNorm(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject * {
    if (n != 7) Refuse("rms_norm: 7 arguments expected");
    RefuseTracing();
    const Matrix x = Take(a[0], "x");
    const c10::Device device = x.t.device();
    const at::ScalarType st = x.t.scalar_type();
    const int type = Type(st, "x");
    const double eps = PyFloat_AsDouble(a[2]);
    if (eps == -1.0 && PyErr_Occurred()) throw Refused();
    const bool i8 = a[6] == Py_True;
    Matrix res, sum, y;
    if (!None(a[3])) res = TakeLike(a[3], "residual", st, x.rows, x.cols, device);
    const float *gain = None(a[1]) ? NULL : TakeVector(a[1], "gain", x.cols, device);
    Codes codes;
    const c10::DeviceGuard guard(device);
    if (!None(a[4])) sum = TakeLike(a[4], "sum_out", st, x.rows, x.cols, device);
    else if (res.given()) sum = Make(x.rows, x.cols, st, device);
    if (i8) codes = TakeCodes(a[5], x.rows, x.cols, device);
    else y = None(a[5]) ? Make(x.rows, x.cols, st, device) : TakeLike(a[5], "out", st, x.rows, x.cols, device);
    const Matrix &out = i8 ? codes.q : y;
    if (x.rows > 0) {
      const void *from = x.data(), *added = res.data();
      void *to_sum = sum.data(), *to = out.data(), *stream = Stream(device);
      float *to_scale = i8 ? static_cast<float *>(codes.scale.data_ptr()) : NULL;
      int rc;
      Py_BEGIN_ALLOW_THREADS
      rc = g_norm(from, x.ld, added, res.ld, type, gain, static_cast<float>(eps), x.rows, static_cast<int>(std::min<int64_t>(x.cols, INT32_MAX)),
                  to_sum, sum.ld, to, out.ld, i8 ? KAMD_I8 : type, to_scale, stream);
      Py_END_ALLOW_THREADS
      Check(rc);
      if (!None(a[4])) Written(sum.t);
      if (!None(a[5])) { Written(out.t); Written(codes.scale); }
    }
    PyObject *h = sum.given() ? sum.wrap() : NULL;
    if (i8) return Pack(out.wrap(), THPVariable_Wrap(codes.scale), h);
    return h ? Pack(out.wrap(), h, NULL) : out.wrap();
  });
}

// (x, offsets, out) -> (codes, scale)
PyObject *QuantizeRows(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject * {
    if (n != 3) Refuse("quantize_rows: 3 arguments expected");
    RefuseTracing();
    const Matrix x = Take(a[0], "x");
    const c10::Device device = x.t.device();
    const int type = Type(x.t.scalar_type(), "x");
    const Py_ssize_t parts = PyTuple_Check(a[1]) ? PyTuple_GET_SIZE(a[1]) : 0;
    if (parts < 1 || parts > KAMD_MAX_OFFSETS) Refuse("offsets: between 1 and " + std::to_string(KAMD_MAX_OFFSETS) + " of them expected");
    int32_t offsets[KAMD_MAX_OFFSETS];
    int64_t lo = INT64_MAX, hi = INT64_MIN;
    for (Py_ssize_t i = 0; i < parts; i++) {
      const long long v = PyLong_AsLongLong(PyTuple_GET_ITEM(a[1], i));
      if (v == -1 && PyErr_Occurred()) throw Refused();
      if (v < INT32_MIN || v > INT32_MAX) Refuse("offsets: out of range");
      offsets[i] = static_cast<int32_t>(v);
      lo = std::min<int64_t>(lo, v); hi = std::max<int64_t>(hi, v);
    }
    const int64_t rows = std::max<int64_t>(0, x.rows - (hi - lo));
    const c10::DeviceGuard guard(device);
    const Codes c = TakeCodes(a[2], rows, x.cols * parts, device);
    if (rows > 0) {
      const void *from = x.data();
      int8_t *to = static_cast<int8_t *>(c.q.data());
      float *to_scale = static_cast<float *>(c.scale.data_ptr());
      void *stream = Stream(device);
      int rc;
      Py_BEGIN_ALLOW_THREADS
      rc = g_quantize(from, x.ld, type, x.rows, static_cast<int>(std::min<int64_t>(x.cols, INT32_MAX)), offsets, static_cast<int>(parts),
                      to, c.q.ld, to_scale, stream);
      Py_END_ALLOW_THREADS
      Check(rc);
      if (!None(a[2])) { Written(c.q.t); Written(c.scale); }
    }
    return Pack(c.q.wrap(), THPVariable_Wrap(c.scale), NULL);
  });
}

// (handle, in_dim, out_dim, device index, codes, scale, dtype, out) -> out
PyObject *Propagate(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject * {
    if (n != 8) Refuse("propagate: 8 arguments expected");
    RefuseTracing();
    const kamd_component_i8 *handle = static_cast<const kamd_component_i8 *>(PyLong_AsVoidPtr(a[0]));
    const int64_t in_dim = PyLong_AsLongLong(a[1]), out_dim = PyLong_AsLongLong(a[2]);
    const c10::Device device(c10::DeviceType::CUDA, static_cast<c10::DeviceIndex>(PyLong_AsLong(a[3])));
    if (PyErr_Occurred()) throw Refused();
    if (!THPDtype_Check(a[6])) Refuse("dtype: a torch.dtype is expected");
    const at::ScalarType st = reinterpret_cast<THPDtype *>(a[6])->scalar_type;
    const int type = Type(st, "dtype");
    Matrix q = Take(a[4], "codes");
    if (q.t.scalar_type() != at::kChar) Refuse("codes: torch.int8 expected, got " + Name(q.t.scalar_type()));
    if (q.cols != in_dim || q.t.device() != device)
      Refuse("codes: [rows, " + std::to_string(in_dim) + "] on " + device.str() + " expected, got " + Shape(q.t.sizes()) + " on " + q.t.device().str());
    if (q.rows <= 1) q.ld = (in_dim + 15) / 16 * 16;
    if (q.ld % 16 != 0 || reinterpret_cast<uintptr_t>(q.data()) % 16 != 0) Refuse("codes: rows begin on multiples of 16 bytes (int8.empty_codes has the layout)");
    if (in_dim % 16 != 0 && q.rows > 0 &&
        static_cast<int64_t>(q.t.storage().nbytes()) - q.t.storage_offset() < (q.rows - 1) * q.ld + (in_dim + 15) / 16 * 16)
      Refuse("codes: the last row ends inside a block of 16 bytes that is not the tensor's own");
    const float *scale = TakeVector(a[5], "scale", q.rows, device);
    const c10::DeviceGuard guard(device);
    const Matrix out = None(a[7]) ? Make(q.rows, out_dim, st, device) : TakeLike(a[7], "out", st, q.rows, out_dim, device);
    if (q.rows > 0) {
      const int8_t *from = static_cast<const int8_t *>(q.data());
      void *to = out.data(), *stream = Stream(device);
      int rc;
      Py_BEGIN_ALLOW_THREADS
      rc = g_propagate(handle, from, q.ld, scale, q.rows, to, out.ld, type, stream);
      Py_END_ALLOW_THREADS
      Check(rc);
      if (!None(a[7])) Written(out.t);
    }
    return out.wrap();
  });
}

// (tensor, name): refused unless its memory holds its values, and nothing else is to be known of them
PyObject *Plain(PyObject *, PyObject *const *a, Py_ssize_t n) {
  return Guarded([&]() -> PyObject * {
    if (n != 2 || !THPVariable_Check(a[0])) Refuse("plain: a tensor and its name expected");
    RefuseTracing();
    const char *what = PyUnicode_AsUTF8(a[1]);
    if (!what) throw Refused();
    RefuseHollow(THPVariable_Unpack(a[0]), what);
    RefuseGradient(THPVariable_Unpack(a[0]), what);
    Py_RETURN_NONE;
  });
}

// (KamdError, stream function, addresses of kamd_rms_norm_device, kamd_quantize_rows_device, kamd_component_i8_propagate, kamd_last_error)
PyObject *Init(PyObject *, PyObject *const *a, Py_ssize_t n) {
  if (n != 6) { PyErr_SetString(PyExc_TypeError, "init: 6 arguments expected"); return NULL; }
  void *f[4];
  for (int i = 0; i < 4; i++) {
    f[i] = PyLong_AsVoidPtr(a[2 + i]);
    if (!f[i]) { if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "init: null entry point"); return NULL; }
  }
  Py_INCREF(a[0]); Py_INCREF(a[1]);
  g_error = a[0]; g_stream = a[1];
  g_norm = reinterpret_cast<decltype(g_norm)>(f[0]); g_quantize = reinterpret_cast<decltype(g_quantize)>(f[1]);
  g_propagate = reinterpret_cast<decltype(g_propagate)>(f[2]); g_last_error = reinterpret_cast<decltype(g_last_error)>(f[3]);
  Py_RETURN_NONE;
}

template <typename F> PyCFunction Fast(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)(void)>(f)); }
PyMethodDef g_methods[] = {{"init", Fast(Init), METH_FASTCALL, NULL},
                           {"plain", Fast(Plain), METH_FASTCALL, NULL},
                           {"rms_norm", Fast(RmsNorm), METH_FASTCALL, NULL},
                           {"quantize_rows", Fast(QuantizeRows), METH_FASTCALL, NULL},
                           {"propagate", Fast(Propagate), METH_FASTCALL, NULL},
                           {NULL, NULL, 0, NULL}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_int8", NULL, -1, g_methods, NULL, NULL, NULL, NULL};

}  // namespace

PyMODINIT_FUNC PyInit__torch_int8(void) { return PyModule_Create(&g_module); }

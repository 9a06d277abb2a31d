// Python entries of the 4-bit operators without per-argument work in Python: a call
// checks its tensors, packs their descriptors and calls the C ABI (include/bdh_hip.h)
// in about 2 us where the ctypes route of bdh_hip_ext.py takes 6 to 9, which is what
// a call of a generate step costs beside its launches.
//
// Every entry takes what its operator takes, then the device index and stream of the
// call, and returns None where an argument is not as the operator wants it (wrong
// shapes, types, devices, strides, gradients): nothing has been launched then, and the
// caller's Python checks, which it left out, say what is wrong or make the call.  Else
// it returns the C ABI's code, or the result.
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/utils/pybind.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>

#include "bdh_hip.h"

namespace {

// The library's functions, by address (bdh_hip_ext.py has loaded it).
struct Api {
  decltype(&bdh_mx4_quantize) quantize;
  decltype(&bdh_mx4_dequantize) dequantize;
  decltype(&bdh_mx4_rope) rope;
  decltype(&bdh_mx4_decode_workspace) decode_workspace;
  decltype(&bdh_mx4_decode) decode;
  decltype(&bdh_mx4_gemm_workspace) gemm_workspace;
  decltype(&bdh_mx4_gemm) gemm;
} api{};

// A call's GPU: the current one, and its stream.
struct Where {
  int64_t device;
  bdh_stream stream;
};

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool here(const at::Tensor& t, const Where& w) { return t.is_cuda() && t.get_device() == w.device; }
// Gradients or a forward-mode tangent, which a result would lose (level 0 is autograd's only one).
bool needs_grad(const at::Tensor& t) {
  return (t.requires_grad() && c10::GradMode::is_enabled()) || t._fw_grad(0).defined();
}

bool unit(const at::Tensor& t) { return t.size(-1) <= 1 || t.stride(-1) == 1; }

// A float32 or bfloat16 tensor of 1 to 4 dims, unit stride in the last, on the call's GPU.
bool describe(const at::Tensor& t, const Where& w, bdh_tensor4& d) {
  const int64_t n = t.dim();
  if (n < 1 || n > 4 || !here(t, w) || !unit(t)) return false;
  if (t.scalar_type() == at::kFloat)
    d.dtype = BDH_F32;
  else if (t.scalar_type() == at::kBFloat16)
    d.dtype = BDH_BF16;
  else
    return false;
  d.data = t.data_ptr();
  d.reserved = 0;
  for (int64_t i = 0; i < 4; ++i) {
    const bool has = i >= 4 - n;
    d.size[i] = has ? t.size(i - (4 - n)) : 1;
    d.stride[i] = has ? t.stride(i - (4 - n)) : 1;
  }
  return true;
}

// The same broadcast to the sizes of x.
bool describe_over(const at::Tensor& t, const bdh_tensor4& x, int64_t x_dims, const Where& w, bdh_tensor4& d) {
  if (t.dim() > x_dims || !describe(t, w, d)) return false;
  for (int i = 0; i < 4; ++i) {
    if (d.size[i] != x.size[i]) {
      if (d.size[i] != 1 || i == 3) return false;
      d.size[i] = x.size[i];
      d.stride[i] = 0;
    }
  }
  return true;
}

// The rows of a kernels.Mx4: codes, scales, width (checked to fit: the kernels take their
// addresses from the width).
struct Rows {
  const at::Tensor *codes, *scales;
  int64_t dims;
  bdh_mx4 d;
};
PyObject *s_codes, *s_scales, *s_width;

bool describe_rows(PyObject* m, const Where& w, Rows& r) {
  PyObject* c = PyObject_GetAttr(m, s_codes);
  PyObject* s = c != nullptr ? PyObject_GetAttr(m, s_scales) : nullptr;
  PyObject* n = s != nullptr ? PyObject_GetAttr(m, s_width) : nullptr;
  const int64_t width = n != nullptr ? PyLong_AsLongLong(n) : -1;
  r.codes = c != nullptr ? tensor(c) : nullptr;
  r.scales = s != nullptr ? tensor(s) : nullptr;
  // (m keeps both: the references go back at once)
  Py_XDECREF(c);
  Py_XDECREF(s);
  Py_XDECREF(n);
  if (PyErr_Occurred()) {
    PyErr_Clear();
    return false;
  }
  if (r.codes == nullptr || r.scales == nullptr || width < 0) return false;
  const int64_t dims = r.codes->dim();
  if (dims < 1 || dims > 4 || r.scales->dim() != dims || !here(*r.codes, w) || !here(*r.scales, w)) return false;
  if (r.codes->scalar_type() != at::kByte || r.scales->scalar_type() != at::kByte || !unit(*r.codes) || !unit(*r.scales) ||
      r.scales->size(-1) != width / 32 + (width % 32 != 0) || r.codes->size(-1) != 16 * r.scales->size(-1))
    return false;
  r.dims = dims;
  r.d.codes = r.codes->data_ptr();
  r.d.scales = r.scales->data_ptr();
  for (int64_t i = 0; i < 3; ++i) {
    const int64_t k = i - (4 - dims);
    r.d.size[i] = k >= 0 ? r.codes->size(k) : 1;
    r.d.code_stride[i] = k >= 0 ? r.codes->stride(k) : 1;
    r.d.scale_stride[i] = k >= 0 ? r.scales->stride(k) : 1;
    if (k >= 0 && r.scales->size(k) != r.d.size[i]) return false;
  }
  r.d.size[3] = width;
  return true;
}

bool same_size(const bdh_mx4& m, const bdh_tensor4& t) {
  for (int i = 0; i < 4; ++i)
    if (m.size[i] != t.size[i]) return false;
  return true;
}
bool same_size(const bdh_tensor4& a, const bdh_tensor4& b) {
  for (int i = 0; i < 4; ++i)
    if (a.size[i] != b.size[i]) return false;
  return true;
}

PyObject* none() { Py_RETURN_NONE; }

bool where(PyObject* const* args, Where& w) {
  w.device = PyLong_AsLongLong(args[0]);
  w.stream = reinterpret_cast<bdh_stream>(PyLong_AsUnsignedLongLong(args[1]));
  return !PyErr_Occurred();
}

// The error entries share: wrong counts of arguments are mistakes of the binding.
bool counts(Py_ssize_t n, Py_ssize_t want) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%zd arguments wanted, got %zd", want, n);
  return false;
}

// quantize(x, m, device, stream)
PyObject* quantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Where w;
  if (!counts(n, 4) || !where(a + 2, w)) return nullptr;
  const at::Tensor* x = tensor(a[0]);
  bdh_tensor4 dx;
  Rows m;
  if (x == nullptr || needs_grad(*x) || !describe(*x, w, dx) || !describe_rows(a[1], w, m) || m.dims != x->dim() ||
      !same_size(m.d, dx))
    return none();
  return PyLong_FromLong(api.quantize(&dx, &m.d, w.stream));
  END_HANDLE_TH_ERRORS
}

// dequantize(m, out, device, stream)
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Where w;
  if (!counts(n, 4) || !where(a + 2, w)) return nullptr;
  const at::Tensor* out = tensor(a[1]);
  bdh_tensor4 d;
  Rows m;
  if (out == nullptr || needs_grad(*out) || !describe(*out, w, d) || !describe_rows(a[0], w, m) || m.dims != out->dim() ||
      !same_size(m.d, d))
    return none();
  return PyLong_FromLong(api.dequantize(&m.d, &d, w.stream));
  END_HANDLE_TH_ERRORS
}

// rope(x, cos, sin, slot, out or None, device, stream)
PyObject* rope(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Where w;
  if (!counts(n, 7) || !where(a + 5, w)) return nullptr;
  const at::Tensor *x = tensor(a[0]), *cos = tensor(a[1]), *sin = tensor(a[2]), *out = tensor(a[4]);
  bdh_tensor4 dx, dc, ds, dout;
  Rows m;
  if (x == nullptr || cos == nullptr || sin == nullptr || (out == nullptr && a[4] != Py_None)) return none();
  if (needs_grad(*x) || needs_grad(*cos) || needs_grad(*sin) || (out != nullptr && needs_grad(*out))) return none();
  if (cos->sizes() != sin->sizes() || !describe(*x, w, dx) || dx.size[3] % 2 != 0 || !describe_over(*cos, dx, x->dim(), w, dc) ||
      !describe_over(*sin, dx, x->dim(), w, ds) || dc.dtype != BDH_F32 || ds.dtype != BDH_F32)
    return none();
  if (!describe_rows(a[3], w, m) || m.dims != x->dim() || !same_size(m.d, dx)) return none();
  if (out != nullptr && (!describe(*out, w, dout) || out->sizes() != x->sizes())) return none();
  return PyLong_FromLong(api.rope(&dx, &dc, &ds, &m.d, out != nullptr ? &dout : nullptr, w.stream));
  END_HANDLE_TH_ERRORS
}

// decode(q, k_past, v_past, device, stream): the result, or the code
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Where w;
  if (!counts(n, 5) || !where(a + 3, w)) return nullptr;
  const at::Tensor *q = tensor(a[0]), *v = tensor(a[2]);
  bdh_tensor4 dq, dv, dout;
  Rows k;
  if (q == nullptr || v == nullptr || q->dim() != 4 || v->dim() != 4 || needs_grad(*q) || needs_grad(*v)) return none();
  if (!describe(*q, w, dq) || !describe(*v, w, dv) || !describe_rows(a[1], w, k) || k.dims != 4) return none();
  if (k.d.size[0] != dq.size[0] || k.d.size[1] != dq.size[1] || k.d.size[3] != dq.size[3] || dv.size[0] != dq.size[0] ||
      dv.size[2] != k.d.size[2] || (dv.size[1] != 1 && dv.size[1] != dq.size[1]))
    return none();
  at::Tensor out = at::empty({dq.size[0], dq.size[1], dq.size[2], dv.size[3]}, q->options().requires_grad(false));
  if (!describe(out, w, dout)) return none();
  const size_t nb =
      api.decode_workspace(dq.size[0], dq.size[1], dq.size[2], k.d.size[2], dq.size[3], dv.size[3]);
  at::Tensor ws;
  if (nb > 0) ws = at::empty({int64_t(nb)}, k.codes->options());
  const int rc = api.decode(&dq, &k.d, &dv, &dout, nb > 0 ? ws.data_ptr() : nullptr, nb, w.stream);
  return rc == BDH_OK ? THPVariable_Wrap(std::move(out)) : PyLong_FromLong(rc);
  END_HANDLE_TH_ERRORS
}

// gemm(a (tensor or Mx4), wt, relu, mul or None, out or None, out_bf16, device, stream): the
// result, or the code
PyObject* gemm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  Where w;
  if (!counts(n, 8) || !where(a + 6, w)) return nullptr;
  const at::Tensor *x = tensor(a[0]), *mul = tensor(a[3]), *given = tensor(a[4]);
  bdh_tensor4 dx, dmul, dout;
  Rows x4, wt;
  if (!describe_rows(a[1], w, wt) || wt.dims < 2 || wt.dims > 3) return none();
  if (x != nullptr) {
    if (!describe(*x, w, dx) || x->dim() != wt.dims || dx.dtype != BDH_BF16 || needs_grad(*x)) return none();
  } else if (!describe_rows(a[0], w, x4) || x4.dims != wt.dims) {
    return none();
  }
  const int64_t* xs = x != nullptr ? dx.size : x4.d.size;
  if (xs[1] != wt.d.size[1] || xs[3] != wt.d.size[3]) return none();
  if ((mul == nullptr && a[3] != Py_None) || (given == nullptr && a[4] != Py_None)) return none();
  const int relu = PyObject_IsTrue(a[2]), bf16 = PyObject_IsTrue(a[5]);
  if (relu < 0 || bf16 < 0) return nullptr;
  at::Tensor out;
  if (given != nullptr) {
    if (given->dim() != wt.dims || needs_grad(*given)) return none();
    out = *given;
  } else {
    const auto o = wt.codes->options().dtype(bf16 ? at::kBFloat16 : at::kFloat);
    out = wt.dims == 3 ? at::empty({xs[1], xs[2], wt.d.size[2]}, o) : at::empty({xs[2], wt.d.size[2]}, o);
  }
  if (!describe(out, w, dout) || dout.size[1] != xs[1] || dout.size[2] != xs[2] || dout.size[3] != wt.d.size[2]) return none();
  if (mul != nullptr &&
      (!describe(*mul, w, dmul) || mul->dim() != wt.dims || needs_grad(*mul) || !same_size(dmul, dout)))
    return none();
  const bdh_tensor4* pa = x != nullptr ? &dx : nullptr;
  const bdh_mx4* pa4 = x != nullptr ? nullptr : &x4.d;
  const size_t nb = api.gemm_workspace(pa, pa4, &wt.d);
  at::Tensor ws;
  if (nb > 0) ws = at::empty({int64_t(nb)}, wt.codes->options());
  const int rc = api.gemm(pa, pa4, &wt.d, mul != nullptr ? &dmul : nullptr, relu, &dout, nb > 0 ? ws.data_ptr() : nullptr,
                          nb, w.stream);
  if (rc != BDH_OK) return PyLong_FromLong(rc);
  if (given != nullptr) {
    Py_INCREF(a[4]);
    return a[4];
  }
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// use(addresses): the seven functions of Api, in its order
PyObject* use(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!counts(n, 7)) return nullptr;
  void* p[7];
  for (int i = 0; i < 7; ++i) p[i] = PyLong_AsVoidPtr(a[i]);
  if (PyErr_Occurred()) return nullptr;
  api.quantize = reinterpret_cast<decltype(api.quantize)>(p[0]);
  api.dequantize = reinterpret_cast<decltype(api.dequantize)>(p[1]);
  api.rope = reinterpret_cast<decltype(api.rope)>(p[2]);
  api.decode_workspace = reinterpret_cast<decltype(api.decode_workspace)>(p[3]);
  api.decode = reinterpret_cast<decltype(api.decode)>(p[4]);
  api.gemm_workspace = reinterpret_cast<decltype(api.gemm_workspace)>(p[5]);
  api.gemm = reinterpret_cast<decltype(api.gemm)>(p[6]);
  Py_RETURN_NONE;
}

#define BDH_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {BDH_METHOD(use),  BDH_METHOD(quantize), BDH_METHOD(dequantize), BDH_METHOD(rope),
                         BDH_METHOD(decode), BDH_METHOD(gemm),     {nullptr, nullptr, 0, nullptr}};
PyModuleDef module_def = {PyModuleDef_HEAD_INIT, "bdh_bind", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_bdh_bind() {
  s_codes = PyUnicode_InternFromString("codes");
  s_scales = PyUnicode_InternFromString("scales");
  s_width = PyUnicode_InternFromString("width");
  if (s_codes == nullptr || s_scales == nullptr || s_width == nullptr) return nullptr;
  return PyModule_Create(&module_def);
}

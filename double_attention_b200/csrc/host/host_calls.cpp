// The host side of the eight-bit operators' ordinary calls, as a Python extension module.
//
// A call on one token is over on the device in 2 to 4 us; from Python, checking the tensors, allocating the outputs
// and converting the arguments takes 8 to 15.  The functions here do the same for tensors that lie as the kernels
// want them (dense, on the current device, of the right types, nothing requiring a gradient or carrying a tangent) in
// 4 to 6 us, launch included, and return None for anything else, which the Python functions then check, copy or
// refuse.  The kernels and their C entry points are the same either way.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/ops/slice.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "da_b200.h"

namespace {

PyObject* g_check = nullptr;  // check(name, status): raises the package's exception for a status

using at::Tensor;

// A float type's code, or -1.
int code_of(at::ScalarType t) {
  switch (t) {
    case at::kHalf: return DA_F16;
    case at::kBFloat16: return DA_BF16;
    case at::kFloat: return DA_F32;
    default: return -1;
  }
}
at::ScalarType type_of(int64_t code) {
  return code == DA_F16 ? at::kHalf : code == DA_BF16 ? at::kBFloat16 : at::kFloat;
}

// The tensor of an argument; null for None.  Sets `ok` to false for anything else, and where a kernel could not read
// the tensor in place: off the device, not dense, or part of a gradient or of a forward-mode derivative.
const Tensor* plain(PyObject* o, c10::DeviceIndex device, bool dense, bool* ok) {
  if (o == Py_None) return nullptr;
  if (!THPVariable_Check(o)) {
    *ok = false;
    return nullptr;
  }
  const Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.get_device() != device || (dense && !t.is_contiguous()) ||
      (t.requires_grad() && c10::GradMode::is_enabled()) ||
      (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined()))
    *ok = false;
  return &t;
}

struct Call {
  c10::DeviceIndex device = c10::cuda::current_device();
  bool ok = true;
  const Tensor* dense(PyObject* o) { return plain(o, device, true, &ok); }
  const Tensor* any(PyObject* o) { return plain(o, device, false, &ok); }
  void* stream() const { return c10::cuda::getCurrentCUDAStream(device).stream(); }
  Tensor empty(at::IntArrayRef sizes, at::ScalarType type) const {
    return at::detail::empty_cuda(sizes, type, c10::Device(c10::kCUDA, device), std::nullopt);
  }
};

void* data(const Tensor* t) { return t ? t->data_ptr() : nullptr; }
int code(const Tensor* t) { return t ? code_of(t->scalar_type()) : 0; }

// The result of a call: the given object, or the exception for its status.
PyObject* done(const char* name, int status, PyObject* result) {
  if (status == DA_OK) return result;
  Py_XDECREF(result);
  PyObject* r = PyObject_CallFunction(g_check, "si", name, status);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_Format(PyExc_RuntimeError, "%s failed with status %d", name, status);
  return nullptr;
}

// Whether a [..., K] int8 matrix can be read with 16-byte rows in place; its rows and their stride.
bool matrix16(const Tensor& t, int64_t* rows, int64_t* stride) {
  const int64_t nd = t.dim();
  if (t.scalar_type() != at::kChar || nd < 1 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
  const int64_t k = t.size(nd - 1);
  if (k < 1 || (k > 1 && t.stride(nd - 1) != 1)) return false;
  if (t.is_contiguous() && k % 16 == 0) {
    *rows = t.numel() / k;
    *stride = k;
    return true;
  }
  if (nd != 2) return false;
  *rows = t.size(0);
  *stride = *rows == 1 ? (k + 15) / 16 * 16 : t.stride(0);
  return *stride >= k && *stride % 16 == 0;
}
bool scales_of(const Tensor& s, const Tensor& values) {
  return s.scalar_type() == at::kFloat && s.is_contiguous() && s.sizes() == values.sizes().slice(0, values.dim() - 1);
}

// norm(x, branch, weight, bias, kind, eps) -> (x_out, values, scale)
PyObject* norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return PyErr_Format(PyExc_TypeError, "norm takes 6 arguments");
  Call c;
  const Tensor *x = c.dense(a[0]), *branch = c.dense(a[1]), *weight = c.dense(a[2]), *bias = c.dense(a[3]);
  const long kind = PyLong_AsLong(a[4]);
  const double eps = PyFloat_AsDouble(a[5]);
  if (PyErr_Occurred()) return nullptr;
  if (!c.ok || !x || x->dim() < 1) Py_RETURN_NONE;
  const at::IntArrayRef sizes = x->sizes();
  const int64_t d = sizes.back(), rows = d ? x->numel() / d : 0;
  if (rows < 1 || code(x) < 0 || (branch && (code(branch) < 0 || branch->sizes() != sizes))) Py_RETURN_NONE;
  if ((weight && (code(weight) < 0 || weight->dim() != 1 || weight->size(0) != d)) ||
      (bias && (!weight || code(bias) < 0 || bias->dim() != 1 || bias->size(0) != d)))
    Py_RETURN_NONE;
  const int64_t pitch = (d + 15) / 16 * 16;
  c10::SmallVector<int64_t, 6> wide(sizes.begin(), sizes.end());
  wide.back() = pitch;
  Tensor q = c.empty(wide, at::kChar), scale = c.empty(sizes.slice(0, sizes.size() - 1), at::kFloat), out;
  if (branch) out = c.empty(sizes, x->scalar_type());
  const int status =
      da_norm_int8(x->data_ptr(), code(x), d, data(branch), code(branch), d, data(weight), code(weight), data(bias),
                   code(bias), (int)kind, rows, d, (float)eps, branch ? out.data_ptr() : nullptr, d,
                   static_cast<int8_t*>(q.data_ptr()), pitch, static_cast<float*>(scale.data_ptr()), c.stream());
  if (status) return done("da_norm_int8", status, nullptr);
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, branch ? THPVariable_Wrap(std::move(out)) : (Py_INCREF(Py_None), Py_None));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(pitch == d ? std::move(q) : at::slice(q, -1, 0, d)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(scale)));
  return r;
  END_HANDLE_TH_ERRORS
}

// dequantize(values, scale, code) -> the values they stand for
PyObject* dequantize(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) return PyErr_Format(PyExc_TypeError, "dequantize takes 3 arguments");
  Call c;
  const Tensor *q = c.any(a[0]), *scale = c.dense(a[1]);
  const long out_code = PyLong_AsLong(a[2]);
  if (PyErr_Occurred()) return nullptr;
  int64_t rows = 0, stride = 0;
  if (!c.ok || !q || !scale || !matrix16(*q, &rows, &stride) || rows < 1 || !scales_of(*scale, *q)) Py_RETURN_NONE;
  const int64_t d = q->sizes().back();
  Tensor out = c.empty(q->sizes(), type_of(out_code));
  const int status = da_dequant_int8(static_cast<const int8_t*>(q->data_ptr()), stride,
                                     static_cast<const float*>(scale->data_ptr()), rows, d, out.data_ptr(), (int)out_code,
                                     d, c.stream());
  if (status) return done("da_dequant_int8", status, nullptr);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// linear(x values, x scale, weight values, weight scale, bias, gelu, code, status word) -> y
PyObject* linear(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8) return PyErr_Format(PyExc_TypeError, "linear takes 8 arguments");
  Call c;
  const Tensor *x = c.any(a[0]), *xs = c.dense(a[1]), *w = c.any(a[2]), *ws = c.dense(a[3]), *bias = c.dense(a[4]);
  const Tensor* word = c.dense(a[7]);
  const int gelu = PyObject_IsTrue(a[5]);
  const long out_code = PyLong_AsLong(a[6]);
  if (PyErr_Occurred()) return nullptr;
  int64_t m = 0, ldx = 0, nn = 0, ldw = 0;
  if (!c.ok || !x || !xs || !w || !ws || !word || w->dim() != 2 || !matrix16(*x, &m, &ldx) || !matrix16(*w, &nn, &ldw) ||
      m < 1 || nn < 1 || !scales_of(*xs, *x) || !scales_of(*ws, *w))
    Py_RETURN_NONE;
  const int64_t k = w->size(1);
  if (x->sizes().back() != k || k > 131071 || (bias && (code(bias) < 0 || bias->dim() != 1 || bias->size(0) != nn)))
    Py_RETURN_NONE;
  c10::SmallVector<int64_t, 6> sizes(x->sizes().begin(), x->sizes().end());
  sizes.back() = nn;
  Tensor y = c.empty(sizes, type_of(out_code));
  const int status =
      da_gemm_i8(static_cast<const int8_t*>(x->data_ptr()), ldx, static_cast<const float*>(xs->data_ptr()),
                 static_cast<const int8_t*>(w->data_ptr()), ldw, static_cast<const float*>(ws->data_ptr()), data(bias),
                 code(bias), gelu, y.data_ptr(), nn, (int)out_code, m, nn, k, static_cast<int*>(word->data_ptr()),
                 c.stream());
  if (status) return done("da_gemm_i8", status, nullptr);
  return THPVariable_Wrap(std::move(y));
  END_HANDLE_TH_ERRORS
}

bool half(const Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// checkpoint(x, gelu) -> (h, values, exponent)
PyObject* checkpoint(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 2) return PyErr_Format(PyExc_TypeError, "checkpoint takes 2 arguments");
  Call c;
  const Tensor* x = c.dense(a[0]);
  const int gelu = PyObject_IsTrue(a[1]);
  if (!c.ok || !x || x->dim() < 1 || x->numel() < 1 || !half(*x)) Py_RETURN_NONE;
  const int64_t d = x->sizes().back(), rows = x->numel() / d, blocks = (d + 31) / 32;
  Tensor q = c.empty({rows, blocks * 32}, at::kChar), e = c.empty({rows, blocks}, at::kChar), h;
  if (gelu) h = c.empty(x->sizes(), x->scalar_type());
  const int status = da_checkpoint8(x->data_ptr(), code(x), d, rows, d, gelu, gelu ? h.data_ptr() : nullptr, d,
                                    static_cast<int8_t*>(q.data_ptr()), static_cast<int8_t*>(e.data_ptr()), c.stream());
  if (status) return done("da_checkpoint8", status, nullptr);
  PyObject* r = PyTuple_New(3);
  PyTuple_SET_ITEM(r, 0, gelu ? THPVariable_Wrap(std::move(h)) : (Py_INCREF(Py_None), Py_None));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(q)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(e)));
  return r;
  END_HANDLE_TH_ERRORS
}

// A checkpoint of [rows, d], d being the last size of its activation.
bool kept_ok(const Tensor* q, const Tensor* e, int64_t rows, int64_t d) {
  const int64_t blocks = (d + 31) / 32;
  return q && e && q->scalar_type() == at::kChar && e->scalar_type() == at::kChar && q->dim() == 2 && e->dim() == 2 &&
         rows > 0 && d > 0 && q->size(0) == rows && q->size(1) == blocks * 32 && e->size(0) == rows &&
         e->size(1) == blocks && reinterpret_cast<uintptr_t>(q->data_ptr()) % 16 == 0;
}

// gelu_backward(dh, values, exponent) -> (dz, h); the caller has matched dh's shape and type with the checkpoint's
PyObject* gelu_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 3) return PyErr_Format(PyExc_TypeError, "gelu_backward takes 3 arguments");
  Call c;
  const Tensor *dh = c.dense(a[0]), *q = c.dense(a[1]), *e = c.dense(a[2]);
  if (!c.ok || !dh || dh->dim() < 1 || dh->numel() < 1 || !half(*dh)) Py_RETURN_NONE;
  const int64_t d = dh->sizes().back(), rows = dh->numel() / d;
  if (!kept_ok(q, e, rows, d)) Py_RETURN_NONE;
  Tensor dz = c.empty(dh->sizes(), dh->scalar_type()), h = c.empty(dh->sizes(), dh->scalar_type());
  const int status = da_checkpoint8_gelu_bwd(dh->data_ptr(), code(dh), d, static_cast<const int8_t*>(q->data_ptr()),
                                             static_cast<const int8_t*>(e->data_ptr()), rows, d, dz.data_ptr(), d,
                                             h.data_ptr(), d, c.stream());
  if (status) return done("da_checkpoint8_gelu_bwd", status, nullptr);
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(dz)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(h)));
  return r;
  END_HANDLE_TH_ERRORS
}

// weight_grad(dy, values, exponent, K, code, status word) -> dW; the caller has matched dy with the checkpoint
PyObject* weight_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6) return PyErr_Format(PyExc_TypeError, "weight_grad takes 6 arguments");
  Call c;
  const Tensor *dy = c.dense(a[0]), *q = c.dense(a[1]), *e = c.dense(a[2]), *word = c.dense(a[5]);
  const int64_t k = PyLong_AsLongLong(a[3]);
  const long out_code = PyLong_AsLong(a[4]);
  if (PyErr_Occurred()) return nullptr;
  if (!c.ok || !dy || !word || dy->dim() < 1 || dy->numel() < 1 || !half(*dy)) Py_RETURN_NONE;
  const int64_t nn = dy->sizes().back(), rows = dy->numel() / nn;
  if (!kept_ok(q, e, rows, k)) Py_RETURN_NONE;
  Tensor padded;  // rows on 16 bytes
  if (nn % 8 == 0 && reinterpret_cast<uintptr_t>(dy->data_ptr()) % 16) {
    padded = c.empty({rows, nn}, dy->scalar_type());
    padded.copy_(dy->view({rows, nn}));
    dy = &padded;
  }
  Tensor dw = c.empty({nn, k}, type_of(out_code)), work;
  const int64_t elems = da_checkpoint8_wgrad_workspace_elems(rows, nn, k);
  if (elems > 0) work = c.empty({elems}, at::kFloat);
  const int status = da_checkpoint8_wgrad(dy->data_ptr(), code(dy), nn, static_cast<const int8_t*>(q->data_ptr()),
                                          static_cast<const int8_t*>(e->data_ptr()), rows, nn, k, dw.data_ptr(),
                                          (int)out_code, k, elems > 0 ? static_cast<float*>(work.data_ptr()) : nullptr,
                                          elems, static_cast<int*>(word->data_ptr()), c.stream());
  if (status) return done("da_checkpoint8_wgrad", status, nullptr);
  return THPVariable_Wrap(std::move(dw));
  END_HANDLE_TH_ERRORS
}

// set_check(check): what raises the exception for a status
PyObject* set_check(PyObject*, PyObject* check) {
  Py_INCREF(check);
  Py_XSETREF(g_check, check);
  Py_RETURN_NONE;
}

template <PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)>
PyCFunction fast() {
  return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f));
}

PyMethodDef g_methods[] = {{"norm", fast<norm>(), METH_FASTCALL, nullptr},
                           {"dequantize", fast<dequantize>(), METH_FASTCALL, nullptr},
                           {"linear", fast<linear>(), METH_FASTCALL, nullptr},
                           {"checkpoint", fast<checkpoint>(), METH_FASTCALL, nullptr},
                           {"gelu_backward", fast<gelu_backward>(), METH_FASTCALL, nullptr},
                           {"weight_grad", fast<weight_grad>(), METH_FASTCALL, nullptr},
                           {"set_check", set_check, METH_O, nullptr},
                           {nullptr, nullptr, 0, nullptr}};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_host_calls", nullptr, -1, g_methods};

}  // namespace

PyMODINIT_FUNC PyInit__host_calls(void) {
  PyObject* m = PyModule_Create(&g_module);
  if (m && PyModule_AddStringConstant(m, "torch_version", DA_TORCH_VERSION) < 0) {  // whose C++ interface it was built for
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}

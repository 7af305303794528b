// The plain case of the training-step operators' Python calls, without a Python frame for every check: tensors that are
// contiguous, of the right types and shapes and on the current device.  Each function returns None for any other call,
// which the Python wrappers of the same operators (gncde/engine.py) then take: they lay out, switch devices or refuse.
// A call costs 7 us instead of 13 (read-out loss), a list of 200 tensors 20 instead of 110.
//
// Host code only: it fills the arguments of the C entry points of include/gncde.h, whose addresses Python hands over.  The
// module says which sources it was compiled from (this file and that header), and Python refuses it beside others.
#include <Python.h>

#include <ATen/Functions.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <vector>

#include "../../include/gncde.h"

namespace {

struct Entry {
  decltype(&gncde_linear_cross_entropy_workspace_bytes) loss_bytes;
  decltype(&gncde_linear_cross_entropy) loss;
  decltype(&gncde_linear_cross_entropy_grad) grad;
  decltype(&gncde_global_norm_workspace_bytes) list_bytes;
  decltype(&gncde_global_norm) norm;
  decltype(&gncde_clip_by_global_norm) clip;
  PyObject* get_stream;  // device index -> raw stream
  PyObject* check;       // error code -> None, or raises
  PyObject* no_memory;   // the error class of an allocation that failed
};
Entry g = {};

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

bool plain(const at::Tensor* t, const at::Tensor& like) {
  return t && t->layout() == at::kStrided && t->device() == like.device() && t->is_contiguous();
}

// Index of the device of t where it is the current one, else -1.
int current(const at::Tensor& t) {
  if (!t.is_cuda()) return -1;
  const c10::Device now = c10::impl::getDeviceGuardImpl(t.device().type())->getDevice();
  return t.device() == now ? now.index() : -1;
}

bool stream_of(int device, void*& out) {
  PyObject* i = PyLong_FromLong(device);
  PyObject* s = i ? PyObject_CallFunctionObjArgs(g.get_stream, i, nullptr) : nullptr;
  Py_XDECREF(i);
  if (!s) return false;
  out = PyLong_AsVoidPtr(s);
  Py_DECREF(s);
  return !PyErr_Occurred();
}

bool checked(int rc) {
  if (rc == 0) return true;
  PyObject* c = PyLong_FromLong(rc);
  PyObject* r = c ? PyObject_CallFunctionObjArgs(g.check, c, nullptr) : nullptr;  // raises
  Py_XDECREF(c);
  Py_XDECREF(r);
  if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, "gncde call failed");
  return false;
}

// Runs f; a C++ exception becomes a Python error.  Every look at a tensor belongs in here: memory runs out, and tensors
// without sizes or memory of their own throw where they are asked for them.
template <class F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const c10::OutOfMemoryError& e) {
    PyErr_SetString(g.no_memory, e.what_without_backtrace());
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

struct Readout {
  const at::Tensor *x, *W, *b, *target, *mask;
  int64_t rows, hidden, classes;
  int32_t dtype, kind;
  int device;
};

// (x, W, b, target, mask) of a plain call.
bool readout(PyObject* const* a, Readout& r) {
  r.x = tensor(a[0]), r.W = tensor(a[1]), r.target = tensor(a[3]);
  r.b = a[2] == Py_None ? nullptr : tensor(a[2]);
  r.mask = a[4] == Py_None ? nullptr : tensor(a[4]);
  if (!r.x || (a[2] != Py_None && !r.b) || (a[4] != Py_None && !r.mask)) return false;
  const at::Tensor& x = *r.x;
  if (!plain(&x, x) || !plain(r.W, x) || !plain(r.target, x) || (r.b && !plain(r.b, x)) || (r.mask && !plain(r.mask, x)))
    return false;
  const auto type = x.scalar_type();
  if (type == at::kFloat) r.dtype = GNCDE_DTYPE_FP32;
  else if (type == at::kBFloat16) r.dtype = GNCDE_DTYPE_BF16;
  else return false;
  if (r.W->scalar_type() != type || (r.b && r.b->scalar_type() != type)) return false;
  if (x.dim() < 1 || r.W->dim() != 2 || r.W->numel() == 0) return false;
  r.classes = r.W->size(0), r.hidden = r.W->size(1);
  const auto lead = x.sizes().slice(0, x.dim() - 1);
  if (x.size(-1) != r.hidden || (r.b && (r.b->dim() != 1 || r.b->size(0) != r.classes))) return false;
  if (r.mask && (r.mask->scalar_type() != at::kBool || r.mask->sizes() != lead)) return false;
  const auto want = r.target->sizes();
  switch (r.target->scalar_type()) {
    case at::kInt: r.kind = GNCDE_TARGET_INDEX32; break;
    case at::kLong: r.kind = GNCDE_TARGET_INDEX64; break;
    case at::kFloat: r.kind = GNCDE_TARGET_ROWS; break;
    default: return false;
  }
  if (r.kind == GNCDE_TARGET_ROWS) {
    if (want.size() != lead.size() + 1 || want.back() != r.classes || want.slice(0, lead.size()) != lead) return false;
  } else if (want != lead) {
    return false;
  }
  r.rows = x.numel() / r.hidden;
  r.device = current(x);
  return r.device >= 0;
}

void* ptr(const at::Tensor* t) { return t ? t->data_ptr() : nullptr; }

PyObject* py_loss(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    Readout r;
    if (n != 5 || !readout(a, r)) Py_RETURN_NONE;
    const auto opt = r.x->options().dtype(at::kFloat).requires_grad(false);
    const auto lead = r.x->sizes().slice(0, r.x->dim() - 1);
    at::Tensor loss = at::empty(lead, opt);
    std::vector<int64_t> two(lead.begin(), lead.end());
    two.push_back(2);
    at::Tensor stats = at::empty(two, opt);
    const size_t bytes = g.loss_bytes(r.rows, r.hidden, r.classes, r.dtype, 0);
    at::Tensor ws = at::empty({(int64_t)bytes}, opt.dtype(at::kByte));
    void* stream;
    if (!stream_of(r.device, stream) ||
        !checked(g.loss(r.rows, r.hidden, r.classes, r.dtype, ptr(r.x), ptr(r.W), ptr(r.b), r.kind, ptr(r.target),
                        static_cast<const uint8_t*>(ptr(r.mask)), loss.data_ptr<float>(), stats.data_ptr<float>(),
                        ws.data_ptr(), bytes, stream)))
      return nullptr;
    return Py_BuildValue("(NN)", THPVariable_Wrap(loss), THPVariable_Wrap(stats));
  });
}

PyObject* wrap(const at::Tensor& t) {
  if (t.defined()) return THPVariable_Wrap(t);
  Py_RETURN_NONE;
}

PyObject* py_grad(PyObject*, PyObject* const* a, Py_ssize_t n) {
  // (x, W, b, target, mask, stats, g, need_x, need_w, need_b)
  return guarded([&]() -> PyObject* {
    Readout r;
    if (n != 10 || !readout(a, r)) Py_RETURN_NONE;
    const at::Tensor *stats = tensor(a[5]), *cot = tensor(a[6]);
    if (!plain(stats, *r.x) || !plain(cot, *r.x) || stats->scalar_type() != at::kFloat ||
        cot->scalar_type() != at::kFloat)
      Py_RETURN_NONE;
    const auto lead = r.x->sizes().slice(0, r.x->dim() - 1);
    if (cot->sizes() != lead || stats->dim() != r.x->dim() || stats->sizes().back() != 2 ||
        stats->sizes().slice(0, lead.size()) != lead)
      Py_RETURN_NONE;
    const int nx = PyObject_IsTrue(a[7]), nw = PyObject_IsTrue(a[8]), nb = PyObject_IsTrue(a[9]);
    if (nx < 0 || nw < 0 || nb < 0) return nullptr;
    const auto opt = r.x->options().requires_grad(false);
    at::Tensor gx, gW, gb;
    if (nx) gx = at::empty(r.x->sizes(), opt);
    if (nw) gW = at::empty(r.W->sizes(), opt);
    if (nb && r.b) gb = at::empty(r.b->sizes(), opt);
    const size_t bytes = g.loss_bytes(r.rows, r.hidden, r.classes, r.dtype, 1);
    at::Tensor ws = at::empty({(int64_t)bytes}, opt.dtype(at::kByte));
    auto out = [](at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    void* stream;
    if (!stream_of(r.device, stream) ||
        !checked(g.grad(r.rows, r.hidden, r.classes, r.dtype, ptr(r.x), ptr(r.W), ptr(r.b), r.kind, ptr(r.target),
                        static_cast<const uint8_t*>(ptr(r.mask)), stats->data_ptr<float>(), cot->data_ptr<float>(),
                        out(gx), out(gW), out(gb), ws.data_ptr(), bytes, stream)))
      return nullptr;
    return Py_BuildValue("(NNN)", wrap(gx), wrap(gW), wrap(gb));
  });
}

// Outputs that meet each other, or a tensor that is not their own, would be written while they are read.
bool overlaps(const std::vector<GncdeTensor>& ts) {
  struct Span {
    uintptr_t at, end;
    const GncdeTensor* of;
  };
  auto bytes = [](const GncdeTensor& t) { return (uintptr_t)t.numel * (t.dtype == GNCDE_DTYPE_FP32 ? 4 : 2); };
  std::vector<Span> outs;
  outs.reserve(ts.size());
  for (const auto& t : ts)
    if (t.numel > 0) outs.push_back({(uintptr_t)t.out, (uintptr_t)t.out + bytes(t), &t});
  std::sort(outs.begin(), outs.end(), [](const Span& p, const Span& q) { return p.at < q.at; });
  for (size_t i = 1; i < outs.size(); ++i)
    if (outs[i].at < outs[i - 1].end) return true;
  for (const auto& t : ts) {
    if (t.numel == 0) continue;
    const uintptr_t at = (uintptr_t)t.in, end = at + bytes(t);
    auto it = std::upper_bound(outs.begin(), outs.end(), at, [](uintptr_t v, const Span& s) { return v < s.end; });
    for (; it != outs.end() && it->at < end; ++it)
      if (it->of != &t || t.in != t.out) return true;
  }
  return false;
}

int dtype_of(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return GNCDE_DTYPE_FP32;
    case at::kBFloat16: return GNCDE_DTYPE_BF16;
    case at::kHalf: return GNCDE_DTYPE_FP16;
    default: return -1;
  }
}

// (tensors, outputs or None, max_norm): the norm's stats, and with outputs the clipped tensors in them.
PyObject* py_list(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 3 || !PyList_CheckExact(a[0]) || (a[1] != Py_None && !PyList_CheckExact(a[1]))) Py_RETURN_NONE;
  const Py_ssize_t count = PyList_GET_SIZE(a[0]);
  const bool clip = a[1] != Py_None;
  if (count == 0 || count > (1 << 30) || (clip && PyList_GET_SIZE(a[1]) != count)) Py_RETURN_NONE;
  const double max_norm = clip ? PyFloat_AsDouble(a[2]) : 0.0;
  if (PyErr_Occurred()) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor* first = tensor(PyList_GET_ITEM(a[0], 0));
    const int device = first ? current(*first) : -1;
    if (device < 0) Py_RETURN_NONE;
    std::vector<GncdeTensor> ts((size_t)count);
    for (Py_ssize_t i = 0; i < count; ++i) {
      const at::Tensor* t = tensor(PyList_GET_ITEM(a[0], i));
      if (!plain(t, *first) || dtype_of(*t) < 0) Py_RETURN_NONE;
      GncdeTensor& e = ts[(size_t)i];
      e = {t->data_ptr(), nullptr, t->numel(), dtype_of(*t), 0};
      if (clip) {
        const at::Tensor* o = a[1] == a[0] ? t : tensor(PyList_GET_ITEM(a[1], i));
        if (!plain(o, *first) || o->scalar_type() != t->scalar_type() || o->numel() != t->numel()) Py_RETURN_NONE;
        e.out = o->data_ptr();
      }
    }
    if (clip && overlaps(ts)) Py_RETURN_NONE;  // Python says which way
    const auto opt = first->options().requires_grad(false);
    at::Tensor stats = at::empty({2}, opt.dtype(at::kFloat));
    const size_t bytes = g.list_bytes((int32_t)count);
    at::Tensor ws = at::empty({(int64_t)bytes}, opt.dtype(at::kByte));
    void* stream;
    if (!stream_of(device, stream)) return nullptr;
    const int rc = clip ? g.clip((int32_t)count, ts.data(), (float)max_norm, stats.data_ptr<float>(), ws.data_ptr(),
                                 bytes, stream)
                        : g.norm((int32_t)count, ts.data(), stats.data_ptr<float>(), ws.data_ptr(), bytes, stream);
    return checked(rc) ? THPVariable_Wrap(stats) : nullptr;
  });
}

// (addresses of the six entry points in Entry's order, get_stream, check, no_memory)
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "bind takes six addresses, two callables and an error class");
    return nullptr;
  }
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "a null entry point");
      return nullptr;
    }
  }
  g.loss_bytes = reinterpret_cast<decltype(g.loss_bytes)>(p[0]);
  g.loss = reinterpret_cast<decltype(g.loss)>(p[1]);
  g.grad = reinterpret_cast<decltype(g.grad)>(p[2]);
  g.list_bytes = reinterpret_cast<decltype(g.list_bytes)>(p[3]);
  g.norm = reinterpret_cast<decltype(g.norm)>(p[4]);
  g.clip = reinterpret_cast<decltype(g.clip)>(p[5]);
  PyObject** held[3] = {&g.get_stream, &g.check, &g.no_memory};
  for (int i = 0; i < 3; ++i) {
    Py_INCREF(a[6 + i]);
    Py_XDECREF(*held[i]);
    *held[i] = a[6 + i];
  }
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"bind", (PyCFunction)(void*)py_bind, METH_FASTCALL, nullptr},
    {"readout_loss", (PyCFunction)(void*)py_loss, METH_FASTCALL, nullptr},
    {"readout_grad", (PyCFunction)(void*)py_grad, METH_FASTCALL, nullptr},
    {"tensor_list", (PyCFunction)(void*)py_list, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__calls(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "source_sha256", GNCDE_CALLS_SHA256) < 0) Py_CLEAR(m);
  return m;
}

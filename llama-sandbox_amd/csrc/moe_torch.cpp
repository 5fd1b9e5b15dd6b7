// moe_torch.cpp -- the calls of the operators around the expert products from torch
// tensors: compares the tensors with what a call needs and makes it.  For moe_block.py,
// which names what is wrong where a function here returns None, and makes the
// call itself where this module was not built.  Host code only.  The smallest calls are bound
// by it: with the comparisons in Python and the call through ctypes one token's dispatch
// takes 6.7 us (2.5 of the kernel) and 3.7 so, a combine of 37 tokens 7.4 and 3.9, a quantiser and
// a product of one row 15.5 and 7.1, call after call on one set of inputs.
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include "../../include/moe_block.h"

#include <climits>

// The library's entry points, by address: a context's own library, whichever file it came from.
struct entries {
  decltype(&moe_dispatch) dispatch;
  decltype(&moe_dispatch_grad) dispatch_grad;
  decltype(&moe_combine) combine;
  decltype(&moe_combine_grad) combine_grad;
  decltype(&moe_quantize_i8) quantize_i8;
  decltype(&moe_matmul_i8) matmul_i8;
};

static PyObject *current_stream;  // a function: device -> handle of torch's current stream

static PyObject *set_current_stream(PyObject *, PyObject *f) {
  Py_INCREF(f);
  Py_XDECREF(current_stream);
  current_stream = f;
  Py_RETURN_NONE;
}

// What a call needs of its arguments; fine: all of it held so far.
struct call {
  const entries *lib;
  moe_ctx *ctx;
  int device;
  PyObject *device_arg, *stream_arg;
  bool fine;

  // args: entries' address, context handle, device, ..., stream (None: the device's current one)
  call(PyObject *const *args, Py_ssize_t n, Py_ssize_t want) {
    fine = n == want && PyLong_Check(args[0]) && PyLong_Check(args[1]) && PyLong_Check(args[2]);
    if (!fine) return;
    lib = (const entries *)PyLong_AsVoidPtr(args[0]);
    ctx = (moe_ctx *)PyLong_AsVoidPtr(args[1]);
    device = (int)PyLong_AsLong(args[2]);
    device_arg = args[2];
    stream_arg = args[n - 1];
    fine = !PyErr_Occurred() && (stream_arg == Py_None ? current_stream != nullptr : PyLong_Check(stream_arg));
  }

  // o as a contiguous tensor on the device that is not empty
  const at::Tensor *tensor(PyObject *o) {
    if (!fine || !THPVariable_Check(o)) return fine = false, nullptr;
    const at::Tensor &t = THPVariable_Unpack(o);
    fine = t.defined() && t.layout() == at::kStrided && t.is_cuda() && t.get_device() == device && t.is_contiguous() &&
           t.numel() > 0;
    for (int i = 0; fine && i < t.dim(); i++) fine = t.size(i) <= INT_MAX;
    return fine ? &t : nullptr;
  }
  // ... of a type and shape
  const at::Tensor *array(PyObject *o, at::ScalarType type, at::IntArrayRef shape) {
    const at::Tensor *t = tensor(o);
    if (t) fine = t->scalar_type() == type && t->sizes() == shape;
    return t;
  }
  // ... of rows; *type: the ggml type of their elements
  const at::Tensor *rows(PyObject *o, int *type) {
    const at::Tensor *t = tensor(o);
    if (!t) return t;
    const at::ScalarType s = t->scalar_type();
    *type = s == at::kFloat ? MOE_GGML_F32 : s == at::kHalf ? MOE_GGML_F16 : MOE_GGML_BF16;
    fine = t->dim() == 2 && (s == at::kFloat || s == at::kHalf || s == at::kBFloat16);
    return t;
  }
  // ... a pair map of T tokens; *k: its slots
  const at::Tensor *pairs(PyObject *o, int64_t T, int *k) {
    const at::Tensor *t = tensor(o);
    if (!t) return t;
    fine = t->scalar_type() == at::kInt && t->dim() == 1 && t->numel() % T == 0 && t->numel() / T <= 64;
    if (fine) *k = (int)(t->numel() / T);
    return t;
  }

  template <typename F>
  PyObject *make(F f) {
    void *stream;
    if (stream_arg == Py_None) {
      PyObject *s = PyObject_CallOneArg(current_stream, device_arg);
      if (!s) return nullptr;
      stream = PyLong_AsVoidPtr(s);
      Py_DECREF(s);
    } else {
      stream = PyLong_AsVoidPtr(stream_arg);
    }
    if (PyErr_Occurred()) return nullptr;
    moe_status st;
    PyThreadState *ts = PyEval_SaveThread();
    try {
      st = f(stream);
    } catch (...) {  // a tensor without memory
      PyEval_RestoreThread(ts);
      return nullptr;
    }
    PyEval_RestoreThread(ts);
    return PyLong_FromLong(st);
  }
};

// f's result, or None where it says nothing (or throws: the checks in Python say why).
template <typename F>
static PyObject *try_call(F f) {
  PyObject *r = nullptr;
  try {
    r = f();
  } catch (...) {
  }
  if (r) return r;
  PyErr_Clear();
  Py_RETURN_NONE;
}

typedef PyObject *const *args_t;

// (entries, ctx, device, x, inv, rows, stream)
static PyObject *dispatch(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 7);
    int xt = 0, rt = 0, k = 0;
    const at::Tensor *x = c.fine ? c.rows(a[3], &xt) : nullptr, *rows = c.fine ? c.rows(a[5], &rt) : nullptr;
    if (!c.fine || rows->size(1) != x->size(1)) return nullptr;
    const at::Tensor *inv = c.pairs(a[4], x->size(0), &k);
    if (!c.fine) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->dispatch(c.ctx, x->const_data_ptr(), xt, (const int32_t *)inv->const_data_ptr(), (int)x->size(0), k,
                             (int)x->size(1), (int)rows->size(0), rows->data_ptr(), rt, stream);
    });
  });
}

// (entries, ctx, device, drows, inv, dx, stream)
static PyObject *dispatch_grad(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 7);
    int xt = 0, rt = 0, k = 0;
    const at::Tensor *rows = c.fine ? c.rows(a[3], &rt) : nullptr, *dx = c.fine ? c.rows(a[5], &xt) : nullptr;
    if (!c.fine || rows->size(1) != dx->size(1)) return nullptr;
    const at::Tensor *inv = c.pairs(a[4], dx->size(0), &k);
    if (!c.fine) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->dispatch_grad(c.ctx, rows->const_data_ptr(), rt, (int)rows->size(0),
                                  (const int32_t *)inv->const_data_ptr(), (int)dx->size(0), k, (int)dx->size(1),
                                  dx->data_ptr(), xt, stream);
    });
  });
}

// (entries, ctx, device, rows, wts, inv, out, stream)
static PyObject *combine(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 8);
    int ot = 0, rt = 0, k = 0;
    const at::Tensor *rows = c.fine ? c.rows(a[3], &rt) : nullptr, *out = c.fine ? c.rows(a[6], &ot) : nullptr;
    if (!c.fine || rows->size(1) != out->size(1)) return nullptr;
    const int64_t T = out->size(0);
    const at::Tensor *inv = c.pairs(a[5], T, &k);
    const at::Tensor *wts = c.fine ? c.array(a[4], at::kFloat, {T, k}) : nullptr;
    if (!c.fine) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->combine(c.ctx, rows->const_data_ptr(), rt, (int)rows->size(0), (const float *)wts->const_data_ptr(),
                            (const int32_t *)inv->const_data_ptr(), (int)T, k, (int)out->size(1), out->data_ptr(), ot,
                            stream);
    });
  });
}

// (entries, ctx, device, dout, rows, wts, inv, drows, dwts, stream)
static PyObject *combine_grad(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 10);
    int dt = 0, rt = 0, k = 0;
    const at::Tensor *dout = c.fine ? c.rows(a[3], &dt) : nullptr, *rows = c.fine ? c.rows(a[4], &rt) : nullptr;
    if (!c.fine || rows->size(1) != dout->size(1)) return nullptr;
    const int64_t T = dout->size(0);
    const at::Tensor *inv = c.pairs(a[6], T, &k);
    const at::Tensor *wts = c.fine ? c.array(a[5], at::kFloat, {T, k}) : nullptr;
    const at::Tensor *drows = c.fine ? c.array(a[7], rows->scalar_type(), rows->sizes()) : nullptr;
    const at::Tensor *dwts = c.fine ? c.array(a[8], at::kFloat, {T, k}) : nullptr;
    if (!c.fine) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->combine_grad(c.ctx, dout->const_data_ptr(), dt, rows->const_data_ptr(), rt, (int)rows->size(0),
                                 (const float *)wts->const_data_ptr(), (const int32_t *)inv->const_data_ptr(), (int)T, k,
                                 (int)dout->size(1), drows->data_ptr(), (float *)dwts->data_ptr(), stream);
    });
  });
}

// (entries, ctx, device, x, q, scale, stream)
static PyObject *quantize_i8(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 7);
    int xt = 0;
    const at::Tensor *x = c.fine ? c.rows(a[3], &xt) : nullptr;
    if (!c.fine) return nullptr;
    const at::Tensor *q = c.array(a[4], at::kChar, x->sizes());
    const at::Tensor *scale = c.fine ? c.array(a[5], at::kFloat, {x->size(0)}) : nullptr;
    if (!c.fine) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->quantize_i8(c.ctx, x->const_data_ptr(), xt, (int)x->size(0), (int)x->size(1), (int8_t *)q->data_ptr(),
                                (float *)scale->data_ptr(), stream);
    });
  });
}

// (entries, ctx, device, q, scale, w, w_scale, out, offsets or None, perm or None, k, swiglu, clamp, stream)
static PyObject *matmul_i8(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 14);
    if (!c.fine || !PyLong_Check(a[10]) || !PyFloat_Check(a[12])) return nullptr;
    const long k = PyLong_AsLong(a[10]);
    const int swiglu = PyObject_IsTrue(a[11]);
    if (PyErr_Occurred() || swiglu < 0 || k < INT_MIN || k > INT_MAX) return nullptr;
    const float clamp = (float)PyFloat_AS_DOUBLE(a[12]);
    int ot = 0;
    const bool grouped = a[8] != Py_None;
    const at::Tensor *q = c.tensor(a[3]), *w = c.fine ? c.tensor(a[5]) : nullptr;
    const at::Tensor *out = c.fine ? c.rows(a[7], &ot) : nullptr;
    if (!c.fine || q->scalar_type() != at::kChar || q->dim() != 2 || w->scalar_type() != at::kChar ||
        w->dim() != (grouped ? 3 : 2))
      return nullptr;
    const int64_t S = q->size(0), K = q->size(1), M = out->size(0), E = grouped ? w->size(0) : 1, N = w->size(w->dim() - 2);
    const at::Tensor *offsets = grouped ? c.array(a[8], at::kInt, {E + 1}) : nullptr;
    if (!c.fine || w->size(w->dim() - 1) != K || (swiglu && N % 2) || out->size(1) != (swiglu ? N / 2 : N)) return nullptr;
    const at::Tensor *scale = c.array(a[4], at::kFloat, {S}), *perm = nullptr;
    const at::Tensor *w_scale = !c.fine    ? nullptr
                                : grouped ? c.array(a[6], at::kFloat, {E, N})
                                           : c.array(a[6], at::kFloat, {N});
    if (a[9] != Py_None) perm = c.fine ? c.array(a[9], at::kInt, {M}) : nullptr;
    else c.fine = c.fine && k == 1 && S == M;
    if (!c.fine) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->matmul_i8(c.ctx, (const int8_t *)q->const_data_ptr(), (const float *)scale->const_data_ptr(), (int)S,
                              (const int8_t *)w->const_data_ptr(), (const float *)w_scale->const_data_ptr(), (int)E,
                              offsets ? (const int32_t *)offsets->const_data_ptr() : nullptr,
                              perm ? (const int32_t *)perm->const_data_ptr() : nullptr, (int)k, (int)M, (int)N, (int)K,
                              swiglu ? MOE_MM_SWIGLU : 0, clamp, out->data_ptr(), ot, stream);
    });
  });
}

#define METHOD(f) {#f, (PyCFunction)(void (*)())f, METH_FASTCALL, nullptr}
static PyMethodDef methods[] = {METHOD(dispatch),     METHOD(dispatch_grad), METHOD(combine), METHOD(combine_grad),
                                METHOD(quantize_i8), METHOD(matmul_i8),
                                {"set_current_stream", set_current_stream, METH_O, nullptr},
                                {nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "moe_torch", nullptr, -1, methods};

PyMODINIT_FUNC PyInit_moe_torch() {
  PyObject *m = PyModule_Create(&module);
  if (m) PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION);  // it is built against
  return m;
}

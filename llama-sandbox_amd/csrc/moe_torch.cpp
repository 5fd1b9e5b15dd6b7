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
  decltype(&moe_rms_norm) rms_norm;
  decltype(&moe_rms_norm_grad) rms_norm_grad;
  decltype(&moe_route_groups) route_groups;
  decltype(&moe_route_grad) route_grad;
  decltype(&moe_adapters) adapters;
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
  const at::Tensor *rows(PyObject *o, int *type, int dim = 2) {
    const at::Tensor *t = tensor(o);
    if (!t) return t;
    const at::ScalarType s = t->scalar_type();
    *type = s == at::kFloat ? MOE_GGML_F32 : s == at::kHalf ? MOE_GGML_F16 : MOE_GGML_BF16;
    fine = t->dim() == dim && (s == at::kFloat || s == at::kHalf || s == at::kBFloat16);
    return t;
  }
  // ... of this shape
  const at::Tensor *rows_of(PyObject *o, int *type, at::IntArrayRef shape) {
    const at::Tensor *t = rows(o, type, (int)shape.size());
    if (t && fine) fine = t->sizes() == shape;
    return t;
  }
  // ... of a size that the library checks
  const at::Tensor *workspace(PyObject *o) {
    const at::Tensor *t = tensor(o);
    if (t) fine = t->scalar_type() == at::kFloat && t->dim() == 1;
    return t;
  }
  // a whole number and a float of the arguments
  int whole(PyObject *o) {
    const long v = fine && PyLong_Check(o) ? PyLong_AsLong(o) : (fine = false, 0);
    if (PyErr_Occurred() || v < INT_MIN || v > INT_MAX) fine = false;
    return (int)v;
  }
  float real(PyObject *o) {
    if (!fine || !PyFloat_Check(o)) return fine = false, 0.0f;
    return (float)PyFloat_AS_DOUBLE(o);
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

static void *data(const at::Tensor *t) { return t ? t->data_ptr() : nullptr; }
template <typename T>
static const T *read(const at::Tensor *t) { return t ? (const T *)t->const_data_ptr() : nullptr; }

// (entries, ctx, device, x, w, eps, residual, total, y, q, scale, rstd, stream); from residual on None: absent
static PyObject *rms_norm(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 13);
    int xt = 0, wt = 0, rt = 0, tt = 0, yt = 0;
    const at::Tensor *x = c.fine ? c.rows(a[3], &xt) : nullptr;
    if (!c.fine) return nullptr;
    const int64_t T = x->size(0), H = x->size(1);
    const at::Tensor *w = c.rows_of(a[4], &wt, {H});
    const float eps = c.real(a[5]);
    auto rows = [&](PyObject *o, int *type) { return !c.fine || o == Py_None ? nullptr : c.rows_of(o, type, {T, H}); };
    auto column = [&](PyObject *o) { return !c.fine || o == Py_None ? nullptr : c.array(o, at::kFloat, {T}); };
    const at::Tensor *res = rows(a[6], &rt), *total = rows(a[7], &tt), *y = rows(a[8], &yt);
    const at::Tensor *q = !c.fine || a[9] == Py_None ? nullptr : c.array(a[9], at::kChar, {T, H});
    const at::Tensor *scale = column(a[10]), *rstd = column(a[11]);
    if (!c.fine || !res != !total || rt != tt || !q != !scale || (!y && !q)) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->rms_norm(c.ctx, x->const_data_ptr(), xt, read<void>(res), data(total), rt, w->const_data_ptr(), wt, eps,
                             (int)T, (int)H, data(y), yt, (int8_t *)data(q), (float *)data(scale), (float *)data(rstd), stream);
    });
  });
}

// (entries, ctx, device, dy, h, w, rstd, dx, dw, part, dres or None, stream)
static PyObject *rms_norm_grad(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 12);
    int dt = 0, ht = 0, wt = 0, xt = 0, rt = 0;
    const at::Tensor *dy = c.fine ? c.rows(a[3], &dt) : nullptr;
    if (!c.fine) return nullptr;
    const int64_t T = dy->size(0), H = dy->size(1);
    const at::Tensor *h = c.rows_of(a[4], &ht, {T, H});
    const at::Tensor *w = c.fine ? c.rows_of(a[5], &wt, {H}) : nullptr;
    const at::Tensor *rstd = c.fine ? c.array(a[6], at::kFloat, {T}) : nullptr;
    const at::Tensor *dx = c.fine ? c.rows_of(a[7], &xt, {T, H}) : nullptr;
    const at::Tensor *dw = c.fine ? c.array(a[8], at::kFloat, {H}) : nullptr;
    const at::Tensor *part = c.fine ? c.workspace(a[9]) : nullptr;
    const at::Tensor *dres = !c.fine || a[10] == Py_None ? nullptr : c.rows_of(a[10], &rt, {T, H});
    if (!c.fine || (dres && rt != xt)) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->rms_norm_grad(c.ctx, dy->const_data_ptr(), dt, h->const_data_ptr(), ht, w->const_data_ptr(), wt,
                                  read<float>(rstd), read<void>(dres), (int)T, (int)H, dx->data_ptr(), xt, (float *)data(dw),
                                  (float *)data(part), (size_t)part->numel(), stream);
    });
  });
}

// (entries, ctx, device, logits, k, mode, norm, scale, ids, wts, bias or None, n_group, keep, top, scores or None, stream)
static PyObject *route_groups(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 16);
    int lt = 0;
    const at::Tensor *l = c.fine ? c.rows(a[3], &lt) : nullptr;
    if (!c.fine) return nullptr;
    const int64_t T = l->size(0), E = l->size(1);
    const int k = c.whole(a[4]), mode = c.whole(a[5]), norm = PyObject_IsTrue(a[6]);
    const float scale = c.real(a[7]);
    const at::Tensor *ids = c.fine ? c.array(a[8], at::kInt, {T, k}) : nullptr;
    const at::Tensor *wts = c.fine ? c.array(a[9], at::kFloat, {T, k}) : nullptr;
    const at::Tensor *bias = !c.fine || a[10] == Py_None ? nullptr : c.array(a[10], at::kFloat, {E});
    const int n_group = c.whole(a[11]), keep = c.whole(a[12]), top = c.whole(a[13]);
    const at::Tensor *scores = !c.fine || a[14] == Py_None ? nullptr : c.array(a[14], at::kFloat, {T, E});
    if (!c.fine || norm < 0) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->route_groups(c.ctx, l->const_data_ptr(), lt, read<float>(bias), (int)T, (int)E, k, mode, n_group, keep, top,
                                 norm, scale, (int32_t *)data(ids), (float *)data(wts), (float *)data(scores), stream);
    });
  });
}

// (entries, ctx, device, logits, ids, dwts, mode, norm, scale, dlogits, dscores or None, stream)
static PyObject *route_grad(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 12);
    int lt = 0, dt = 0;
    const at::Tensor *l = c.fine ? c.rows(a[3], &lt) : nullptr;
    if (!c.fine) return nullptr;
    const int64_t T = l->size(0), E = l->size(1);
    const at::Tensor *ids = c.tensor(a[4]);
    if (!c.fine || ids->scalar_type() != at::kInt || ids->dim() != 2 || ids->size(0) != T) return nullptr;
    const int64_t k = ids->size(1);
    const at::Tensor *dwts = c.array(a[5], at::kFloat, {T, k});
    const int mode = c.whole(a[6]), norm = PyObject_IsTrue(a[7]);
    const float scale = c.real(a[8]);
    const at::Tensor *dl = c.fine ? c.rows_of(a[9], &dt, {T, E}) : nullptr;
    const at::Tensor *ds = !c.fine || a[10] == Py_None ? nullptr : c.array(a[10], at::kFloat, {T, E});
    if (!c.fine || norm < 0) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->route_grad(c.ctx, l->const_data_ptr(), lt, read<int32_t>(ids), read<float>(dwts), read<float>(ds), (int)T,
                               (int)E, (int)k, mode, norm, scale, dl->data_ptr(), dt, stream);
    });
  });
}

// (entries, ctx, device, x, a, b, scale or None, offsets, perm, base, out, mid, stream)
static PyObject *adapters(PyObject *, args_t a, Py_ssize_t n) {
  return try_call([&]() -> PyObject * {
    call c(a, n, 13);
    int xt = 0, at_ = 0, bt = 0, st = 0, ot = 0;
    const at::Tensor *x = c.fine ? c.rows(a[3], &xt) : nullptr, *A = c.fine ? c.rows(a[4], &at_, 3) : nullptr;
    const at::Tensor *B = c.fine ? c.rows(a[5], &bt, 3) : nullptr;
    if (!c.fine || at_ != xt || bt != xt) return nullptr;
    const int64_t M = x->size(0), K = x->size(1), na = A->size(0), R = A->size(1), N = B->size(1);
    if (A->size(2) != K || B->size(0) != na || B->size(2) != R) return nullptr;
    const at::Tensor *scale = a[6] == Py_None ? nullptr : c.array(a[6], at::kFloat, {na});
    const at::Tensor *offsets = c.fine ? c.array(a[7], at::kInt, {na + 1}) : nullptr;
    const at::Tensor *perm = c.fine ? c.array(a[8], at::kInt, {M}) : nullptr;
    const at::Tensor *base = c.fine ? c.rows_of(a[9], &st, {M, N}) : nullptr;
    const at::Tensor *out = c.fine ? c.rows_of(a[10], &ot, {M, N}) : nullptr;
    const at::Tensor *mid = c.fine ? c.workspace(a[11]) : nullptr;
    if (!c.fine || st != ot) return nullptr;
    return c.make([&](void *stream) {
      return c.lib->adapters(c.ctx, x->const_data_ptr(), A->const_data_ptr(), B->const_data_ptr(), xt, read<float>(scale),
                             (int)na, read<int32_t>(offsets), read<int32_t>(perm), (int)M, (int)K, (int)R, (int)N,
                             base->const_data_ptr(), out->data_ptr(), ot, (float *)data(mid), (size_t)mid->numel(), stream);
    });
  });
}

#define METHOD(f) {#f, (PyCFunction)(void (*)())f, METH_FASTCALL, nullptr}
static PyMethodDef methods[] = {METHOD(dispatch),     METHOD(dispatch_grad), METHOD(combine), METHOD(combine_grad),
                                METHOD(quantize_i8),  METHOD(matmul_i8),     METHOD(rms_norm), METHOD(rms_norm_grad),
                                METHOD(route_groups), METHOD(route_grad),    METHOD(adapters),
                                {"set_current_stream", set_current_stream, METH_O, nullptr},
                                {nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "moe_torch", nullptr, -1, methods};

PyMODINIT_FUNC PyInit_moe_torch() {
  PyObject *m = PyModule_Create(&module);
  if (m) PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION);  // it is built against
  return m;
}

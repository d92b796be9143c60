/*
 * Direct Python entry points of libtb200's window attention, paged attention and gated residual RMSNorm
 * calls: the same arguments as in include/tb200.h, with pointers as integers (None: null) and stride arrays
 * as tuples. A ctypes call with twenty to forty arguments converts them in 5 us, as much as the launch of a
 * small kernel; here the conversion takes well under one. The library itself keeps its C ABI.
 */
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include "../../include/tb200.h"

/* Arguments in order; the first failure sticks. */
typedef struct {
  PyObject* const* args;
  Py_ssize_t n, at;
  int failed;
} Args;

static PyObject* next_arg(Args* a) {
  if (a->failed) return NULL;
  if (a->at >= a->n) {
    PyErr_SetString(PyExc_TypeError, "too few arguments");
    a->failed = 1;
    return NULL;
  }
  return a->args[a->at++];
}
static int64_t integer(Args* a) {
  PyObject* o = next_arg(a);
  if (!o) return 0;
  int64_t v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) a->failed = 1;
  return v;
}
static void* pointer(Args* a) {
  PyObject* o = next_arg(a);
  if (!o || o == Py_None) return NULL;
  void* v = PyLong_AsVoidPtr(o);
  if (!v && PyErr_Occurred()) a->failed = 1;
  return v;
}
static float real(Args* a) {
  PyObject* o = next_arg(a);
  if (!o) return 0.f;
  double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) a->failed = 1;
  return (float)v;
}
static int64_t* strides(Args* a, int64_t* out, Py_ssize_t count) {
  PyObject* o = next_arg(a);
  if (!o) return out;
  if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != count) {
    PyErr_Format(PyExc_TypeError, "a tuple of %zd strides is expected", count);
    a->failed = 1;
    return out;
  }
  for (Py_ssize_t i = 0; i < count; ++i) {
    out[i] = PyLong_AsLongLong(PyTuple_GET_ITEM(o, i));
    if (out[i] == -1 && PyErr_Occurred()) a->failed = 1;
  }
  return out;
}
static int ready(Args* a) {
  if (!a->failed && a->at != a->n) {
    PyErr_SetString(PyExc_TypeError, "too many arguments");
    a->failed = 1;
  }
  return !a->failed;
}

#define BEGIN                     \
  Args a = {args, n, 0, 0};       \
  int status = 0;                 \
  (void)self
/* (the lock is released around the call: a launch may wait for room in the stream) */
#define CALL(call)                \
  if (!ready(&a)) return NULL;    \
  Py_BEGIN_ALLOW_THREADS          \
  status = call;                  \
  Py_END_ALLOW_THREADS            \
  return PyLong_FromLong(status)

static PyObject* gated_residual_rms_norm_fwd(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void *h = pointer(&a), *y = pointer(&a), *rms1 = pointer(&a), *rms2 = pointer(&a), *x = pointer(&a), *r = pointer(&a);
  void *w1 = pointer(&a), *w2 = pointer(&a), *gate = pointer(&a);
  int64_t rows = integer(&a), cols = integer(&a), per_gate = integer(&a);
  float scale = real(&a), eps = real(&a);
  int dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_gated_residual_rms_norm_fwd(h, y, rms1, rms2, x, r, w1, w2, gate, rows, cols, per_gate, scale, eps, dtype, stream));
}

static PyObject* gated_residual_rms_norm_bwd(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void* p[15];
  for (int i = 0; i < 15; ++i) p[i] = pointer(&a);
  size_t bytes = (size_t)integer(&a);
  int64_t rows = integer(&a), cols = integer(&a), per_gate = integer(&a);
  float scale = real(&a), eps = real(&a);
  int dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_gated_residual_rms_norm_bwd(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], p[10], p[11], p[12], p[13],
                                         p[14], bytes, rows, cols, per_gate, scale, eps, dtype, stream));
}

static PyObject* window_attention_fwd(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void *out = pointer(&a), *lse = pointer(&a), *q = pointer(&a), *k = pointer(&a), *v = pointer(&a);
  int64_t d[5], s[4][4];
  for (int i = 0; i < 5; ++i) d[i] = integer(&a);
  for (int i = 0; i < 4; ++i) strides(&a, s[i], 4);
  int64_t window = integer(&a), sinks = integer(&a);
  float scale = real(&a);
  int dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_window_attention_fwd(out, lse, q, k, v, d[0], d[1], d[2], d[3], d[4], s[0], s[1], s[2], s[3], window, sinks, scale,
                                  dtype, stream));
}

static PyObject* window_attention_bwd(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void* p[10];
  for (int i = 0; i < 10; ++i) p[i] = pointer(&a);
  size_t bytes = (size_t)integer(&a);
  int64_t d[5], s[8][4];
  for (int i = 0; i < 5; ++i) d[i] = integer(&a);
  for (int i = 0; i < 8; ++i) strides(&a, s[i], 4);
  int64_t window = integer(&a), sinks = integer(&a);
  float scale = real(&a);
  int dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_window_attention_bwd(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], bytes, d[0], d[1], d[2], d[3], d[4],
                                  s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], window, sinks, scale, dtype, stream));
}

static PyObject* window_attention_fwd_low(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void *out = pointer(&a), *low = pointer(&a), *lse = pointer(&a), *q = pointer(&a), *k = pointer(&a), *v = pointer(&a);
  int64_t d[5], s[4][4];
  for (int i = 0; i < 5; ++i) d[i] = integer(&a);
  for (int i = 0; i < 4; ++i) strides(&a, s[i], 4);
  int64_t window = integer(&a), sinks = integer(&a);
  float scale = real(&a);
  int dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_window_attention_fwd_low(out, low, lse, q, k, v, d[0], d[1], d[2], d[3], d[4], s[0], s[1], s[2], s[3], window, sinks,
                                      scale, dtype, stream));
}

static PyObject* window_attention_bwd_low(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void* p[11];
  for (int i = 0; i < 11; ++i) p[i] = pointer(&a);
  size_t bytes = (size_t)integer(&a);
  int64_t d[5], s[8][4];
  for (int i = 0; i < 5; ++i) d[i] = integer(&a);
  for (int i = 0; i < 8; ++i) strides(&a, s[i], 4);
  int64_t window = integer(&a), sinks = integer(&a);
  float scale = real(&a);
  int dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_window_attention_bwd_low(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], p[10], bytes, d[0], d[1], d[2],
                                      d[3], d[4], s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7], window, sinks, scale, dtype,
                                      stream));
}

static PyObject* paged_attention(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void* p[8];
  for (int i = 0; i < 8; ++i) p[i] = pointer(&a);
  size_t bytes = (size_t)integer(&a);
  int64_t d[9], q[3], k[4], v[4], o[3], m[4];
  for (int i = 0; i < 9; ++i) d[i] = integer(&a);
  strides(&a, q, 3);
  strides(&a, k, 4);
  strides(&a, v, 4);
  strides(&a, o, 3);
  for (int i = 0; i < 4; ++i) m[i] = integer(&a);
  float scale = real(&a);
  int zero_rest = (int)integer(&a), dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_paged_attention(p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], bytes, d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7],
                             d[8], q, k, v, o, m[0], m[1], m[2], m[3], scale, zero_rest, dtype, stream));
}

static PyObject* paged_cache_append(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  BEGIN;
  void* p[7];
  for (int i = 0; i < 7; ++i) p[i] = pointer(&a);
  int64_t d[8], kc[4], vc[4], k[3], v[3];
  for (int i = 0; i < 8; ++i) d[i] = integer(&a);
  strides(&a, kc, 4);
  strides(&a, vc, 4);
  strides(&a, k, 3);
  strides(&a, v, 3);
  int dtype = (int)integer(&a);
  void* stream = pointer(&a);
  CALL(tb200_paged_cache_append(p[0], p[1], p[2], p[3], p[4], p[5], p[6], d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7], kc, vc, k,
                                v, dtype, stream));
}

#define METHOD(name) {"tb200_" #name, (PyCFunction)(void (*)(void))name, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {
    METHOD(gated_residual_rms_norm_fwd), METHOD(gated_residual_rms_norm_bwd), METHOD(window_attention_fwd),
    METHOD(window_attention_bwd),        METHOD(window_attention_fwd_low),    METHOD(window_attention_bwd_low),
    METHOD(paged_attention),             METHOD(paged_cache_append),
    {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_fastcall", NULL, -1, methods, NULL, NULL, NULL, NULL};
PyMODINIT_FUNC PyInit__fastcall(void) { return PyModule_Create(&module); }

/* Direct calls of the 4-bit and rotary entry points for the Python binding (module `hom_calls`).
 *
 * ctypes takes 1.3 to 2.5 us to convert the 7 to 15 arguments of such a call, on top of the 1.7 us
 * that a launch costs the host, and the smallest of these operators run 1.5 to 2.5 us on the
 * device: a loop of them was bound by the conversion.  Here a memref argument is two attribute
 * reads.  Optional: built when the interpreter's headers are there (stable ABI), and the binding
 * goes through ctypes without it.
 *
 * Every function returns None, or the error code that the entry point recorded. */
#define PY_SSIZE_T_CLEAN
#define Py_LIMITED_API 0x030A0000
#include <Python.h>

#include "hom_nvgpu_runner_utils.h"

static PyTypeObject *memref_type;    /* the binding's MemRef */
static PyObject *to_memref;          /* makes one of a tensor */
static PyObject *s_rank, *s_address; /* attribute names */

enum { kMaxMemrefs = 6 };
typedef struct {
  int64_t rank[kMaxMemrefs];
  void *descriptor[kMaxMemrefs];
  PyObject *made[kMaxMemrefs]; /* converted here, released after the call */
  int count;
} Memrefs;

static void release(Memrefs *m) {
  for (int i = 0; i < m->count; ++i) Py_XDECREF(m->made[i]);
}

static int take(Memrefs *m, PyObject *x) {
  const int i = m->count++;
  m->rank[i] = 0;
  m->descriptor[i] = NULL;
  m->made[i] = NULL;
  if (x == Py_None) return 1;
  if (Py_TYPE(x) != memref_type) {
    x = m->made[i] = PyObject_CallFunctionObjArgs(to_memref, x, NULL);
    if (!x) return 0;
  }
  PyObject *rank = PyObject_GetAttr(x, s_rank);
  PyObject *address = rank ? PyObject_GetAttr(x, s_address) : NULL;
  if (address) {
    m->rank[i] = PyLong_AsLongLong(rank);
    m->descriptor[i] = PyLong_AsVoidPtr(address);
  }
  Py_XDECREF(rank);
  Py_XDECREF(address);
  return address && !PyErr_Occurred();
}

static int arguments(const char *name, Py_ssize_t have, Py_ssize_t want) {
  if (have == want) return 1;
  PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, want, have);
  return 0;
}

static PyObject *outcome(void) {
  const int code = homGetLastError();
  if (code == 0) Py_RETURN_NONE;
  return PyLong_FromLong(code);
}

typedef void (*Quantize)(int64_t, void *, bool, int64_t, void *, int64_t, void *);
static PyObject *quantize(Quantize call, const char *name, PyObject *const *args, Py_ssize_t n) {
  Memrefs m = {.count = 0};
  if (!arguments(name, n, 4)) return NULL;
  const int transposed = PyObject_IsTrue(args[3]);
  if (transposed < 0 || !take(&m, args[0]) || !take(&m, args[1]) || !take(&m, args[2])) {
    release(&m);
    return NULL;
  }
  Py_BEGIN_ALLOW_THREADS
  call(m.rank[0], m.descriptor[0], transposed != 0, m.rank[1], m.descriptor[1], m.rank[2], m.descriptor[2]);
  Py_END_ALLOW_THREADS
  release(&m);
  return outcome();
}

typedef void (*Dequantize)(int64_t, void *, int64_t, void *, int64_t, void *);
static PyObject *dequantize(Dequantize call, const char *name, PyObject *const *args, Py_ssize_t n) {
  Memrefs m = {.count = 0};
  if (!arguments(name, n, 3)) return NULL;
  if (!take(&m, args[0]) || !take(&m, args[1]) || !take(&m, args[2])) {
    release(&m);
    return NULL;
  }
  Py_BEGIN_ALLOW_THREADS
  call(m.rank[0], m.descriptor[0], m.rank[1], m.descriptor[1], m.rank[2], m.descriptor[2]);
  Py_END_ALLOW_THREADS
  release(&m);
  return outcome();
}

static PyObject *product(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  (void)self;
  Memrefs m = {.count = 0};
  if (!arguments("homGemmMxF4F16", n, 9)) return NULL;
  const long long activation = PyLong_AsLongLong(args[6]);
  const double alpha = PyFloat_AsDouble(args[7]), beta = PyFloat_AsDouble(args[8]);
  int ok = !PyErr_Occurred();
  for (int i = 0; ok && i < 6; ++i) ok = take(&m, args[i]);
  if (!ok) {
    release(&m);
    return NULL;
  }
  Py_BEGIN_ALLOW_THREADS
  homGemmMxF4F16(m.rank[0], m.descriptor[0], m.rank[1], m.descriptor[1], m.rank[2], m.descriptor[2], m.rank[3],
                 m.descriptor[3], m.rank[4], m.descriptor[4], m.rank[5], m.descriptor[5], activation, (float)alpha,
                 (float)beta);
  Py_END_ALLOW_THREADS
  release(&m);
  return outcome();
}

typedef void (*Rotary)(int64_t, void *, int64_t, void *, int64_t, void *, int64_t, void *, bool, bool, float);
static PyObject *rotary(Rotary call, const char *name, PyObject *const *args, Py_ssize_t n) {
  Memrefs m = {.count = 0};
  if (!arguments(name, n, 7)) return NULL;
  const int interleaved = PyObject_IsTrue(args[4]), backward = PyObject_IsTrue(args[5]);
  const double magnitude = PyFloat_AsDouble(args[6]);
  int ok = interleaved >= 0 && backward >= 0 && !PyErr_Occurred();
  for (int i = 0; ok && i < 4; ++i) ok = take(&m, args[i]);
  if (!ok) {
    release(&m);
    return NULL;
  }
  Py_BEGIN_ALLOW_THREADS
  call(m.rank[0], m.descriptor[0], m.rank[1], m.descriptor[1], m.rank[2], m.descriptor[2], m.rank[3], m.descriptor[3],
       interleaved != 0, backward != 0, (float)magnitude);
  Py_END_ALLOW_THREADS
  release(&m);
  return outcome();
}

#define FORWARD(NAME, THROUGH)                                                          \
  static PyObject *NAME##_(PyObject *self, PyObject *const *args, Py_ssize_t n) {       \
    (void)self;                                                                         \
    return THROUGH(NAME, #NAME, args, n);                                               \
  }
FORWARD(homQuantizeMxF4F16, quantize)
FORWARD(homQuantizeMxF4F32, quantize)
FORWARD(homDequantizeMxF4F16, dequantize)
FORWARD(homDequantizeMxF4F32, dequantize)
FORWARD(homRotaryF16, rotary)
FORWARD(homRotaryF32, rotary)

/* bind(MemRef, MemRef.of): the descriptor type, with the attributes `rank` and `address`, and what
 * makes one of anything else. */
static PyObject *bind(PyObject *self, PyObject *const *args, Py_ssize_t n) {
  (void)self;
  if (!arguments("bind", n, 2)) return NULL;
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  Py_XDECREF((PyObject *)memref_type);
  Py_XDECREF(to_memref);
  memref_type = (PyTypeObject *)args[0];
  to_memref = args[1];
  Py_RETURN_NONE;
}

#define METHOD(NAME, FN) {NAME, (PyCFunction)(void (*)(void))FN, METH_FASTCALL, NULL}
static PyMethodDef methods[] = {
    METHOD("bind", bind),
    METHOD("homQuantizeMxF4F16", homQuantizeMxF4F16_),
    METHOD("homQuantizeMxF4F32", homQuantizeMxF4F32_),
    METHOD("homDequantizeMxF4F16", homDequantizeMxF4F16_),
    METHOD("homDequantizeMxF4F32", homDequantizeMxF4F32_),
    METHOD("homGemmMxF4F16", product),
    METHOD("homRotaryF16", homRotaryF16_),
    METHOD("homRotaryF32", homRotaryF32_),
    {NULL, NULL, 0, NULL},
};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "hom_calls", NULL, -1, methods, NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit_hom_calls(void) {
  s_rank = PyUnicode_InternFromString("rank");
  s_address = PyUnicode_InternFromString("address");
  return s_rank && s_address ? PyModule_Create(&module) : NULL;
}

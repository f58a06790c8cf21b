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

/* One for each time the module is loaded: every copy of the package has a MemRef of its own. */
typedef struct {
  PyTypeObject *memref_type;    /* the binding's MemRef */
  PyObject *to_memref;          /* makes one of a tensor */
  PyObject *s_rank, *s_address; /* attribute names */
} State;

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

static int take(const State *state, Memrefs *m, PyObject *x) {
  const int i = m->count++;
  m->rank[i] = 0;
  m->descriptor[i] = NULL;
  m->made[i] = NULL;
  if (x == Py_None) return 1;
  if (Py_TYPE(x) != state->memref_type) {
    if (!state->memref_type) {
      PyErr_SetString(PyExc_RuntimeError, "hom_calls: not bound");
      return 0;
    }
    if (!PyType_IsSubtype(Py_TYPE(x), state->memref_type)) {
      x = m->made[i] = PyObject_CallFunctionObjArgs(state->to_memref, x, NULL);
      if (!x) return 0;
    }
  }
  PyObject *rank = PyObject_GetAttr(x, state->s_rank);
  PyObject *address = rank ? PyObject_GetAttr(x, state->s_address) : NULL;
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
static PyObject *quantize(PyObject *self, Quantize call, const char *name, PyObject *const *args, Py_ssize_t n) {
  const State *state = PyModule_GetState(self);
  Memrefs m = {.count = 0};
  if (!arguments(name, n, 4)) return NULL;
  const int transposed = PyObject_IsTrue(args[3]);
  if (transposed < 0 || !take(state, &m, args[0]) || !take(state, &m, args[1]) || !take(state, &m, args[2])) {
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
static PyObject *dequantize(PyObject *self, Dequantize call, const char *name, PyObject *const *args, Py_ssize_t n) {
  const State *state = PyModule_GetState(self);
  Memrefs m = {.count = 0};
  if (!arguments(name, n, 3)) return NULL;
  if (!take(state, &m, args[0]) || !take(state, &m, args[1]) || !take(state, &m, args[2])) {
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
  const State *state = PyModule_GetState(self);
  Memrefs m = {.count = 0};
  if (!arguments("homGemmMxF4F16", n, 9)) return NULL;
  const long long activation = PyLong_AsLongLong(args[6]);
  const double alpha = PyFloat_AsDouble(args[7]), beta = PyFloat_AsDouble(args[8]);
  int ok = !PyErr_Occurred();
  for (int i = 0; ok && i < 6; ++i) ok = take(state, &m, args[i]);
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
static PyObject *rotary(PyObject *self, Rotary call, const char *name, PyObject *const *args, Py_ssize_t n) {
  const State *state = PyModule_GetState(self);
  Memrefs m = {.count = 0};
  if (!arguments(name, n, 7)) return NULL;
  const int interleaved = PyObject_IsTrue(args[4]), backward = PyObject_IsTrue(args[5]);
  const double magnitude = PyFloat_AsDouble(args[6]);
  int ok = interleaved >= 0 && backward >= 0 && !PyErr_Occurred();
  for (int i = 0; ok && i < 4; ++i) ok = take(state, &m, args[i]);
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
    return THROUGH(self, NAME, #NAME, args, n);                                         \
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
  State *state = PyModule_GetState(self);
  if (!arguments("bind", n, 2)) return NULL;
  if (!PyType_Check(args[0])) {
    PyErr_SetString(PyExc_TypeError, "bind takes a class and what makes one of its objects");
    return NULL;
  }
  PyObject *type = (PyObject *)state->memref_type, *make = state->to_memref;
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  state->memref_type = (PyTypeObject *)args[0];
  state->to_memref = args[1];
  Py_XDECREF(type);
  Py_XDECREF(make);
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

static int execute(PyObject *self) {
  State *state = PyModule_GetState(self);
  state->s_rank = PyUnicode_InternFromString("rank");
  state->s_address = PyUnicode_InternFromString("address");
  return state->s_rank && state->s_address ? 0 : -1;
}

static int traverse(PyObject *self, visitproc visit, void *arg) {
  State *state = PyModule_GetState(self);
  Py_VISIT(state->memref_type);
  Py_VISIT(state->to_memref);
  return 0;
}

static int clear(PyObject *self) {
  State *state = PyModule_GetState(self);
  Py_CLEAR(state->memref_type);
  Py_CLEAR(state->to_memref);
  Py_CLEAR(state->s_rank);
  Py_CLEAR(state->s_address);
  return 0;
}

static void release_state(void *self) { clear(self); }

static PyModuleDef_Slot slots[] = {{Py_mod_exec, execute}, {0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "hom_calls", NULL, sizeof(State), methods, slots, traverse, clear,
                                    release_state};

PyMODINIT_FUNC PyInit_hom_calls(void) { return PyModuleDef_Init(&module); }

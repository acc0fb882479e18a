// Direct calls of the entry points that single decoding steps go through, for
// Python.  ctypes converts an argument in about 0.15 us, which for 20 to 36 of
// them is more than the launch itself; here an argument list is read from the
// interpreter's own array.  The module holds no code of the library: bind()
// gives it the addresses of the one that is loaded.
//
// Arguments are ints (pointers too; None is NULL), bools and floats, as in
// hier_b200.h; an int that its C type cannot hold is refused.

#define PY_SSIZE_T_CLEAN
#define Py_LIMITED_API 0x030A0000
#include <Python.h>
#include <stdint.h>
#include <string.h>

#include "hier_b200.h"

enum { kMaxArgs = 40 };

typedef struct {
  int64_t w[kMaxArgs];
  float f;  // no entry has more than one
} words;

// `sig` names the parameters: p pointer, q int64, i int32, f float
static int read_words(const char* name, const char* sig, PyObject* const* a, Py_ssize_t n, words* out) {
  if (n != (Py_ssize_t)strlen(sig)) {
    PyErr_Format(PyExc_TypeError, "%s takes %zd arguments, got %zd", name, (Py_ssize_t)strlen(sig), n);
    return 0;
  }
  for (Py_ssize_t i = 0; i < n; ++i) {
    if (sig[i] == 'f') {
      out->f = (float)PyFloat_AsDouble(a[i]);
      if (out->f == -1.f && PyErr_Occurred()) return 0;
      continue;
    }
    if (sig[i] == 'p' && a[i] == Py_None) {
      out->w[i] = 0;
      continue;
    }
    const long long v = PyLong_AsLongLong(a[i]);
    if (v == -1 && PyErr_Occurred()) return 0;
    if (sig[i] == 'i' && (v < INT32_MIN || v > INT32_MAX)) {
      PyErr_Format(PyExc_ValueError, "%s: argument %zd (%lld) passes 32 bits", name, i, v);
      return 0;
    }
    out->w[i] = v;
  }
  return 1;
}

#define P(i) ((void*)(uintptr_t)x.w[i])
#define Q(i) (x.w[i])
#define I(i) ((int32_t)x.w[i])

// One entry: its bound address, and a method that reads `SIG` (its doc string
// too) and calls it.
#define ENTRY(NAME, SIG, ...)                                                              \
  static const char SIG_##NAME[] = SIG;                                                    \
  static __typeof__(&NAME) at_##NAME;                                                      \
  static PyObject* py_##NAME(PyObject* self, PyObject* const* a, Py_ssize_t n) {           \
    words x;                                                                               \
    int rc;                                                                                \
    (void)self;                                                                            \
    if (!read_words(#NAME, SIG_##NAME, a, n, &x)) return NULL;                                    \
    if (!at_##NAME) {                                                                      \
      PyErr_SetString(PyExc_RuntimeError, #NAME " is not bound");                          \
      return NULL;                                                                         \
    }                                                                                      \
    Py_BEGIN_ALLOW_THREADS rc = at_##NAME(__VA_ARGS__);                                    \
    Py_END_ALLOW_THREADS return PyLong_FromLong(rc);                                       \
  }

ENTRY(hier_head_norm_rope, "pqpqqiiippipqpfpqpqpqpqipp", P(0), Q(1), P(2), Q(3), Q(4), I(5), I(6),
      I(7), P(8), P(9), I(10), P(11), Q(12), P(13), x.f, P(15), Q(16), P(17), Q(18), P(19), Q(20),
      P(21), Q(22), I(23), P(24), P(25))
ENTRY(hier_head_norm_rope_bwd, "pqpqqiiippipqpfpqpqpqpqpipppp", P(0), Q(1), P(2), Q(3), Q(4), I(5),
      I(6), I(7), P(8), P(9), I(10), P(11), Q(12), P(13), x.f, P(15), Q(16), P(17), Q(18), P(19),
      Q(20), P(21), Q(22), P(23), I(24), P(25), P(26), P(27), P(28))
ENTRY(hier_page_step, "ppipqipipiippppppp", P(0), P(1), I(2), P(3), Q(4), I(5), P(6), I(7), P(8),
      I(9), I(10), P(11), P(12), P(13), P(14), P(15), P(16), P(17))
ENTRY(hier_paged8_append, "pqpqiiippppipqippipp", P(0), Q(1), P(2), Q(3), I(4), I(5), I(6), P(7),
      P(8), P(9), P(10), I(11), P(12), Q(13), I(14), P(15), P(16), I(17), P(18), P(19))
ENTRY(hier_paged8_attn, "pqiiiiippppipqippiiiifipqpipppp", P(0), Q(1), I(2), I(3), I(4), I(5),
      I(6), P(7), P(8), P(9), P(10), I(11), P(12), Q(13), I(14), P(15), P(16), I(17), I(18), I(19),
      I(20), x.f, I(22), P(23), Q(24), P(25), I(26), P(27), P(28), P(29), P(30))

typedef struct {
  const char* name;
  void** at;
} entry;

static const entry entries[] = {
    {"hier_head_norm_rope", (void**)&at_hier_head_norm_rope},
    {"hier_head_norm_rope_bwd", (void**)&at_hier_head_norm_rope_bwd},
    {"hier_page_step", (void**)&at_hier_page_step},
    {"hier_paged8_append", (void**)&at_hier_paged8_append},
    {"hier_paged8_attn", (void**)&at_hier_paged8_attn},
};

static PyObject* bind(PyObject* self, PyObject* const* a, Py_ssize_t n) {
  (void)self;
  if (n != 2) {
    PyErr_SetString(PyExc_TypeError, "bind(name, address)");
    return NULL;
  }
  const char* name = PyUnicode_AsUTF8AndSize(a[0], NULL);
  if (!name) return NULL;
  void* address = PyLong_AsVoidPtr(a[1]);
  if (!address && PyErr_Occurred()) return NULL;
  for (size_t i = 0; i < sizeof(entries) / sizeof(entries[0]); ++i)
    if (!strcmp(entries[i].name, name)) {
      memcpy(entries[i].at, &address, sizeof(address));
      Py_INCREF(Py_None);
      return Py_None;
    }
  return PyErr_Format(PyExc_ValueError, "no entry %s", name);
}

#define METHOD(NAME, FN, DOC) {NAME, (PyCFunction)(void (*)(void))FN, METH_FASTCALL, DOC}

static PyMethodDef methods[] = {
    METHOD("bind", bind, "bind(name, address): where an entry point is"),
    METHOD("hier_head_norm_rope", py_hier_head_norm_rope, SIG_hier_head_norm_rope),
    METHOD("hier_head_norm_rope_bwd", py_hier_head_norm_rope_bwd, SIG_hier_head_norm_rope_bwd),
    METHOD("hier_page_step", py_hier_page_step, SIG_hier_page_step),
    METHOD("hier_paged8_append", py_hier_paged8_append, SIG_hier_paged8_append),
    METHOD("hier_paged8_attn", py_hier_paged8_attn, SIG_hier_paged8_attn),
    {NULL, NULL, 0, NULL}};

static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls",
                                    "Direct calls of libhier_b200's entry points.", -1, methods,
                                    NULL, NULL, NULL, NULL};

PyMODINIT_FUNC PyInit__calls(void) { return PyModule_Create(&module); }

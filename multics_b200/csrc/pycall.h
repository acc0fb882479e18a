// Calls from Python whose bodies may throw: the interpreter lock is held again
// whatever way a body ends.
#pragma once

#include <Python.h>

#include <exception>

namespace pycall {

// The interpreter lock given up for a scope.
struct Unlocked {
  PyThreadState* state = PyEval_SaveThread();
  Unlocked() = default;
  Unlocked(const Unlocked&) = delete;
  ~Unlocked() { PyEval_RestoreThread(state); }
};

// f() without the lock; an exception of f leaves with the lock held.
template <class F>
auto unlocked(F f) {
  const Unlocked scope;
  return f();
}

// A reference dropped at the end of a scope.
struct Owned {
  PyObject* o;
  ~Owned() { Py_DECREF(o); }
};

// f()'s result; None, not a call for this path, where f returns NULL without an
// error or throws (a tensor without data, memory run out: Python's to report).
template <class F>
PyObject* attempt(F f) {
  try {
    if (PyObject* r = f()) return r;
  } catch (const std::exception&) {
  }
  if (PyErr_Occurred()) return nullptr;
  Py_RETURN_NONE;
}

}  // namespace pycall

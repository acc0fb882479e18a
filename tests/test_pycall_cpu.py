"""The helpers under the bind module's calls: the interpreter lock is held again
whatever way a body ends (no GPU work)."""

import importlib.util
import os
import subprocess
import sys
import sysconfig
import threading
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "multics_b200" / "csrc"

SOURCE = r"""
#include "pycall.h"
#include <stdexcept>
#include <string>

static PyObject* run(PyObject*, PyObject* kind) {
  const std::string k = PyUnicode_AsUTF8(kind);
  return pycall::attempt([&]() -> PyObject* {
    PyObject* made = PyList_New(0);
    const pycall::Owned owned{made};
    const int v = pycall::unlocked([&] {
      if (k == "throw") throw std::runtime_error("no memory");
      return PyGILState_Check() ? -1 : 7;
    });
    if (k == "error") PyErr_SetString(PyExc_ValueError, "refused");
    if (k == "none" || k == "error") return nullptr;
    return PyLong_FromLong(v);
  });
}

static PyMethodDef methods[] = {{"run", run, METH_O, ""}, {nullptr, nullptr, 0, nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "throwing", "", -1, methods};
PyMODINIT_FUNC PyInit_throwing(void) { return PyModule_Create(&module); }
"""


@pytest.fixture(scope="module")
def throwing(tmp_path_factory):
    at = tmp_path_factory.mktemp("pycall")
    (at / "throwing.cpp").write_text(SOURCE)
    out = at / "throwing.so"
    subprocess.run([os.environ.get("CXX") or "g++", "-O2", "-std=c++17", "-shared", "-fPIC", f"-I{CSRC}",
                    f"-I{sysconfig.get_paths()['include']}", "-o", str(out), str(at / "throwing.cpp")], check=True)
    return out


def test_a_body_that_throws_leaves_the_lock_held(throwing):
    """In a process of its own: without the lock the next call of Python ends it."""
    code = (f"import importlib.util as u\n"
            f"s = u.spec_from_file_location('throwing', {str(throwing)!r})\n"
            f"m = u.module_from_spec(s); s.loader.exec_module(m)\n"
            f"for _ in range(100): assert m.run('throw') is None\n"
            f"assert m.run('value') == 7 and m.run('none') is None\nprint('alive')")
    got = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert got.returncode == 0 and got.stdout == "alive\n", got.stderr


def test_values_errors_and_threads(throwing):
    spec = importlib.util.spec_from_file_location("throwing", throwing)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    with pytest.raises(ValueError, match="refused"):
        m.run("error")
    seen = []
    threads = [threading.Thread(target=lambda: seen.extend(m.run("throw" if i % 2 else "value") for i in range(500)))
               for _ in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert seen.count(7) == seen.count(None) == 1000

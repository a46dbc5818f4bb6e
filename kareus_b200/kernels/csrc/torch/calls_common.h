// What the extension modules share (fastcall.cpp, opcalls.cpp): which tensors they take, how a call ends, how they are set up.
// Included once by each of them; every module has state of its own.
#pragma once
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstdio>
#include <cstdlib>

namespace {

constexpr int MAX_DEVICES = 64;
int* g_status[MAX_DEVICES];        // status word of each device (owned by kernels/cuda.py)
PyObject* g_counter = nullptr;     // one-element list: kernels launched so far
PyObject* g_check = nullptr;       // callable(rc, what) that raises

bool baseline() {
  const char* e = std::getenv("KAREUS_B200_LIBRARY_BASELINE");
  return e && e[0] == '1' && e[1] == 0;
}

// A plain CUDA tensor of this type with storage of its own, on a device whose status word is known; null otherwise.
const at::Tensor* plain(PyObject* o, at::ScalarType type) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.scalar_type() != type || t.layout() != at::kStrided || !t.has_storage() ||
      t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::Functionalize})))
    return nullptr;
  const int dev = t.device().index();
  return dev >= 0 && dev < MAX_DEVICES && g_status[dev] ? &t : nullptr;
}

// Called with the GIL held; false with a Python error set.
bool finish(int rc, const char* what, long launches) {
  if (rc != 0) {
    PyObject* r = PyObject_CallFunction(g_check, "is", rc, what);
    Py_XDECREF(r);
    if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, what);
    return false;
  }
  const long n = PyLong_AsLong(PyList_GET_ITEM(g_counter, 0));
  return !PyErr_Occurred() && PyList_SetItem(g_counter, 0, PyLong_FromLong(n + launches)) == 0;
}

template <typename F>
int without_gil(F f) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = f();
  Py_END_ALLOW_THREADS
  return rc;
}

// init(counter list, check callable); set_status(device index, address of the device's status word)
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2 || !PyList_Check(args[0]) || PyList_GET_SIZE(args[0]) != 1 || !PyCallable_Check(args[1])) {
    PyErr_SetString(PyExc_TypeError, "init(counter, check)");
    return nullptr;
  }
  Py_INCREF(args[0]);
  Py_INCREF(args[1]);
  Py_XSETREF(g_counter, args[0]);
  Py_XSETREF(g_check, args[1]);
  Py_RETURN_NONE;
}

PyObject* set_status(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  if (nargs != 2) {
    PyErr_SetString(PyExc_TypeError, "set_status(device, address)");
    return nullptr;
  }
  const long dev = PyLong_AsLong(args[0]);
  void* p = PyLong_AsVoidPtr(args[1]);
  if (PyErr_Occurred()) return nullptr;
  if (dev < 0 || dev >= MAX_DEVICES || !g_counter) {
    PyErr_SetString(PyExc_ValueError, "set_status: bad device, or init() has not run");
    return nullptr;
  }
  g_status[dev] = static_cast<int*>(p);
  Py_RETURN_NONE;
}

}  // namespace

// views.cpp -- what the Python binding asks of a torch tensor before a call, in one step each: a
// CPython extension on torch's headers (a call from Python checks up to a dozen operands, and the
// attribute reads of that took longer than the smallest kernels).
//
//   matrix(t, rows, cols, dtype) -> (pointer, row stride) of a CUDA tensor [rows, >= cols] of that
//                                   dtype whose columns are adjacent and rows do not overlap
//   vector(t, n, dtype)          -> pointer of a contiguous CUDA tensor [n] of that dtype
//
// dtype: 0 float32, 1 int32, 2 uint8.  None where the tensor is anything else; the binding then
// looks again and says what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

namespace {

const at::Tensor* tensor_of(PyObject* o, long dtype) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided) return nullptr;
  const at::ScalarType want = dtype == 0 ? at::kFloat : dtype == 1 ? at::kInt : at::kByte;
  return t.scalar_type() == want ? &t : nullptr;
}

PyObject* matrix(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) return PyErr_Format(PyExc_TypeError, "matrix takes four arguments");
  const long long rows = PyLong_AsLongLong(args[1]), cols = PyLong_AsLongLong(args[2]);
  const long dtype = PyLong_AsLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* t = tensor_of(args[0], dtype);
  if (!t || t->dim() != 2 || t->size(0) != rows || t->size(1) < cols || t->stride(1) != 1 || t->stride(0) < t->size(1)) Py_RETURN_NONE;
  PyObject* out = PyTuple_New(2);
  if (!out) return nullptr;
  PyTuple_SET_ITEM(out, 0, PyLong_FromUnsignedLongLong(reinterpret_cast<unsigned long long>(t->data_ptr())));
  PyTuple_SET_ITEM(out, 1, PyLong_FromLongLong(t->stride(0)));
  return out;
}

PyObject* vector(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 3) return PyErr_Format(PyExc_TypeError, "vector takes three arguments");
  const long long len = PyLong_AsLongLong(args[1]);
  const long dtype = PyLong_AsLong(args[2]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* t = tensor_of(args[0], dtype);
  if (!t || t->dim() != 1 || t->size(0) != len || (len > 1 && t->stride(0) != 1)) Py_RETURN_NONE;
  return PyLong_FromUnsignedLongLong(reinterpret_cast<unsigned long long>(t->data_ptr()));
}

PyMethodDef methods[] = {
    {"matrix", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(matrix)), METH_FASTCALL, nullptr},
    {"vector", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(vector)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_views", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__views() { return PyModule_Create(&module); }

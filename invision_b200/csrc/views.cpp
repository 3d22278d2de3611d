// views.cpp -- calls of the Python binding whose operands are torch tensors: a CPython extension on
// torch's headers (a call checks up to a dozen operands and packs a structure, and the attribute
// reads of that took longer than the smallest kernels).
//
//   call(function, use_device, flags, spec, ...) -> status of function(structure, flags), after that
//                                   of use_device(operands' device, follow, stream) (unless 0): the
//                                   library has to run there, and with FOLLOW in flags is put on
//                                   torch's current stream.  The structure is packed from the
//                                   operands by `spec`, a letter a field: M matrix (tensor, rows,
//                                   cols) and its row stride, E the same of exactly cols columns, V
//                                   float vector (tensor, n), I int vector, P contiguous float matrix
//                                   (tensor, rows, cols), J int matrix, p pointer, q int64, i int32,
//                                   f float; None is NULL
//   matrix(t, rows, cols, dtype) -> (pointer, row stride) of a CUDA tensor [rows, >= cols] of that
//                                   dtype whose columns are adjacent and rows do not overlap
//   vector(t, n, dtype)          -> pointer of a contiguous CUDA tensor [n] of that dtype
//
// dtype: 0 float32, 1 int32, 2 uint8.  None (and no call) where a tensor is anything else or lives on
// another device than the first; the binding then looks again and says what is wrong.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstring>

namespace {

const at::Tensor* tensor_of(PyObject* o, long dtype) {
  if (!THPVariable_Check(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda() || t.layout() != at::kStrided) return nullptr;
  const at::ScalarType want = dtype == 0 ? at::kFloat : dtype == 1 ? at::kInt : at::kByte;
  return t.scalar_type() == want ? &t : nullptr;
}

bool is_matrix(const at::Tensor* t, long long rows, long long cols) {
  return t && t->dim() == 2 && t->size(0) == rows && t->size(1) >= cols && t->stride(1) == 1 && t->stride(0) >= t->size(1);
}

PyObject* matrix(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 4) return PyErr_Format(PyExc_TypeError, "matrix takes four arguments");
  const long long rows = PyLong_AsLongLong(args[1]), cols = PyLong_AsLongLong(args[2]);
  const long dtype = PyLong_AsLong(args[3]);
  if (PyErr_Occurred()) return nullptr;
  const at::Tensor* t = tensor_of(args[0], dtype);
  if (!is_matrix(t, rows, cols)) Py_RETURN_NONE;
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

PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  constexpr Py_ssize_t MOST = 256;  // bytes of a structure
  constexpr int FOLLOW = 1 << 16;  // in flags, for this function alone
  if (n < 4) return PyErr_Format(PyExc_TypeError, "call takes a function, a device check, flags, a spec and operands");
  auto* fn = reinterpret_cast<int (*)(const void*, int)>(PyLong_AsUnsignedLongLong(args[0]));
  auto* use_device = reinterpret_cast<int (*)(int, int, void*)>(PyLong_AsUnsignedLongLong(args[1]));
  const int flags = (int)PyLong_AsLong(args[2]);
  const char* spec = PyUnicode_AsUTF8(args[3]);
  if (PyErr_Occurred()) return nullptr;
  alignas(8) unsigned char packed[MOST] = {};
  Py_ssize_t at = 0, i = 4;
  int device = -1;
  auto put = [&](const void* v, Py_ssize_t size) {
    at = (at + size - 1) / size * size;
    memcpy(packed + at, v, size);
    at += size;
  };
  for (; *spec; ++spec) {
    const Py_ssize_t takes = strchr("MEPJ", *spec) ? 3 : strchr("VI", *spec) ? 2 : 1;
    if (i + takes > n || at + 16 > MOST) return PyErr_Format(PyExc_TypeError, "call: the operands do not match the spec");
    if (takes == 1) {
      if (*spec == 'f') {
        const double v = PyFloat_AsDouble(args[i]);
        if (std::isfinite(v) && std::isinf((float)v)) return PyErr_Format(PyExc_OverflowError, "argument does not fit 32 bits");
        const float f = (float)v;
        put(&f, 4);
      } else if (*spec == 'i') {
        const long v = PyLong_AsLong(args[i]);
        if ((v != -1 || !PyErr_Occurred()) && v != (int)v) return PyErr_Format(PyExc_OverflowError, "argument does not fit 32 bits");
        const int v32 = (int)v;
        put(&v32, 4);
      } else {
        const long long v = *spec == 'p' ? (long long)PyLong_AsUnsignedLongLong(args[i]) : PyLong_AsLongLong(args[i]);
        put(&v, 8);
      }
    } else {
      const long long rows = PyLong_AsLongLong(args[i + 1]), cols = takes == 3 ? PyLong_AsLongLong(args[i + 2]) : 0;
      if (PyErr_Occurred()) return nullptr;
      const void* ptr = nullptr;
      int64_t ld = 0;
      if (args[i] != Py_None) {
        const at::Tensor* t = tensor_of(args[i], *spec == 'I' || *spec == 'J' ? 1 : 0);
        if (!t) Py_RETURN_NONE;
        if (takes == 2) {
          if (t->dim() != 1 || t->size(0) != rows || (rows > 1 && t->stride(0) != 1)) Py_RETURN_NONE;
        } else {
          if (!is_matrix(t, rows, cols)) Py_RETURN_NONE;
          ld = t->stride(0);
          if (*spec != 'M' && t->size(1) != cols) Py_RETURN_NONE;
          if ((*spec == 'P' || *spec == 'J') && rows > 1 && ld != cols) Py_RETURN_NONE;
        }
        ptr = t->data_ptr();
        if (device < 0) device = t->device().index();
        if (t->device().index() != device) Py_RETURN_NONE;
      }
      put(&ptr, 8);
      if (*spec == 'M' || *spec == 'E') put(&ld, 8);
    }
    if (PyErr_Occurred()) return nullptr;
    i += takes;
  }
  if (i != n || device < 0) {
    if (i == n) Py_RETURN_NONE;
    return PyErr_Format(PyExc_TypeError, "call: the operands do not match the spec");
  }
  void* stream = nullptr;
  const int follow = (flags & FOLLOW) != 0;
  if (follow) {
    stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)device).stream();
    if (!stream) stream = reinterpret_cast<void*>(1);  // cudaStreamLegacy, by its own name
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = use_device ? use_device(device, follow, stream) : 0;
  if (rc == 0) rc = fn(packed, flags & ~FOLLOW);
  Py_END_ALLOW_THREADS
  return PyLong_FromLong(rc);
}

// A tensor without plain storage (nested, functional, ..) throws where it is asked for its sizes or
// its memory: it is one of those that the binding looks at again.
template <PyObject* (*F)(PyObject*, PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject* self, PyObject* const* args, Py_ssize_t n) {
  try {
    return F(self, args, n);
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

PyMethodDef methods[] = {
    {"call", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<call>)), METH_FASTCALL, nullptr},
    {"matrix", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<matrix>)), METH_FASTCALL, nullptr},
    {"vector", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(guarded<vector>)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_views", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

// `stamp` says what the module was built from and for; the binding loads no other.
PyMODINIT_FUNC PyInit__views() {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "stamp", ENVG_VIEWS_STAMP) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}

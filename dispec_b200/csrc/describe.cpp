// Python module: describe(*tensors) -> bytes, one DspTensor (tensor_desc.h) for each tensor, None included.
//
// What an entry point has to know of a tensor, and checks, is read here in one go.  Asked for attribute by attribute from Python, the eight
// tensors of an attention call cost the host some 7 us, beside 2.5 us for a launch; so, under 1 us.
#include <Python.h>
#include <torch/csrc/autograd/python_variable.h>

#include "tensor_desc.h"

static PyObject* describe(PyObject*, PyObject* const* args, Py_ssize_t n) {
  PyObject* bytes = PyBytes_FromStringAndSize(nullptr, n * (Py_ssize_t)sizeof(DspTensor));
  if (bytes == nullptr) return nullptr;
  DspTensor* out = reinterpret_cast<DspTensor*>(PyBytes_AS_STRING(bytes));
  for (Py_ssize_t i = 0; i < n; ++i) {
    DspTensor d = {};
    d.dims = -1;
    if (args[i] != Py_None) {
      if (!THPVariable_Check(args[i])) {
        Py_DECREF(bytes);
        return PyErr_Format(PyExc_TypeError, "a tensor or None expected, not %s", Py_TYPE(args[i])->tp_name);
      }
      try {
        const at::Tensor& t = THPVariable_Unpack(args[i]);
        d.data = t.data_ptr();
        const auto type = t.scalar_type();
        d.dtype = type == at::kFloat ? DSP_T_F32 : type == at::kBFloat16 ? DSP_T_BF16 : type == at::kInt ? DSP_T_I32
                : type == at::kLong ? DSP_T_I64 : DSP_T_OTHER;
        d.device = t.is_cuda() ? t.get_device() : -1;
        d.dims = (int)t.dim();
        d.contiguous = t.is_contiguous();
        for (int k = 0; k < d.dims && k < DSP_T_DIMS; ++k) {
          d.size[k] = t.size(k);
          d.stride[k] = t.stride(k);
        }
      } catch (const std::exception& e) {
        Py_DECREF(bytes);
        PyErr_SetString(PyExc_RuntimeError, e.what());
        return nullptr;
      }
    }
    out[i] = d;
  }
  return bytes;
}

static PyMethodDef methods[] = {{"describe", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(describe)), METH_FASTCALL,
                                 "describe(*tensors) -> bytes"},
                                {nullptr, nullptr, 0, nullptr}};
static PyModuleDef module = {PyModuleDef_HEAD_INIT, "dispec_b200_describe", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};
PyMODINIT_FUNC PyInit_dispec_b200_describe(void) { return PyModule_Create(&module); }

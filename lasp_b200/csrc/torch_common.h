// Shared by the operators as PyTorch sees them (torch_ops.cpp: attention; torch_recurrent.cpp: convolution and scan).
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/SavedTensorHooks.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/CUDAGraphsUtils.cuh>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/library.h>

#include <nvtx3/nvToolsExt.h>

#include <cstdlib>
#include <string>

#include "lasp_b200.h"

namespace lasp_torch {

struct Range {   // NVTX range around a library call (LASP_B200_NVTX=1)
  bool on;
  explicit Range(const char* name) : on(enabled()) {
    if (on) nvtxRangePushA(name);
  }
  ~Range() {
    if (on) nvtxRangePop();
  }
  static bool enabled() {
    static const bool v = [] {
      const char* e = std::getenv("LASP_B200_NVTX");
      return e && e[0] == '1';
    }();
    return v;
  }
};

// A negative status becomes lasp_b200._cabi.LaspStatusError, on whatever thread this is (autograd's workers too).
inline void check_status(const char* fn, int status) {
  if (status >= 0) return;
  std::string text = lasp_b200_strerror(status);
  if (status == LASP_ERR_CUDA) text += std::string(": ") + lasp_b200_last_cuda_error();
  PyGILState_STATE gil = PyGILState_Ensure();
  PyObject* mod = PyImport_ImportModule("lasp_b200._cabi");
  PyObject* cls = mod ? PyObject_GetAttrString(mod, "LaspStatusError") : nullptr;
  PyObject* exc = cls ? PyObject_CallFunction(cls, "sis", fn, status, text.c_str()) : nullptr;
  if (exc) PyErr_SetObject(cls, exc);
  Py_XDECREF(exc);
  Py_XDECREF(cls);
  Py_XDECREF(mod);
  python_error err;
  err.persist();
  PyGILState_Release(gil);
  throw err;
}

inline int32_t lasp_dtype_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return LASP_F32;
    case at::kBFloat16: return LASP_BF16;
    case at::kHalf: return LASP_F16;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t, "; use float32, bfloat16 or float16");
  }
}

// Methods of the module, defined in torch_recurrent.cpp.
PyObject* py_causal_conv(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* py_causal_conv_step(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* py_selective_scan(PyObject*, PyObject* const* args, Py_ssize_t nargs);
PyObject* py_selective_scan_step(PyObject*, PyObject* const* args, Py_ssize_t nargs);

}  // namespace lasp_torch

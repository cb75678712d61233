// What the two sources of the CPython module _host share.
#pragma once
#include <torch/csrc/autograd/python_variable.h>
#include <c10/hip/HIPStream.h>

namespace {

// An ordinary tensor (or Parameter), or null.
const at::Tensor* tensor_of(PyObject* o) { return THPVariable_CheckExact(o) ? &THPVariable_Unpack(o) : nullptr; }

// The GIL given up for the scope (and taken again when an exception leaves it):
// a launch or an allocation may wait for the GPU, and a host callback that the
// GPU waits for may need Python.
struct WithoutGil {
  PyThreadState* state = PyEval_SaveThread();
  ~WithoutGil() { PyEval_RestoreThread(state); }
};

void* stream_of(int dev) { return (void*)c10::hip::getCurrentHIPStream((c10::DeviceIndex)dev).stream(); }

}  // namespace

// The serving operators' methods (host_serve.cpp).
extern PyMethodDef bf16x_serve_methods[];

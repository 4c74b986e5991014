// What the parts of the extension share: references, the test for a plain tensor, and the module's functions beside LinearCall.
#pragma once
#include <Python.h>

#include <ATen/ATen.h>
#include <torch/csrc/autograd/python_variable.h>

#include <utility>

namespace ksana_host {

// A strong reference.
struct Ref {
  PyObject* p = nullptr;
  Ref() = default;
  explicit Ref(PyObject* o) : p(o) { Py_XINCREF(p); }
  Ref(Ref&& o) noexcept : p(o.p) { o.p = nullptr; }
  Ref(const Ref& o) : p(o.p) { Py_XINCREF(p); }
  Ref& operator=(Ref o) noexcept {
    std::swap(p, o.p);
    return *this;
  }
  ~Ref() { Py_XDECREF(p); }
};

// An exact tensor with memory of its own, not one that a transform wraps.
inline bool plain_tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return false;
  const at::Tensor& t = THPVariable_Unpack(o);
  const c10::DispatchKeySet wrapped({c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                     c10::DispatchKey::Python, c10::DispatchKey::Batched});
  return t.defined() && t.has_storage() && t.layout() == at::kStrided && !t.key_set().has_any(wrapped) && !t.is_conj() && !t.is_neg();
}

extern PyMethodDef op_methods[];  // host_ops.cpp

}  // namespace ksana_host

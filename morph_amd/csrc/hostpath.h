// What the host extension's sources share: plain tensors, as their native paths take them.
#pragma once

#include <ATen/TensorSubclassLikeUtils.h>
#include <pybind11/pybind11.h>
#include <pybind11/stl.h>
#include <torch/csrc/autograd/python_variable.h>

namespace py = pybind11;

// at::isTensorSubclassLike without its question for a dispatch mode, which a call asks once.
inline bool plain(const at::Tensor& t) {
  return (t.key_set() & at::kTensorSubclassLike).empty() && t.has_storage();
}

inline const at::Tensor* plain_tensor(PyObject* o) {
  if (o == nullptr || !THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  return t.defined() && plain(t) ? &t : nullptr;
}

// Whether t is n contiguous elements of `type`.
inline bool holds(const at::Tensor& t, at::ScalarType type, int64_t n) {
  return t.numel() == n && t.scalar_type() == type && t.is_contiguous();
}

void bind_layers(py::module_& m);  // hostlayers.cpp

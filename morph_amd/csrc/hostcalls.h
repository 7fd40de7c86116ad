// What the native calls of the operators share: the current device and its stream, outputs there, and plain
// tensors of a layout that needs no preparation.
#pragma once

#include "hostpath.h"

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>

#include "../../include/morph_layers.h"

namespace {

int code(at::ScalarType t) {
  return t == at::kFloat      ? MORPH_DTYPE_F32
         : t == at::kHalf     ? MORPH_DTYPE_F16
         : t == at::kBFloat16 ? MORPH_DTYPE_BF16
                              : MORPH_DTYPE_NONE;
}

// The current device and its stream, and outputs there; asked for a call whose first tensor
// is on a GPU.
struct Here {
  c10::Device device{c10::DeviceType::CPU};
  explicit Here(py::handle first) {
    const at::Tensor* t = plain_tensor(first.ptr());
    if (t != nullptr && t->is_cuda()) device = c10::Device(c10::DeviceType::CUDA, c10::hip::current_device());
  }
  void* stream() const { return c10::hip::getCurrentHIPStream(device.index()).stream(); }
  at::Tensor empty(at::IntArrayRef shape, at::ScalarType type) const {
    return at::empty(shape, at::TensorOptions().device(device).dtype(type));
  }
  // o as a plain tensor on this device, or null.
  const at::Tensor* tensor(py::handle o) const {
    const at::Tensor* t = plain_tensor(o.ptr());
    return t != nullptr && t->is_cuda() && t->layout() == at::kStrided && t->device() == device ? t : nullptr;
  }
};

// A 2-D tensor of this shape with contiguous rows: its row stride, or 0.
int64_t rows_of(const at::Tensor& t, at::ScalarType type, int64_t rows, int64_t cols) {
  if (t.dim() != 2 || t.scalar_type() != type || t.size(0) != rows || t.size(1) != cols) return 0;
  if (t.is_contiguous()) return cols;
  return t.stride(1) == 1 && t.stride(0) >= cols ? t.stride(0) : 0;
}

py::object wrap(at::Tensor t) { return py::reinterpret_steal<py::object>(THPVariable_Wrap(std::move(t))); }

// The GIL is released around the library: a launch waits when the queue is full.
template <typename F>
int released(F&& f) {
  const py::gil_scoped_release nogil;
  return f();
}

}  // namespace

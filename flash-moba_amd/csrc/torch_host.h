// What the translation units of the eager host module share: error checks and the tests for plain eager work on ordinary tensors.
#pragma once

#include <torch/extension.h>

#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <algorithm>
#include <atomic>

#include "../../include/flash_moba_hip.h"

namespace fmoba_host {

using at::Tensor;

inline void check(int rc) {
  if (rc != 0) throw std::runtime_error(fmoba_last_error());
}

// A C++ exception of the base class becomes RuntimeError in Python.  The device check is made once per device.
inline void check_device(int index) {
  static std::atomic<uint64_t> ok{0};
  const uint64_t bit = uint64_t(1) << (index & 63);
  if (index < 64 && (ok.load(std::memory_order_relaxed) & bit)) return;
  check(fmoba_check_device());
  if (index < 64) ok.fetch_or(bit);
}

inline PyObject *g_parameter_class = nullptr;  // torch.nn.Parameter

// an ordinary tensor (or parameter): no subclass, no wrapper of a transform, no lazy conjugate, no tangent of forward-mode
// differentiation (a dual tensor has the key set of an ordinary one; the path in Python refuses it, having no derivative of that kind)
inline bool plain(const py::handle &h) {
  if (!THPVariable_CheckExact(h.ptr()) && reinterpret_cast<PyObject *>(Py_TYPE(h.ptr())) != g_parameter_class) return false;
  const Tensor &t = THPVariable_Unpack(h.ptr());
  return t.defined() && t.is_cuda() && !t.is_sparse() && !t._fw_grad(/*level=*/0).defined() &&
         !t.key_set().has_any(c10::DispatchKeySet({c10::DispatchKey::Python, c10::DispatchKey::FuncTorchBatched, c10::DispatchKey::FuncTorchGradWrapper,
                                                   c10::DispatchKey::Functionalize, c10::DispatchKey::Conjugate, c10::DispatchKey::Negative}));
}

inline bool eager() { return !c10::impl::TorchDispatchModeTLS::any_modes_set() && !torch::jit::tracer::isTracing(); }

inline bool is_cu(const Tensor &t, int64_t n, const at::Device &dev) {
  return t.scalar_type() == at::kInt && t.dim() == 1 && t.numel() == n && t.is_contiguous() && t.device() == dev;
}

// (rows, heads, dim), last dimension dense, 16-byte vectors
inline bool is_rows(const Tensor &t, at::ScalarType dt, const at::Device &dev) {
  return t.dim() == 3 && t.scalar_type() == dt && t.device() == dev && t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 &&
         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}

inline Tensor bytes_like(const Tensor &q, size_t n) { return at::empty({static_cast<int64_t>(std::max<size_t>(n, 1))}, q.options().dtype(at::kByte)); }
inline size_t up256(size_t x) { return (x + 255) & ~size_t(255); }

// The functions of a paged cache and of the positions (torch_cache_ops.cpp), added to the module.
void bind_cache_ops(pybind11::module_ &m);

}  // namespace fmoba_host

// What the sources of the torch module share: argument checks and tensors' parts.
#pragma once
#include <ATen/MemoryOverlap.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>
#include <pybind11/stl.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cstring>
#include <optional>
#include <string>
#include <utility>
#include <vector>

#include "../../include/zorse_amd.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> MaybeTensor;

// Add the functions of nodes_packed.cpp and nodes_muon.cpp to the module.
void bind_packed(py::module_& m);
void bind_muon(py::module_& m);

namespace {

[[noreturn]] inline void bad(const std::string& what) { throw py::value_error(what); }

inline void check(int status, const char* who) {
  if (status == 0) return;
  static const char* const names[] = {"ZK_EINVAL", "ZK_EDTYPE", "ZK_EALIGN", "ZK_EUNSUPPORTED",
                                      "ZK_EWORKSPACE"};
  throw std::runtime_error(std::string(who) + " failed with " +
                           (status < 0 && status >= -5 ? names[-1 - status]
                                                       : "hipError " + std::to_string(status)) +
                           ": " + zk_last_error());
}

inline zk_stream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.get_device()).stream();
}

inline at::ScalarType type_of(int64_t code) {
  return code == ZK_F32 ? at::kFloat : code == ZK_F16 ? at::kHalf : at::kBFloat16;
}
inline int code_of(at::ScalarType t) {
  return t == at::kFloat ? ZK_F32 : t == at::kHalf ? ZK_F16 : t == at::kBFloat16 ? ZK_BF16 : -1;
}
inline int float_code(const char* name, at::ScalarType t) {
  const int code = code_of(t);
  if (code < 0) bad(c10::str("unsupported ", name, " dtype ", t));
  return code;
}

constexpr const char* kNeedGpu = "zorse_amd kernels need GPU tensors (got a CPU tensor)";

inline void one_gpu(std::initializer_list<const Tensor*> tensors) {
  const Tensor& first = **tensors.begin();
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    if (!t->is_cuda()) bad(kNeedGpu);
    if (t->get_device() != first.get_device()) bad("tensors are on different devices");
  }
}

inline void* address(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

inline Tensor given(const MaybeTensor& t) { return t.has_value() ? *t : Tensor(); }

inline Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes > 0 ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// Forward-mode derivatives: a dual tensor carries its tangent beside its values.
inline bool is_dual(const Tensor& t) { return t.defined() && t._fw_grad(/*level=*/0).defined(); }

// Unit stride along d (expanded heads and gradients have none).
inline Tensor rows_of(const Tensor& t) {
  return !t.defined() || t.dim() == 0 || t.stride(-1) == 1 ? t : t.contiguous();
}

inline MaybeTensor maybe(const Tensor& t) { return t.defined() ? MaybeTensor(t) : MaybeTensor(); }

}  // namespace

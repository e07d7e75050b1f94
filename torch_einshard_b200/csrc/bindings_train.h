// Registers the bindings of bindings_train.cpp and bindings_saved8.cpp.
#pragma once

#include <torch/extension.h>

#include <atomic>
#include <vector>

namespace es {

// `launches` counts native launches.
void bind_training_ops(pybind11::module_& m, std::atomic<long long>& launches);

// The products that the contractions of 8-bit operands are made of (the last argument is the device's error word).
struct GemmOps {
  at::Tensor (*product)(const at::Tensor&, const at::Tensor&, const at::Tensor&);
  c10::optional<at::Tensor> (*sum)(const std::vector<at::Tensor>&, const std::vector<at::Tensor>&, const at::Tensor&);
  std::vector<at::Tensor> (*silu)(const at::Tensor&, const at::Tensor&, const at::Tensor&);
  std::vector<at::Tensor> (*silu_grad)(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                       const at::Tensor&);
};
void bind_saved8_ops(pybind11::module_& m, const GemmOps& ops);

// What the codes [rows, d] stand for (contiguous), its silu, or grad times its silu' (mode 0, 1, 2).
at::Tensor restore8_op(const at::Tensor& codes, const at::Tensor& exps, const c10::optional<at::Tensor>& grad,
                       int64_t dtype, int64_t mode);

// The number of the capture that the device's current stream takes part in (each has its own), or 0.
int64_t capture_of(c10::DeviceIndex device);

// The kernels read raw memory: a view that only says it is negated is written out.
at::Tensor plain(const at::Tensor& t);

// `grads` as results of `from`, where a graph of the backward pass is wanted: they have no derivatives of their own,
// using them further raises.
void finalise(std::vector<at::Tensor>& grads, const std::vector<at::Tensor>& from);

}  // namespace es

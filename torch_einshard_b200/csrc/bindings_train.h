// Registers the bindings of bindings_train.cpp; `launches` counts native launches.
#pragma once

#include <torch/extension.h>

#include <atomic>

namespace es {

void bind_training_ops(pybind11::module_& m, std::atomic<long long>& launches);

}  // namespace es

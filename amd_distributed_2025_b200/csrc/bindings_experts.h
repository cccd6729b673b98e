// Python calls of the operators around a GPU's experts (see bindings_experts.cpp).
#pragma once
#include <torch/extension.h>

namespace b200 {
void bind_experts(pybind11::module& m);
}  // namespace b200

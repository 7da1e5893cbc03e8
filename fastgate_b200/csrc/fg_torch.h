// Shared by the translation units of the pybind extension.
#pragma once
#include <torch/extension.h>

// Operators around the linears of a serving step (fg_torch_serving.cpp).
void bind_serving(pybind11::module& m);

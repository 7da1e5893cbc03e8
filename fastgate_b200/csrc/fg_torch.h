// Shared by the translation units of the pybind extension.
#pragma once
#include <cuda_runtime.h>
#include <torch/extension.h>

// The cleared workspace of a call that is being captured on `stream` (fg_torch_graph.cpp); nullptr: no capture.
void* graph_workspace(int device, cudaStream_t stream, size_t bytes);
// The device's status word of the operators that have no workspace (fg_torch_graph.cpp): allocated once and kept, so that
// captured calls may hold it.  workspace_status() reads it too.
int* linear_status(int device);

// Operators around the linears of a serving step (fg_torch_serving.cpp).
void bind_serving(pybind11::module& m);

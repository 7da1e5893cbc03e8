// Shared by the translation units of the pybind extension.
#pragma once
#include <cuda_runtime.h>
#include <torch/extension.h>

// The cleared workspace of a call that is being captured on `stream` (fg_torch_graph.cpp); nullptr: no capture.
void* graph_workspace(int device, cudaStream_t stream, size_t bytes);
// The status word that workspace_status() reads: of the stream's workspace (fg_torch.cpp).  nullptr while the stream is
// captured and has none yet.
int* linear_status(int64_t device, cudaStream_t stream);

// Operators around the linears of a serving step (fg_torch_serving.cpp).
void bind_serving(pybind11::module& m);

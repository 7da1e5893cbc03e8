// Shared by the translation units of the pybind extension.
#pragma once
#include <cuda_runtime.h>
#include <torch/extension.h>

enum WorkspaceKind { kLinearWorkspace = 0, kAttentionWorkspace = 1 };
// The cleared workspace of a call that is being captured on `stream` (fg_torch_graph.cpp); nullptr: no capture.
void* graph_workspace(int device, cudaStream_t stream, WorkspaceKind kind, size_t bytes);

struct StreamWorkspace {
  at::Tensor buf;   // keeps an eager call's memory alive
  void* ptr = nullptr;
  size_t bytes = 0;
};
// The linears' workspace for N output columns: of the (device, stream), or of the graph being captured (fg_torch.cpp).
StreamWorkspace linear_workspace(int64_t device, cudaStream_t stream, int64_t N);

// Operators around the linears of a serving step (fg_torch_serving.cpp).
void bind_serving(pybind11::module& m);

// Shared by the translation units of the pybind extension.
#pragma once
#include <cuda_runtime.h>
#include <torch/extension.h>

struct StreamWorkspace {
  at::Tensor buf;
  size_t bytes = 0;
};
// The linears' workspace of a (device, stream), with room for N output columns (fg_torch.cpp).
StreamWorkspace stream_workspace(int64_t device, cudaStream_t stream, int64_t N);
// One for a single call that is being captured: from the graph's memory, cleared inside the graph, so that graphs captured
// on one stream may be replayed side by side.
StreamWorkspace captured_workspace(int64_t device, cudaStream_t stream, int64_t N);

// Operators around the linears of a serving step (fg_torch_serving.cpp).
void bind_serving(pybind11::module& m);

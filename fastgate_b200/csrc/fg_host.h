// Host helpers shared by the translation units of libfastgate_b200.so (defined in fg_capi.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

namespace fg {
namespace host {

struct Device {
  int index;
  int sm_count;
  int smem_optin;  // dynamic shared memory one CTA may opt in to
};

// The current device; FG_ERR_NO_DEVICE unless it is an sm_100 part.
int current_device(Device* out);
// 2-D row-major tensor, 128-byte swizzle (see fg_capi.cu).
int encode_tensor(CUtensorMap* tm, CUtensorMapDataType dt, int elem_bytes, const void* base, uint64_t inner, uint64_t rows,
                  uint32_t box_inner, uint32_t box_rows);
// Opts `kernel` in to at least `bytes` of dynamic shared memory on the current device (remembered per device).
int opt_in_smem(const void* kernel, int bytes);
// Status of a launch: counts it, or records the error and returns FG_ERR_CUDA.
int launched(cudaError_t e);

inline bool aligned(const void* p, unsigned bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Launch on `stream`; pdl: the kernel may start while the previous kernel of the stream drains (it calls
// griddepcontrol.wait before it touches memory that others write).
template <typename... Params, typename... Args>
int launch(void (*kern)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, bool pdl, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return launched(cudaLaunchKernelEx(&cfg, kern, static_cast<Params>(args)...));
}

}  // namespace host
}  // namespace fg

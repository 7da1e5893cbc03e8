// What the kernels on int8 activations and weights (fg_linear_w8a8) have in common: their parameters and the way from an
// exact integer sum to an output.
#pragma once
#include "fg_kernels.cuh"

namespace fg {

struct W8A8Params {
  __half* C;               // [M, N], or [M, N / 2] with the SiLU gate
  const void* x_scales;    // [M] fp32 or fp16
  int x_scales_f32;
  const __half* w_scales;  // [N] or nullptr
  const __half* bias;      // [N] or nullptr
  const __half* residual;  // shape of C, or nullptr
  int M, N, K;
  int act;
  int* status;             // or nullptr
};

__device__ __forceinline__ float x_scale(const W8A8Params& p, int m) {
  return p.x_scales_f32 ? static_cast<const float*>(p.x_scales)[m] : __half2float(static_cast<const __half*>(p.x_scales)[m]);
}
// Every product and sum is rounded by itself (no contraction to fused operations): a row has the same bits whichever of the
// kernels computes it.
__device__ __forceinline__ float w8a8_value(int sum, float xs, float ws, float bias) {
  return __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(sum), xs), ws), bias);
}
// The activations are v * sigmoid(t) (the tanh form of GELU too: 1 + tanh(y) = 2 sigmoid(2 y)), with the fast exponential and
// division: 2^-21 or so off, next to an output of 11 bits.  Their exact forms cost a gated tile more time than its MMAs.
__device__ __forceinline__ float times_sigmoid(float v, float t) { return __fdividef(v, 1.f + __expf(-t)); }
template <int ACT>
__device__ __forceinline__ float w8a8_act(float v) {
  if constexpr (ACT == kActSilu) return times_sigmoid(v, v);
  else if constexpr (ACT == kActGeluTanh) return times_sigmoid(v, 1.5957691216057308f * (v + 0.044715f * v * v * v));
  else return act_fn<ACT>(v);
}
__device__ __forceinline__ float w8a8_gate(float g, float u) { return __fmul_rn(w8a8_act<kActSilu>(g), u); }

// Weight row of output column `col` of the gated pair; its up row lies 64 further on.
__device__ __forceinline__ int gate_row(int col) { return col / 64 * 128 + col % 64; }

}  // namespace fg

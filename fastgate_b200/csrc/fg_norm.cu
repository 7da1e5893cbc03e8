// RMS norm with the residual addition, fp16 or int8 output (fg_add_rmsnorm).
//
//   h = x + residual, residual_out = h, rstd = 1 / sqrt(mean h^2 + eps)
//   fp16:  out = h * rstd * w
//   int8:  t = h * w, a = max|t|, out = rint(t * (127 / a)), scale = a * rstd / 127
//
// One pass: a row stays in its CTA's registers between the load and the store, and both statistics (sum of
// squares and largest |t|) go through one block reduction.  The int8 codes are formed from t, not from the
// normalised value: rstd divides out of y / scale, so the reduction's summation order cannot move a code.
// The traffic is the bound: 2 K bytes of x, 4 K (8 K) of residual in and out in fp16 (fp32), 2 K or K of output.  Measured on
// B200, int8 output: 8192 x 4096 with an fp32 residual 56.3 us (6.6 TB/s, a plain copy's rate), with an fp16 one 40.9 (5.8 TB/s); 16 x
// 8192 2.4 us, of which a launch is most.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/fastgate_b200.h"
#include "fg_host.h"
#include "fg_ptx.cuh"

namespace fg {
namespace {

constexpr int kNormMaxThreads = 1024;
constexpr float kLargest = 3.402823466e38f;
// A 32-bit residual reaches values whose squares do not fit 32 bits.  Where their sum has overflowed it is formed again, of
// (2^-80 h)^2: neither do 2^31 of the largest values overflow it nor do its decisive terms underflow.  (Formed always, beside the
// other, it costs 8192 x 4096 rows 58.4 us instead of 56.3.)
constexpr float kFar = 8.271806125530277e-25f;  // 2^-80

struct NormParams {
  const __half* x;
  long long ldx;
  const __half* weight;
  const void* residual;  // nullptr: none
  void* residual_out;
  void* out;
  float* scales;
  int K;
  float eps;
};

// Eight consecutive elements, 16-byte loads.
__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 q = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
  v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
  v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
}
__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  uint4 q;
  uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  *reinterpret_cast<uint4*>(p) = q;
}
__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  *reinterpret_cast<float4*>(p + 4) = make_float4(v[4], v[5], v[6], v[7]);
}
// Codes of eight values, already scaled to [-127, 127], as one 8-byte store.
__device__ __forceinline__ void store8(int8_t* p, const float (&v)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    uint32_t hi;
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, 0;" : "=r"(hi) : "r"(__float2int_rn(v[4 * i + 3])), "r"(__float2int_rn(v[4 * i + 2])));
    asm("cvt.pack.sat.s8.s32.b32 %0, %1, %2, %3;" : "=r"(w[i]) : "r"(__float2int_rn(v[4 * i + 1])), "r"(__float2int_rn(v[4 * i])), "r"(hi));
  }
  *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

// The larger of two values, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// RES: 0 none, 1 fp16, 2 fp32.  VPT: vectors of eight elements a thread keeps; 0: a row too long for the
// registers, read a second time (from L2) instead.
template <int RES, bool INT8, int VPT>
__global__ void __launch_bounds__(kNormMaxThreads) fg_add_rmsnorm_kernel(const NormParams p) {
  using ResT = typename std::conditional<RES == 2, float, __half>::type;
  const long long row = blockIdx.x;
  const int nvec = p.K >> 3, tid = threadIdx.x, threads = blockDim.x;
  const __half* x = p.x + row * p.ldx;
  const ResT* res = static_cast<const ResT*>(p.residual) + row * p.K;
  ResT* res_out = static_cast<ResT*>(p.residual_out) + row * p.K;
  griddep_wait();
  griddep_launch_dependents();

  auto load_h = [&](int v, float (&h)[8]) {
    load8(x + 8 * v, h);
    if (RES != 0) {
      float r[8];
      load8(res + 8 * v, r);
#pragma unroll
      for (int i = 0; i < 8; ++i) h[i] += r[i];
    }
  };
  constexpr int kKeep = VPT > 0 ? VPT : 1;
  float keep[kKeep][8];  // h, or t for int8 output
  float sum = 0.f, top = 0.f;
  auto gather = [&](float (&h)[8], const float (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      sum = fmaf(h[i], h[i], sum);
      h[i] = __fmul_rn(h[i], w[i]);
      if (INT8) top = max_nan(top, fabsf(h[i]));
    }
  };
  if constexpr (VPT > 0) {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (tid + j * threads < nvec) load_h(tid + j * threads, keep[j]);
#pragma unroll
    for (int j = 0; j < VPT; ++j) {
      const int v = tid + j * threads;
      if (v < nvec) {
        if (RES != 0) store8(res_out + 8 * v, keep[j]);
        float w[8];
        load8(p.weight + 8 * v, w);
        gather(keep[j], w);
      }
    }
  } else {
    for (int v = tid; v < nvec; v += threads) {
      float w[8];
      load_h(v, keep[0]);
      load8(p.weight + 8 * v, w);
      gather(keep[0], w);
    }
  }

  __shared__ float2 part[32];
#pragma unroll
  for (int off = 16; off >= 1; off >>= 1) {
    sum += __shfl_xor_sync(0xffffffffu, sum, off);
    if (INT8) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
  }
  if (threads > 32) {
    if ((tid & 31) == 0) part[tid >> 5] = make_float2(sum, top);
    __syncthreads();
    const float2 q = (tid & 31) < (threads >> 5) ? part[tid & 31] : make_float2(0.f, 0.f);
    sum = q.x;
    top = q.y;
#pragma unroll
    for (int off = 16; off >= 1; off >>= 1) {
      sum += __shfl_xor_sync(0xffffffffu, sum, off);
      if (INT8) top = max_nan(top, __shfl_xor_sync(0xffffffffu, top, off));
    }
  }
  float rstd = 1.f / sqrtf(sum / static_cast<float>(p.K) + p.eps);
  if (RES == 2 && !(sum <= kLargest)) {  // (the whole CTA: every thread holds the same sum)
    float far = 0.f;
    for (int v = tid; v < nvec; v += threads) {
      float h[8];
      if constexpr (VPT > 0 && RES == 2) load8(res_out + 8 * v, h);  // what this thread has just stored
      else load_h(v, h);
#pragma unroll
      for (int i = 0; i < 8; ++i) far = fmaf(h[i] * kFar, h[i] * kFar, far);
    }
    __shared__ float far_part[32];
    for (int off = 16; off >= 1; off >>= 1) far += __shfl_xor_sync(0xffffffffu, far, off);
    if ((tid & 31) == 0) far_part[tid >> 5] = far;
    __syncthreads();
    far = 0.f;
    for (int i = 0; i < (threads >> 5); ++i) far += far_part[i];
    rstd = kFar / sqrtf(far / static_cast<float>(p.K) + p.eps * kFar * kFar);
  }
  // The largest finite factor stands in for 127 / a where that overflows (a below 4e-37).
  const float factor = INT8 ? (top > 0.f ? fminf(__fdiv_rn(127.f, top), kLargest) : 0.f) : rstd;
  if (INT8 && tid == 0) {
    // `top` is infinite or NaN if some t is, be it from the row or from the weight
    p.scales[row] = top <= kLargest ? (top > 0.f ? top * rstd / 127.f : 1.f) : __int_as_float(0x7fc00000);
  }

  auto emit = [&](int v, float (&t)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] = __fmul_rn(t[i], factor);
    if constexpr (INT8) store8(static_cast<int8_t*>(p.out) + row * p.K + 8 * v, t);
    else store8(static_cast<__half*>(p.out) + row * p.K + 8 * v, t);
  };
  if constexpr (VPT > 0) {
#pragma unroll
    for (int j = 0; j < VPT; ++j)
      if (tid + j * threads < nvec) emit(tid + j * threads, keep[j]);
  } else {
    for (int v = tid; v < nvec; v += threads) {
      float w[8];
      load_h(v, keep[0]);
      if (RES != 0) store8(res_out + 8 * v, keep[0]);
      load8(p.weight + 8 * v, w);
#pragma unroll
      for (int i = 0; i < 8; ++i) keep[0][i] = __fmul_rn(keep[0][i], w[i]);
      emit(v, keep[0]);
    }
  }
}

using NormFn = void (*)(const NormParams);

template <int RES, bool INT8>
NormFn pick_norm(int vpt) {
  switch (vpt) {
    case 1: return fg_add_rmsnorm_kernel<RES, INT8, 1>;
    case 2: return fg_add_rmsnorm_kernel<RES, INT8, 2>;
    case 4: return fg_add_rmsnorm_kernel<RES, INT8, 4>;
    default: return fg_add_rmsnorm_kernel<RES, INT8, 0>;
  }
}

}  // namespace
}  // namespace fg

extern "C" int fg_add_rmsnorm(const void* x, long long ldx, const void* weight, const void* residual, void* residual_out,
                              int residual_f32, void* out, int out_int8, float* scales, int M, int K, float eps,
                              fg_stream_t stream) {
  using namespace fg;
  if (x == nullptr || weight == nullptr || out == nullptr || (out_int8 && scales == nullptr)) return FG_ERR_NULL;
  if ((residual == nullptr) != (residual_out == nullptr)) return FG_ERR_NULL;
  if (M <= 0 || K <= 0 || (K % 8) != 0 || ldx < K || (ldx % 8) != 0) return FG_ERR_SHAPE;
  if (!(eps >= 0.f)) return FG_ERR_SHAPE;
  if (!host::aligned(x, 16) || !host::aligned(weight, 16) || !host::aligned(residual, 16) || !host::aligned(residual_out, 16) ||
      !host::aligned(out, out_int8 ? 8 : 16) || !host::aligned(scales, 4))
    return FG_ERR_ALIGN;
  host::Device dev;
  const int st = host::current_device(&dev);
  if (st != FG_OK) return st;
  // Few rows: as many threads a row as it has vectors, the latency of one load is all there is (16 x 8192 2.4 us, with 512
  // threads 2.8; 296 x 8192 3.7 / 4.1).  Many rows: 512 threads at most, whose CTAs do not leave an SM half empty between two
  // rows (4096 x 8192, fp16 residual: 42.2 us with 512 threads, 44.5 with 1024; 2048 x 16384: 49.6 / 55.1; fewer threads with
  // more vectors each are slower too: 8192 x 4096 40.9 with 512, 44.5 with 128).
  const int nvec = K / 8, most_threads = M <= 2 * dev.sm_count ? kNormMaxThreads : kNormMaxThreads / 2;
  int vpt = 1;
  while (vpt < 4 && (nvec + vpt - 1) / vpt > most_threads) vpt *= 2;
  int threads = ((nvec + vpt - 1) / vpt + 31) / 32 * 32;
  if (threads > kNormMaxThreads) {
    vpt = 0;
    threads = kNormMaxThreads;
  }
  const int res = residual == nullptr ? 0 : residual_f32 ? 2 : 1;
  NormFn kern = out_int8 ? (res == 0 ? pick_norm<0, true>(vpt) : res == 1 ? pick_norm<1, true>(vpt) : pick_norm<2, true>(vpt))
                         : (res == 0 ? pick_norm<0, false>(vpt) : res == 1 ? pick_norm<1, false>(vpt) : pick_norm<2, false>(vpt));
  NormParams p = {};
  p.x = static_cast<const __half*>(x);
  p.ldx = ldx;
  p.weight = static_cast<const __half*>(weight);
  p.residual = residual;
  p.residual_out = residual_out;
  p.out = out;
  p.scales = scales;
  p.K = K;
  p.eps = eps;
  return host::launch(kern, dim3(static_cast<unsigned>(M)), dim3(threads), 0, reinterpret_cast<cudaStream_t>(stream), true, p);
}

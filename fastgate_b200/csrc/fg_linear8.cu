// fg_linear_w8a8: int8 activations x int8 weights with scales, bias, activation and residual.
//
// One or two token rows: a GEMV (fg_gemv8_kernel).  Up to 128 the weight is still the traffic and the streaming kernel of the fp16 linears runs on it
// (fg_umma_kernel<kOpW8A8NK>: the same bytes per stage, half the bytes per weight); above, the tensor cores are the
// bound (fg_gemm8_kernel).
#include <cuda.h>
#include <cuda_runtime.h>

#include "../../include/fastgate_b200.h"
#include "fg_gemm8.cuh"
#include "fg_gemv8.cuh"
#include "fg_host.h"
#include "fg_layout.h"
#include "fg_umma.cuh"

namespace {

using fg::host::aligned;

constexpr int kStreamRows = 128;       // token rows the streaming kernel takes
constexpr int kMaxK = 131072 - 128;    // k (-128)(-128) < 2^31

struct Args {
  const void *x, *W, *x_scales, *w_scales;
  int x_scales_f32;
  void* C;
  int M, N, K;
  const void *bias, *residual;
  int act;
};

int run_streaming(const Args& a, const fg::host::Device& dev, void* ws, cudaStream_t stream) {
  using StreamFn = void (*)(const CUtensorMap, const CUtensorMap, const fg::KParams);
  const bool gate = a.act == FG_ACT_SILU_GATE;
  fg_plan_t pl;
  int st = fg_plan_w8a8(a.M, a.N, a.K, dev.sm_count, dev.smem_optin, gate ? static_cast<int>(fg::kGateXchBytes) : 0, &pl);
  if (st != FG_OK) return st;
  const StreamFn kern = pl.m_tile == 16   ? fg::fg_umma_kernel<fg::kOpW8A8NK, 16>
                        : pl.m_tile == 32 ? fg::fg_umma_kernel<fg::kOpW8A8NK, 32>
                        : pl.m_tile == 64 ? fg::fg_umma_kernel<fg::kOpW8A8NK, 64>
                                          : fg::fg_umma_kernel<fg::kOpW8A8NK, 128>;
  if ((st = fg::host::opt_in_smem(reinterpret_cast<const void*>(kern), pl.smem_bytes)) != FG_OK) return st;
  CUtensorMap tmW, tmX;
  if ((st = fg::host::encode_tensor(&tmW, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.W, a.K, a.N, 128, 128)) != FG_OK) return st;
  if ((st = fg::host::encode_tensor(&tmX, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.x, a.K, a.M, 128, pl.m_tile)) != FG_OK) return st;
  uint8_t* wsb = static_cast<uint8_t*>(ws);
  fg::KParams p = {};
  p.C = static_cast<__half*>(a.C);
  p.scales = static_cast<const __half*>(a.w_scales);
  p.scale_groups = 1;
  p.x_scales = a.x_scales;
  p.x_scales_f32 = a.x_scales_f32;
  p.partials = reinterpret_cast<float*>(wsb + FG_WS_HEADER_BYTES);
  p.tickets = reinterpret_cast<unsigned int*>(wsb + FG_WS_TICKETS_OFFSET);
  p.status = reinterpret_cast<int*>(wsb);
  p.M = a.M;
  p.N = a.N;
  p.K = a.K;
  p.tiles = pl.tiles;
  p.k_blocks = pl.k_blocks;
  p.chunks_per_stage = pl.k_per_stage / fg_chunk_k(pl.op);
  p.stages = pl.stages;
  p.consumer_warps = pl.consumer_warps;
  p.pdl = pl.pdl;
  p.l2_prefetch = FG_L2_PREFETCH_BYTES / (p.chunks_per_stage * FG_CHUNK_W_BYTES);
  p.bias = static_cast<const __half*>(a.bias);
  p.residual = static_cast<const __half*>(a.residual);
  p.act = a.act;
  p.ldc = a.N;
  return fg::host::launch(kern, dim3(pl.grid), dim3(fg::kUmmaThreads), pl.smem_bytes, stream, true, tmW, tmX, p);
}

int run_gemv(const Args& a, cudaStream_t stream) {
  fg::Gemv8Params p = {};
  p.x = static_cast<const int8_t*>(a.x);
  p.W = static_cast<const int8_t*>(a.W);
  p.out.C = static_cast<__half*>(a.C);
  p.out.scales = static_cast<const __half*>(a.w_scales);
  p.out.x_scales = a.x_scales;
  p.out.x_scales_f32 = a.x_scales_f32;
  p.out.bias = static_cast<const __half*>(a.bias);
  p.out.residual = static_cast<const __half*>(a.residual);
  p.out.act = a.act;
  p.out.M = a.M;
  p.out.N = a.N;
  p.out.K = a.K;
  // the SiLU gate pairs a gate row with its up row in one warp
  const int R = a.act == FG_ACT_SILU_GATE || static_cast<long long>(a.N) * a.K > fg::kGemv8TwoRowBytes ? 2 : 1;
  const long long warps = (a.N + R - 1) / R, grid = (warps + fg::kGemv8Warps - 1) / fg::kGemv8Warps;
  void (*kern)(const fg::Gemv8Params) = a.M == 1 ? (R == 1 ? fg::fg_gemv8_kernel<1, 1> : fg::fg_gemv8_kernel<1, 2>)
                                                 : (R == 1 ? fg::fg_gemv8_kernel<2, 1> : fg::fg_gemv8_kernel<2, 2>);
  return fg::host::launch(kern, dim3(static_cast<unsigned>(grid)), dim3(fg::kGemv8Warps * 32), 0, stream, true, p);
}

template <int CG, int BN>
int run_gemm(const Args& a, const fg::host::Device& dev, void* ws, cudaStream_t stream) {
  const auto kern = fg::fg_gemm8_kernel<CG, BN>;
  int stages = (dev.smem_optin - fg::gemm8_smem_bytes(CG, BN, 0)) / (fg::gemm8_stage_bytes(CG, BN) + 16);
  if (stages > FG_MAX_STAGES) stages = FG_MAX_STAGES;
  if (stages < 2) return FG_ERR_PLAN;
  const int smem = fg::gemm8_smem_bytes(CG, BN, stages);
  int st = fg::host::opt_in_smem(reinterpret_cast<const void*>(kern), smem);
  if (st != FG_OK) return st;
  CUtensorMap tmW, tmX;
  if ((st = fg::host::encode_tensor(&tmX, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.x, a.K, a.M, 128, 128)) != FG_OK) return st;
  if ((st = fg::host::encode_tensor(&tmW, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, a.W, a.K, a.N, 128, BN / CG)) != FG_OK) return st;
  fg::Gemm8Params p = {};
  p.C = static_cast<__half*>(a.C);
  p.x_scales = a.x_scales;
  p.x_scales_f32 = a.x_scales_f32;
  p.w_scales = static_cast<const __half*>(a.w_scales);
  p.bias = static_cast<const __half*>(a.bias);
  p.residual = static_cast<const __half*>(a.residual);
  p.M = a.M;
  p.N = a.N;
  p.K = a.K;
  p.act = a.act;
  p.tiles_m = (a.M + 128 * CG - 1) / (128 * CG);
  p.tiles_n = (a.N + BN - 1) / BN;
  p.stages = stages;
  p.status = static_cast<int*>(ws);
  if (static_cast<long long>(p.tiles_m) * p.tiles_n > 0x3fffffffLL) return FG_ERR_SHAPE;
  const int tiles = p.tiles_m * p.tiles_n, groups = tiles < dev.sm_count / CG ? tiles : dev.sm_count / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups * CG);
  cfg.blockDim = dim3(fg::kGemm8Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 1 ? 1 : 2;
  return fg::host::launched(cudaLaunchKernelEx(&cfg, kern, tmX, tmW, p));
}

}  // namespace

extern "C" int fg_linear_w8a8(const int8_t* x8, const int8_t* W8, const void* x_scales, int x_scales_f32, const void* w_scales, void* C,
                              int M, int N, int K, const void* bias, const void* residual, int act, void* ws, size_t ws_bytes,
                              fg_stream_t stream) {
  if (x8 == nullptr || W8 == nullptr || C == nullptr || x_scales == nullptr) return FG_ERR_NULL;
  if (M <= 0 || N <= 0 || K <= 0 || (N % 128) != 0 || (K % 128) != 0 || K > kMaxK) return FG_ERR_SHAPE;
  if (act < FG_ACT_NONE || act > FG_ACT_SILU_GATE) return FG_ERR_PLAN;
  if (!aligned(x8, 16) || !aligned(W8, 16) || !aligned(C, 16) || !aligned(residual, 16) || !aligned(x_scales, x_scales_f32 ? 4 : 2) ||
      !aligned(w_scales, 2) || !aligned(bias, 2))
    return FG_ERR_ALIGN;
  if (ws == nullptr || !aligned(ws, 256) || ws_bytes < FG_WS_TICKETS_OFFSET + 4 * static_cast<size_t>(N / 128)) return FG_ERR_WORKSPACE;
  fg::host::Device dev;
  const int st = fg::host::current_device(&dev);
  if (st != FG_OK) return st;
  const Args a = {x8, W8, x_scales, w_scales, x_scales_f32, C, M, N, K, bias, residual, act};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (M <= fg::kGemv8MaxM) return run_gemv(a, s);
  if (M <= kStreamRows) return run_streaming(a, dev, ws, s);
  // Pairs of CTAs once their tiles fill the card, single CTAs with smaller tiles below.
  const long long pair_tiles = static_cast<long long>((M + 255) / 256) * ((N + 255) / 256);
  if (2 * pair_tiles >= dev.sm_count) return run_gemm<2, 256>(a, dev, ws, s);
  return run_gemm<1, 128>(a, dev, ws, s);
}

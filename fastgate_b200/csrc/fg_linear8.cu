// fg_linear_w8a8: int8 activations x int8 weights with scales, bias, activation and residual.
//
// One or two token rows: a GEMV (fg_gemv8_kernel); more: a tensor-core kernel (fg_gemm8_kernel) with tiles chosen by size.
#include <cuda.h>
#include <cuda_runtime.h>

#include <mutex>

#include "../../include/fastgate_b200.h"
#include "fg_gemm8.cuh"
#include "fg_gemv8.cuh"
#include "fg_host.h"
#include "fg_layout.h"

namespace {

using fg::host::aligned;

constexpr int kMaxK = 131072 - 128;    // k (-128)(-128) < 2^31

int run_gemv(const fg::W8A8Params& a, const int8_t* x, const int8_t* W, cudaStream_t stream) {
  // the SiLU gate pairs a gate row with its up row in one warp
  const int R = a.act == FG_ACT_SILU_GATE || static_cast<long long>(a.N) * a.K > fg::kGemv8TwoRowBytes ? 2 : 1;
  const long long warps = (a.N + R - 1) / R, grid = (warps + fg::kGemv8Warps - 1) / fg::kGemv8Warps;
  void (*kern)(const fg::Gemv8Params) = a.M == 1 ? (R == 1 ? fg::fg_gemv8_kernel<1, 1> : fg::fg_gemv8_kernel<1, 2>)
                                                 : (R == 1 ? fg::fg_gemv8_kernel<2, 1> : fg::fg_gemv8_kernel<2, 2>);
  const fg::Gemv8Params p = {x, W, a};
  return fg::host::launch(kern, dim3(static_cast<unsigned>(grid)), dim3(fg::kGemv8Warps * 32), 0, stream, true, p);
}

// ---- tiles of the tensor-core kernel ------------------------------------------------------------
struct Tiling {
  int bn;      // weight rows of a tile
  int cg;      // CTAs that share a tile's MMAs: 1 (128 token rows) or 2 (256)
  int splits;  // CTAs that share a tile's k (cg 1)
  int wide;    // cg 2: columns of tiles of full width; the others have `narrow` weight rows
  int narrow;
};

struct TileCost {
  int bn, cg;
  double few_us, many_us;  // one block of 128 k on one CTA (pair), with one row of token tiles and with several
};
// Measured on B200 (M = 3 to 128 and 256 to 4096; N = 1024 to 28672, K = 4096 to 11008): time per wave less 3.5 us, over the
// blocks of k.  Narrow tiles are bound by the issue of their four MMAs a block, wide ones by the tensor cores and L2.
constexpr TileCost kTileCosts[] = {{32, 1, 0.148, 0.155}, {64, 1, 0.163, 0.18}, {96, 1, 0.175, 0.21}, {128, 1, 0.22, 0.25},
                                   {192, 1, 0.265, 0.32}, {256, 1, 0.36, 0.40}, {256, 2, 0.36, 0.36}};
constexpr double kNarrowUs[] = {0.17, 0.22, 0.28};  // the same of a pair's tile with 64, 128 and 192 weight rows
constexpr double kSplitUs = 3.5;    // launch of clusters, two cluster barriers and the exchange between them
constexpr double kDramBytesPerUs = 6.2e6;

int stages_of(const TileCost& c, int smem_optin) {
  const int s = (smem_optin - fg::gemm8_smem_bytes(c.cg, c.bn, 0)) / (fg::gemm8_stage_bytes(c.cg, c.bn) + 16);
  return s < FG_MAX_STAGES ? s : FG_MAX_STAGES;
}

// The tiling with the least estimated time: per wave of tiles its blocks of k or its share of the bytes, whichever takes
// longer (a last wave of a few tiles costs as much as a full one where the tensor cores bound it, little where memory does).
// clusters: how many clusters of 2, 4 and 8 CTAs the device holds at once.
Tiling choose_tiling(int M, int N, int K, bool gated, int sm_count, int smem_optin, const int (&clusters)[3]) {
  const double dram = (static_cast<double>(N) * K + static_cast<double>(M) * K + 2.0 * M * N) / kDramBytesPerUs;
  Tiling best = {128, 1, 1, 0, 0};
  double best_us = 1e30;
  for (const TileCost& c : kTileCosts) {
    if (gated && (c.bn == 96 || c.bn == 192)) continue;  // a gate row and its up row belong to one tile
    const long long tiles = static_cast<long long>((M + 128 * c.cg - 1) / (128 * c.cg)) * ((N + c.bn - 1) / c.bn);
    const int per = fg::gemm8_blocks_per_stage(c.cg, c.bn), k_stages = (K / 128 + per - 1) / per;
    const int ring = stages_of(c, smem_optin) * fg::gemm8_stage_bytes(c.cg, c.bn);
    for (int s = 1, log = 0; s <= (c.cg == 1 ? 8 : 1); s *= 2, ++log) {
      // All clusters run at once (a second wave of a few costs as much again: 16 x 512 x 8192 15.6 us with 16 clusters of 8 on a
      // device that holds fewer).  Every CTA has a stage at least, and the followers' sums fit in the leader's ring.
      if (s > 1 && (tiles > clusters[log - 1] || k_stages < s || (s - 1) * c.bn * 512 > ring)) break;
      const long long at_once = s > 1 ? tiles : sm_count / c.cg;
      const int blocks = s > 1 ? (k_stages + s - 1) / s * per : K / 128;
      const double mma = blocks * (M <= 128 ? c.few_us : c.many_us);
      const long long full = tiles / at_once, rest = tiles % at_once;
      const double full_dram = dram * at_once / tiles, rest_dram = dram * rest / tiles;
      const double us = full * (mma > full_dram ? mma : full_dram) + (rest ? (mma > rest_dram ? mma : rest_dram) : 0.0) + (s > 1 ? kSplitUs : 0.0);
      if (us < best_us) {
        best_us = us;
        best = {c.bn, c.cg, s, (N + c.bn - 1) / c.bn, c.bn};
      }
    }
  }
  // Pairs: a last wave that is far from full may be a wave of narrower tiles instead.  (A row of tiles spans the waves: what counts is
  // how many waves have a wide tile in them and how many have none.  512 x 28672 x 8192: 98.6 us with wide tiles alone, 90.7;
  // 512 x 11008 x 4096: 25.0 / 23.2; 3001 x 4096 x 11008: 100 / 98.8.)
  const int pairs = sm_count / 2, tiles_m = (M + 255) / 256, blocks = K / 128;
  for (int i = 0; i < 3; ++i) {
    const int narrow = 64 * (i + 1);
    if (gated && narrow != 128) continue;
    for (int wide = N / 256; wide >= 0 && wide >= N / 256 - 64; --wide) {
      const long long wide_tiles = static_cast<long long>(tiles_m) * wide, tiles = wide_tiles + static_cast<long long>(tiles_m) * ((N - 256 * wide + narrow - 1) / narrow);
      if (tiles == wide_tiles || wide_tiles < pairs) continue;
      const long long wide_waves = (wide_tiles + pairs - 1) / pairs, waves = (tiles + pairs - 1) / pairs;
      double us = blocks * (wide_waves * 0.36 + (waves - wide_waves) * kNarrowUs[i]);
      if (us < dram) us = dram;
      if (us < 0.98 * best_us) {
        best_us = us;
        best = {256, 2, 1, wide, narrow};
      }
    }
  }
  return best;
}

// A cluster lives in one GPC, and how many SMs of a GPC are in use differs from device to device.  No more than seven eighths of
// the SMs are counted on in any case.
void cluster_limits(int sm_count, int (&clusters)[3]) {
  for (int i = 0; i < 3; ++i) clusters[i] = (sm_count - sm_count / 8) >> (i + 1);
}
constexpr int kMaxDevices = 64;  // as many as fg_capi.cu keeps
int clusters_at_once(const fg::host::Device& dev, int (&clusters)[3]) {
  static std::mutex mu;
  static int known[kMaxDevices][3];  // (no container: an allocation that fails may not throw out of a C entry point)
  static bool asked[kMaxDevices];
  if (dev.index < 0 || dev.index >= kMaxDevices) return FG_ERR_NO_DEVICE;
  std::lock_guard<std::mutex> lk(mu);
  int(&found)[3] = known[dev.index];
  if (!asked[dev.index]) {
    // (Every tiling's ring takes an SM's shared memory, so one kernel speaks for all.)
    const auto kern = fg::fg_gemm8_kernel<1, 64>;
    const int smem = fg::gemm8_smem_bytes(1, 64, stages_of({64, 1, 0.0, 0.0}, dev.smem_optin));
    const int st = fg::host::opt_in_smem(reinterpret_cast<const void*>(kern), smem);
    if (st != FG_OK) return st;
    for (int i = 0; i < 3; ++i) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(dev.sm_count / (2 << i) * (2 << i));
      cfg.blockDim = dim3(fg::kGemm8Threads);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = 2 << i;
      attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr;
      cfg.numAttrs = 1;
      const cudaError_t e = cudaOccupancyMaxActiveClusters(&found[i], kern, &cfg);
      if (e != cudaSuccess) {
        fg::host::launched(e);
        return FG_ERR_CUDA;
      }
    }
    asked[dev.index] = true;
  }
  cluster_limits(dev.sm_count, clusters);
  for (int i = 0; i < 3; ++i) clusters[i] = clusters[i] < found[i] ? clusters[i] : found[i];
  return FG_OK;
}

template <int CG, int BN>
int run_gemm(const fg::W8A8Params& a, const int8_t* x, const int8_t* W, const Tiling& t, const fg::host::Device& dev, cudaStream_t stream) {
  const int splits = t.splits;
  const auto kern = fg::fg_gemm8_kernel<CG, BN>;
  const int stages = stages_of({BN, CG, 0.0, 0.0}, dev.smem_optin);
  if (stages < 2) return FG_ERR_PLAN;
  const int smem = fg::gemm8_smem_bytes(CG, BN, stages);
  int st = fg::host::opt_in_smem(reinterpret_cast<const void*>(kern), smem);
  if (st != FG_OK) return st;
  const int x_rows = CG == 1 && a.M < 128 ? (a.M + 7) / 8 * 8 : 128;
  const int w_rows = fg::gemm8_box_rows(CG, BN, a.act == FG_ACT_SILU_GATE);
  const int wide = CG == 2 ? t.wide : (a.N + BN - 1) / BN, narrow = CG == 2 ? t.narrow : BN;
  CUtensorMap tmW, tmX, tmNarrow;
  if ((st = fg::host::encode_tensor(&tmX, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, x, a.K, a.M, 128, x_rows)) != FG_OK) return st;
  if ((st = fg::host::encode_tensor(&tmW, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, W, a.K, a.N, 128, w_rows)) != FG_OK) return st;
  tmNarrow = tmW;
  if (narrow != BN && (st = fg::host::encode_tensor(&tmNarrow, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, W, a.K, a.N, 128, narrow / CG)) != FG_OK) return st;
  fg::Gemm8Params p = {};
  p.out = a;
  p.tiles_m = (a.M + 128 * CG - 1) / (128 * CG);
  const int rest = a.N - wide * BN;  // (of full columns alone the last may reach over N)
  p.tiles_n = wide + (rest > 0 ? (rest + narrow - 1) / narrow : 0);
  p.wide = wide;
  p.narrow = narrow;
  p.stages = stages;
  p.splits = splits;
  p.x_rows = x_rows;
  if (static_cast<long long>(p.tiles_m) * p.tiles_n > 0x3fffffffLL) return FG_ERR_SHAPE;
  const int cluster = CG * splits, tiles = p.tiles_m * p.tiles_n;
  const int groups = splits > 1 || tiles < dev.sm_count / cluster ? tiles : dev.sm_count / cluster;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(groups * cluster);
  cfg.blockDim = dim3(fg::kGemm8Threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster == 1 ? 1 : 2;
  return fg::host::launched(cudaLaunchKernelEx(&cfg, kern, tmX, tmW, tmNarrow, p));
}

}  // namespace

extern "C" int fg_linear_w8a8(const int8_t* x8, const int8_t* W8, const void* x_scales, int x_scales_f32, const void* w_scales, void* C,
                              int M, int N, int K, const void* bias, const void* residual, int act, int* status_dev,
                              fg_stream_t stream) {
  if (x8 == nullptr || W8 == nullptr || C == nullptr || x_scales == nullptr) return FG_ERR_NULL;
  if (M <= 0 || N <= 0 || K <= 0 || (N % 128) != 0 || (K % 128) != 0 || K > kMaxK) return FG_ERR_SHAPE;
  if (act < FG_ACT_NONE || act > FG_ACT_SILU_GATE) return FG_ERR_PLAN;
  if (!aligned(x8, 16) || !aligned(W8, 16) || !aligned(C, 16) || !aligned(residual, 16) || !aligned(x_scales, x_scales_f32 ? 4 : 2) ||
      !aligned(w_scales, 2) || !aligned(bias, 2) || !aligned(status_dev, 4))
    return FG_ERR_ALIGN;
  fg::host::Device dev;
  int st = fg::host::current_device(&dev);
  if (st != FG_OK) return st;
  fg::W8A8Params a = {};
  a.C = static_cast<__half*>(C);
  a.x_scales = x_scales;
  a.x_scales_f32 = x_scales_f32;
  a.w_scales = static_cast<const __half*>(w_scales);
  a.bias = static_cast<const __half*>(bias);
  a.residual = static_cast<const __half*>(residual);
  a.M = M;
  a.N = N;
  a.K = K;
  a.act = act;
  a.status = status_dev;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (M <= fg::kGemv8MaxM) return run_gemv(a, x8, W8, s);
  int clusters[3];
  if ((st = clusters_at_once(dev, clusters)) != FG_OK) return st;
  const Tiling t = choose_tiling(M, N, K, act == FG_ACT_SILU_GATE, dev.sm_count, dev.smem_optin, clusters);
  if (t.cg == 2) return run_gemm<2, 256>(a, x8, W8, t, dev, s);
  switch (t.bn) {
    case 32: return run_gemm<1, 32>(a, x8, W8, t, dev, s);
    case 64: return run_gemm<1, 64>(a, x8, W8, t, dev, s);
    case 96: return run_gemm<1, 96>(a, x8, W8, t, dev, s);
    case 128: return run_gemm<1, 128>(a, x8, W8, t, dev, s);
    case 192: return run_gemm<1, 192>(a, x8, W8, t, dev, s);
    default: return run_gemm<1, 256>(a, x8, W8, t, dev, s);
  }
}

// Internal (for the tests): the tiling of a call as bn | cg << 16 | splits << 24, as far as the device holds its clusters.
extern "C" int fg_linear_w8a8_tiling(int M, int N, int K, int gated, int sm_count, int smem_optin) {
  int clusters[3];
  cluster_limits(sm_count, clusters);
  const Tiling t = choose_tiling(M, N, K, gated != 0, sm_count, smem_optin, clusters);
  return t.bn | t.cg << 16 | t.splits << 24;
}

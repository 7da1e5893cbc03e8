// int8 x int8 GEMM for many token rows (fg_linear_w8a8 above the streaming kernel's range).
//
//   C[m, n] = act(sx[m] sw[n] sum_k x[m, k] W[n, k] + bias[n]) + residual[m, n]
//
// With hundreds of token rows the weight no longer bounds the call, the tensor cores do: 2 M N K operations against
// M K + N K + 2 M N bytes.  tcgen05.mma.kind::i8, accumulators in tensor memory, 128-byte rows of k staged by TMA:
//
//   CG = 2: two CTAs of a cluster share one 256 x BN tile (cta_group::2).  Each loads its own 128 token rows and half of
//           the tile's weight rows; the tensor cores of both read both halves of the weights.  A CTA alone at 128 x 256
//           would fetch 48 KB from L2 per 128 k for the same 128 x 256 products, the pair fetches 32 KB per CTA, which is
//           what L2 can deliver at full tensor rate.  One thread of the leading CTA issues every MMA.
//   CG = 1: one CTA per 128 x BN tile, for problems with too few tiles to fill the card with pairs.
//
// Persistent: CTAs (pairs) take tiles blockIdx.x, + gridDim.x, ... with the token tiles innermost, so that the tiles in
// flight share weight rows in L2.  Two accumulators alternate: the epilogue of one tile overlaps the MMAs of the next.
// Warps 0-3: epilogue (TMEM lane = token row), 4: copies, 5: MMA.  Sums are exact 32-bit integers.
#pragma once
#include "fg_umma.cuh"

namespace fg {

constexpr int kGemm8Threads = 192;

struct Gemm8Params {
  __half* C;
  const void* x_scales;      // [M] fp32 or fp16
  int x_scales_f32;
  const __half* w_scales;    // [N] or nullptr
  const __half* bias;        // [N] or nullptr
  const __half* residual;    // [M, N] ([M, N/2] with the SiLU gate) or nullptr
  int M, N, K;
  int act;
  int tiles_m, tiles_n;
  int stages;
  int* status;
};

__host__ __device__ constexpr int gemm8_stage_bytes(int cg, int bn) { return (128 + bn / cg) * 128; }
__host__ __device__ constexpr int gemm8_smem_bytes(int cg, int bn, int stages) {
  return 1024 + stages * (gemm8_stage_bytes(cg, bn) + 16) + 64 + bn * 8;
}

// ---- pairs of CTAs -----------------------------------------------------------------------
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t mapped_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(mapped_bar) : "memory");
}
// Load into this CTA's shared memory that counts its bytes on the leading CTA's barrier.
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const void* tmap, uint32_t mapped_bar, int c0, int c1, uint64_t policy) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint"
      " [%0], [%1, {%3, %4}], [%2], %5;" ::"r"(dst),
      "l"(tmap), "r"(mapped_bar), "r"(c0), "r"(c1), "l"(policy)
      : "memory");
}
template <int CG>
__device__ __forceinline__ void gemm8_mma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1) {
    umma_i8(tmem_d, adesc, bdesc, idesc, accumulate);
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// One arrival on the barrier at this offset in every CTA of the group once all MMAs issued so far have completed.
template <int CG>
__device__ __forceinline__ void gemm8_commit(uint32_t bar) {
  if constexpr (CG == 1) {
    umma_commit(bar);
  } else {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
                 "h"(static_cast<uint16_t>(3))
                 : "memory");
  }
}

template <int CG, int BN>
__global__ void __launch_bounds__(kGemm8Threads, 1)
    fg_gemm8_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW, const Gemm8Params p) {
  constexpr int kStage = gemm8_stage_bytes(CG, BN);
  constexpr uint32_t kCols = 2 * BN;  // TMEM columns: two accumulators of BN
  static_assert(kCols <= 512 && (kCols & (kCols - 1)) == 0, "tensor memory");
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
  const int S = p.stages;
  const uint32_t bar_full = smem_base + S * kStage;   // [S], the leading CTA's are the ones in use
  const uint32_t bar_empty = bar_full + 8 * S;        // [S], each CTA its own
  const uint32_t bar_acc_full = bar_empty + 8 * S;    // [2], each CTA its own
  const uint32_t bar_acc_empty = bar_acc_full + 16;   // [2], the leading CTA's
  const uint32_t tmem_slot = bar_acc_empty + 16;
  volatile uint32_t* tmem_slot_gen = reinterpret_cast<volatile uint32_t*>(smem_gen + (tmem_slot - smem_base));
  float* col_scale = reinterpret_cast<float*>(smem_gen + (tmem_slot + 16 - smem_base));  // [BN]
  float* col_bias = col_scale + BN;                                                      // [BN]

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      mbar_init(bar_full + 8 * s, 1);   // the leader's expect_tx for all CTAs' bytes
      mbar_init(bar_empty + 8 * s, 1);  // one commit
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full + 8 * b, 1);        // one commit
      mbar_init(bar_acc_empty + 8 * b, 4 * CG);  // lane 0 of every epilogue warp
    }
    fence_mbar_init();
    fence_proxy_async();
  }
  if (warp == 5) {
    if constexpr (CG == 1) {
      tmem_alloc(tmem_slot, kCols);
      tmem_relinquish();
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(kCols) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_gen;
  griddep_launch_dependents();
  griddep_wait();

  const int tiles = p.tiles_m * p.tiles_n, groups = gridDim.x / CG, group = blockIdx.x / CG;
  const int k_blocks = p.K / 128;
  bool dead = false;

  if (warp == 4) {
    if (lane == 0) {
      tma_prefetch_desc(&tmX);
      tma_prefetch_desc(&tmW);
      const uint64_t policy = policy_evict_last();  // both operands are read again by other tiles
      int s = 0, filled = 0;
      uint32_t ph = 1;  // the slots start out empty
      for (int t = group; t < tiles && !dead; t += groups) {
        const int m0 = (t % p.tiles_m) * (128 * CG) + 128 * rank, n0 = (t / p.tiles_m) * BN + (BN / CG) * rank;
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(bar_empty + 8 * s, ph, kWaitBudgetNs)) {
            dead = true;
            break;
          }
          const uint32_t dst = smem_base + s * kStage;
          if constexpr (CG == 1) {
            mbar_arrive_expect_tx(bar_full + 8 * s, kStage);
            tma_load_2d(dst, &tmX, bar_full + 8 * s, kb * 128, m0, policy);
            tma_load_2d(dst + 16384, &tmW, bar_full + 8 * s, kb * 128, n0, policy);
          } else {
            const uint32_t lead = map_to_rank(bar_full + 8 * s, 0);
            if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * s, 2 * kStage);
            tma_load_2d_pair(dst, &tmX, lead, kb * 128, m0, policy);
            tma_load_2d_pair(dst + 16384, &tmW, lead, kb * 128, n0, policy);
          }
          ++filled;
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
      }
      // Every copy lands before the CTA may go: each filled slot has been consumed once more.  (After a wait that gave
      // up the same waits, bounded too, are all that can be done.)
      for (int i = 0; i < (filled < S ? filled : S); ++i) {
        const int back = (s - 1 - i + 2 * S) % S;
        const uint32_t use = static_cast<uint32_t>((filled - 1 - i) / S);
        if (!mbar_wait_bounded(bar_empty + 8 * back, use & 1, kWaitBudgetNs)) dead = true;
      }
      if (dead) atomicExch(p.status, kStatusTimeout);
    }
    __syncwarp();
  } else if (warp == 5) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t idesc = umma_idesc_i8(128 * CG, BN);
      constexpr uint64_t desc = umma_smem_desc(0, 1, 64);
      int s = 0, n = 0;
      uint32_t ph = 0;
      for (int t = group; t < tiles && !dead; t += groups, ++n) {
        const uint32_t b = n & 1, use = n >> 1;
        if (!mbar_wait_bounded(bar_acc_empty + 8 * b, (use & 1) ^ 1, kWaitBudgetNs)) {
          dead = true;
          break;
        }
        tc_fence_after_sync();
        for (int kb = 0; kb < k_blocks; ++kb) {
          if (!mbar_wait_bounded(bar_full + 8 * s, ph, kWaitBudgetNs)) {
            dead = true;
            break;
          }
          tc_fence_after_sync();
          const uint32_t at = smem_base + s * kStage;
          const uint64_t a = desc | ((at >> 4) & 0x3FFFu), w = desc | (((at + 16384) >> 4) & 0x3FFFu);
#pragma unroll
          for (int k = 0; k < 4; ++k) gemm8_mma<CG>(tmem_base + b * BN, a + 2 * k, w + 2 * k, idesc, (kb | k) != 0);
          gemm8_commit<CG>(bar_empty + 8 * s);
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!dead) gemm8_commit<CG>(bar_acc_full + 8 * b);
      }
      if (dead) atomicExch(p.status, kStatusTimeout);
    }
    __syncwarp();
  } else {
    const bool gated = p.act == kActSiluGate;
    const int width = gated ? p.N >> 1 : p.N;
    int n = 0;
    for (int t = group; t < tiles; t += groups, ++n) {
      const int m = (t % p.tiles_m) * (128 * CG) + 128 * rank + 32 * warp + lane, n0 = (t / p.tiles_m) * BN;
      const uint32_t b = n & 1, use = n >> 1;
      const bool row = m < p.M;
      float xs = 0.f;
      if (row) xs = p.x_scales_f32 ? static_cast<const float*>(p.x_scales)[m] : __half2float(static_cast<const __half*>(p.x_scales)[m]);
      named_bar_sync(1, 128);  // the previous tile's column values have been read
      for (int j = threadIdx.x; j < BN; j += 128) {
        const bool in = n0 + j < p.N;
        col_scale[j] = in && p.w_scales != nullptr ? __half2float(p.w_scales[n0 + j]) : 1.f;
        col_bias[j] = in && p.bias != nullptr ? __half2float(p.bias[n0 + j]) : 0.f;
      }
      named_bar_sync(1, 128);
      if (!dead && !__all_sync(0xffffffffu, mbar_wait_bounded(bar_acc_full + 8 * b, use & 1, 2 * kWaitBudgetNs))) {
        dead = true;
        if (lane == 0) atomicExch(p.status, kStatusTimeout);
      }
      if (dead) continue;
      tc_fence_after_sync();
      const uint32_t tbase = tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + b * BN;
      // The value of a sum before the activation, rounded step by step as in the other kernels on int8 activations.
      auto value = [&](uint32_t sum, int col) {
        return __fadd_rn(__fmul_rn(__fmul_rn(static_cast<float>(static_cast<int>(sum)), xs), col_scale[col]), col_bias[col]);
      };
      // Thirty-two columns at a time; a row's pieces leave as 16-byte stores.
      auto emit = [&](int col, const float (&v)[32]) {  // col: column of the output
        if (!row) return;
        __half* dst = p.C + static_cast<size_t>(m) * width + col;
        const __half* res = p.residual ? p.residual + static_cast<size_t>(m) * width + col : nullptr;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint4 r = make_uint4(0, 0, 0, 0), o;
          if (res != nullptr) r = *reinterpret_cast<const uint4*>(res + 8 * q);
          const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
          uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float2 f = make_float2(v[8 * q + 2 * i], v[8 * q + 2 * i + 1]);
            if (res != nullptr) {
              const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&rw[i]));
              f.x = __fadd_rn(f.x, a.x);
              f.y = __fadd_rn(f.y, a.y);
            }
            const __half2 h = __floats2half2_rn(f.x, f.y);
            ow[i] = *reinterpret_cast<const uint32_t*>(&h);
          }
          *reinterpret_cast<uint4*>(dst + 8 * q) = o;
        }
      };
      if (gated) {
#pragma unroll 1
        for (int c = 0; c < BN / 64; ++c) {  // (128-row block, half): 32 gate columns and the matching up columns
          const int at = (c >> 1) * 128 + (c & 1) * 32;
          uint32_t g[32], u[32];
          tmem_ld32(tbase + at, g);
          tmem_ld32(tbase + at + 64, u);
          tmem_ld_wait();
          if (n0 + at >= p.N) continue;
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float gv = value(g[i], at + i), uv = value(u[i], at + 64 + i);
            v[i] = __fmul_rn(act_fn<kActSilu>(gv), uv);
          }
          emit((n0 >> 1) + (c >> 1) * 64 + (c & 1) * 32, v);
        }
      } else {
        with_act(p.act, [&](auto tag) {
          constexpr int ACT = decltype(tag)::value;
#pragma unroll 1
          for (int c = 0; c < BN / 32; ++c) {
            uint32_t r[32];
            tmem_ld32(tbase + 32 * c, r);
            tmem_ld_wait();
            if (n0 + 32 * c >= p.N) continue;
            float v[32];
#pragma unroll
            for (int i = 0; i < 32; ++i)
              v[i] = act_fn<ACT>(value(r[i], 32 * c + i));
            emit(n0 + 32 * c, v);
          }
        });
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1) mbar_arrive(bar_acc_empty + 8 * b);
        else mbar_arrive_cluster(map_to_rank(bar_acc_empty + 8 * b, 0));
      }
    }
  }

  // ---- teardown: every MMA has completed (the epilogues have seen them) and the pair leaves together ----
  tc_fence_before_sync();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();
  if (warp == 5) {
    tc_fence_after_sync();
    if constexpr (CG == 1) {
      tmem_dealloc(tmem_base, kCols);
    } else {
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kCols) : "memory");
    }
  }
  if constexpr (CG == 2) cluster_sync();
}

}  // namespace fg

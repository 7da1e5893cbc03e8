// int8 x int8 GEMM (fg_linear_w8a8 from three token rows on).
//
//   C[m, n] = act(sx[m] sw[n] sum_k x[m, k] W[n, k] + bias[n]) + residual[m, n]
//
// 2 M N K operations against M K + N K + 2 M N bytes: the weight's bytes bound the call up to a few hundred token rows, the
// tensor cores above.  tcgen05.mma.kind::i8, accumulators in tensor memory, 128-byte rows of k staged by TMA:
//
//   CG = 2: two CTAs of a cluster share one 256 x 256 tile (cta_group::2).  Each loads its own 128 token rows and half of
//           the tile's weight rows; the tensor cores of both read both halves of the weights.  A CTA alone at 128 x 256
//           would fetch 48 KB from L2 per 128 k for the same 128 x 256 products, the pair fetches 32 KB per CTA, which is
//           what L2 can deliver at full tensor rate.  One thread of the leading CTA issues every MMA.  The last columns of
//           tiles may be narrower, so that the last wave of pairs is no longer than it has to be.
//   CG = 1: one CTA per 128 x BN tile.  BN (32 to 256) is chosen so that the tiles of a small problem fill the card: the
//           token rows beyond M cost no traffic and, next to the weight, no time.  Where even the narrowest tiles are too few,
//           a cluster of 2 to 8 CTAs shares one, each with its part of k: the followers push their sums into the leader's
//           shared memory, which has no copies in flight by then, and the leader finishes the tile.
//
// Persistent: CTAs (pairs) take tiles blockIdx.x, + gridDim.x, ... with the token tiles innermost, so that the tiles in
// flight share weight rows in L2.  Two accumulators alternate: the epilogue of one tile overlaps the MMAs of the next.
// The first ring-full of weights is asked for before the previous kernel of the stream has finished (the weight may not be that
// kernel's output).  Measured on B200: 3001 x 4096 x 11008 98 us (2.8 POP/s, tensor pipe 77 %: two waves of 74 pairs and one of
// narrower tiles), 16 x 28672 x 8192 with the SiLU gate 41 us (5.7 TB/s).  Far from their floor: 16 to 128 x 4096 x 4096 7.6 to 8.1 us
// (2.6 to 2.8) and 16 x 512 x 8192 7.5 (0.7), where each CTA issues four MMAs of 128 token rows for every 4 KB of weight, whatever M.  Warps 0-3: epilogue (TMEM lane = token row), 4: copies, 5: MMA.
// Sums are exact 32-bit integers.
#pragma once
#include "fg_umma.cuh"
#include "fg_w8a8.cuh"

namespace fg {

constexpr int kGemm8Threads = 192;

struct Gemm8Params {
  W8A8Params out;
  int tiles_m, tiles_n;
  int wide, narrow;          // CG = 2: the first `wide` columns of tiles have BN weight rows, the others `narrow` (a multiple of 64)
  int stages;
  int splits;                // CG = 1: CTAs of a cluster that share a tile, each with its part of k (1: none)
  int x_rows;                // token rows of one copy: 128, or fewer when M is below (the tile's other rows are left as they are:
                             // their products are computed from whatever the slot holds and never stored)
};

__host__ __device__ constexpr int gemm8_block_bytes(int cg, int bn) { return (128 + bn / cg) * 128; }
__host__ __device__ constexpr uint32_t gemm8_tmem_cols(int bn) { return bn <= 32 ? 64 : bn <= 64 ? 128 : bn <= 128 ? 256 : 512; }  // two accumulators
// Weight rows of one copy: with the SiLU gate a tile narrower than a block of 128 takes gate rows and up rows separately.
__host__ __device__ constexpr int gemm8_box_rows(int cg, int bn, bool gated) { return gated && bn / cg < 128 ? bn / 2 : bn / cg; }
// k blocks of 128 that a stage holds: the barrier traffic around a stage costs its two threads as much as the copies and MMAs
// of a block, so two where the ring stays three deep.
__host__ __device__ constexpr int gemm8_blocks_per_stage(int cg, int bn) { return gemm8_block_bytes(cg, bn) <= 32768 ? 2 : 1; }
__host__ __device__ constexpr int gemm8_stage_bytes(int cg, int bn) { return gemm8_blocks_per_stage(cg, bn) * gemm8_block_bytes(cg, bn); }
__host__ __device__ constexpr int gemm8_smem_bytes(int cg, int bn, int stages) {
  return 1024 + stages * (gemm8_stage_bytes(cg, bn) + 16) + 64 + bn * 8;
}

// int8 x int8 -> int32: the same operand geometry in bytes as fp16, 32 k per instruction.
__device__ __forceinline__ void umma_i8(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Instruction descriptor, kind::i8: signed A and B, 32-bit integer D, both K-major.
__host__ __device__ constexpr uint32_t umma_idesc_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((static_cast<uint32_t>(n) >> 3) << 17) | ((static_cast<uint32_t>(m) >> 4) << 24);
}

// One lane of a converged warp.  The loops of the copying and the MMA warp run on all lanes and only the instructions
// themselves on one: what they take then stays in uniform registers, where those instructions want it.
__device__ __forceinline__ bool elect_one() {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r != 0;
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
__device__ __forceinline__ void st_cluster(uint32_t mapped, uint32_t v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapped), "r"(v) : "memory");
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

// PIECE columns of this thread's TMEM lane.
template <int PIECE>
__device__ __forceinline__ void load_sums(uint32_t taddr, uint32_t (&r)[PIECE]) {
  if constexpr (PIECE == 32) tmem_ld32(taddr, r);
  else tmem_ld16(taddr, r);
  tmem_ld_wait();
}

template <int CG, int BN>
__global__ void __launch_bounds__(kGemm8Threads, 1)
    fg_gemm8_kernel(const __grid_constant__ CUtensorMap tmX, const __grid_constant__ CUtensorMap tmW,
                    const __grid_constant__ CUtensorMap tmNarrow, const Gemm8Params p) {
  constexpr int kBlock = gemm8_block_bytes(CG, BN), kPer = gemm8_blocks_per_stage(CG, BN), kStage = kPer * kBlock;
  constexpr uint32_t kCols = gemm8_tmem_cols(BN);
  constexpr int kPiece = BN >= 64 ? 32 : 16;       // columns that the epilogue takes at a time
  static_assert(2 * BN <= static_cast<int>(kCols), "tensor memory");
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
  const int splits = CG == 1 ? p.splits : 1;
  const uint32_t in_cluster = CG == 2 || splits > 1 ? cluster_rank() : 0;
  const uint32_t rank = CG == 2 ? in_cluster : 0;                         // which half of a pair's tile
  const int part = CG == 1 ? static_cast<int>(in_cluster) : 0;           // which part of k
  const int cluster = CG * splits;
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
  if (cluster > 1) cluster_sync();
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot_gen;
  const bool gated = p.out.act == kActSiluGate;
  if (warp != 4) {
    griddep_wait();
    griddep_launch_dependents();
  }

  const int tiles = p.tiles_m * p.tiles_n, groups = gridDim.x / cluster, group = blockIdx.x / cluster;
  const int k_blocks = p.out.K / 128, all_stages = (k_blocks + kPer - 1) / kPer;
  const int ks0 = part * all_stages / splits, ks1 = (part + 1) * all_stages / splits;  // this CTA's stages of every tile
  auto first_of = [&](int tn) {  // first weight row of a column of tiles
    if (CG == 2 && tn > p.wide) return p.wide * BN + (tn - p.wide) * p.narrow;
    return tn * BN;
  };
  auto width_of = [&](int tn) { return CG == 2 && tn >= p.wide ? p.narrow : BN; };
  bool dead = false;
  auto report = [&] {
    if (p.out.status != nullptr) atomicExch(p.out.status, kStatusTimeout);
  };

  // Epilogue of a warp's 32 token rows of a tile (TMEM buffer b): scales, bias, activation, residual, kPiece columns at a time; a
  // row's pieces leave as 16-byte stores.  more: followers' sums, [splits - 1][BN][128], or nullptr.
  auto finish = [&](int n0, int bn, int m, bool row, float xs, uint32_t b, const uint32_t* more) {
    const W8A8Params& q = p.out;
    const int width = gated ? q.N >> 1 : q.N;
    if (!__any_sync(0xffffffffu, row)) return;  // a small M: nothing to store for these rows
    const uint32_t tbase = tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + b * BN;
    auto load_piece = [&](int col, uint32_t (&r)[kPiece]) {
      load_sums(tbase + col, r);
      if (CG == 1 && more != nullptr)
        for (int i = 0; i < splits - 1; ++i)
#pragma unroll
          for (int j = 0; j < kPiece; ++j) r[j] += more[(i * BN + col + j) * 128];
    };
    auto emit = [&](int col, const float (&v)[kPiece]) {  // col: column of the output
      if (!row) return;
      __half* dst = q.C + static_cast<size_t>(m) * width + col;
      const __half* res = q.residual ? q.residual + static_cast<size_t>(m) * width + col : nullptr;
#pragma unroll
      for (int h = 0; h < kPiece / 8; ++h) {
        uint4 r = make_uint4(0, 0, 0, 0), o;
        if (res != nullptr) r = *reinterpret_cast<const uint4*>(res + 8 * h);
        const uint32_t rw[4] = {r.x, r.y, r.z, r.w};
        uint32_t* ow = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float2 f = make_float2(v[8 * h + 2 * i], v[8 * h + 2 * i + 1]);
          if (res != nullptr) {
            const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&rw[i]));
            f.x = __fadd_rn(f.x, a.x);
            f.y = __fadd_rn(f.y, a.y);
          }
          const __half2 hv = __floats2half2_rn(f.x, f.y);
          ow[i] = *reinterpret_cast<const uint32_t*>(&hv);
        }
        *reinterpret_cast<uint4*>(dst + 8 * h) = o;
      }
    };
    auto value = [&](uint32_t sum, int col) { return w8a8_value(static_cast<int>(sum), xs, col_scale[col], col_bias[col]); };
    if (gated) {
      // kHalf gate columns, then the matching up columns, per block of 2 kHalf
      constexpr int kHalf = BN < 128 ? BN / 2 : 64;
#pragma unroll 1
      for (int c = 0; c < bn / 2; c += kPiece) {  // column of the tile's output
        const int at = c / kHalf * (2 * kHalf) + c % kHalf;
        uint32_t g[kPiece], u[kPiece];
        load_piece(at, g);
        load_piece(at + kHalf, u);
        if (n0 / 2 + c >= width) continue;
        float v[kPiece];
#pragma unroll
        for (int i = 0; i < kPiece; ++i) v[i] = w8a8_gate(value(g[i], at + i), value(u[i], at + kHalf + i));
        emit(n0 / 2 + c, v);
      }
    } else {
      with_act(q.act, [&](auto tag) {
        constexpr int ACT = decltype(tag)::value;
#pragma unroll 1
        for (int c = 0; c < bn; c += kPiece) {
          uint32_t r[kPiece];
          load_piece(c, r);
          if (n0 + c >= q.N) continue;
          float v[kPiece];
#pragma unroll
          for (int i = 0; i < kPiece; ++i) v[i] = w8a8_act<ACT>(value(r[i], c + i));
          emit(n0 + c, v);
        }
      });
    }
  };

  if (warp == 4) {
    // ------------------------------------ copies ------------------------------------
    const bool one = elect_one();
    const uint64_t pol_x = policy_evict_last();                                              // read again by other tiles
    const uint64_t pol_w = p.tiles_m > 1 ? policy_evict_last() : policy_evict_first();
    const bool two_boxes = BN < 128 && gated;
    const uint32_t full0 = CG == 2 ? map_to_rank(bar_full, 0) : bar_full;  // barriers of the leading CTA
    int m_row = 0, n_row = 0, bn = BN;  // first token row and weight row of this CTA's copies, the tile's width
    auto enter = [&](int t) {
      const int tn = t / p.tiles_m, n0 = first_of(tn);
      bn = width_of(tn);
      m_row = (t - tn * p.tiles_m) * (128 * CG) + 128 * static_cast<int>(rank);
      // with the gate and less than a block of 128: output columns n0 / 2 .., gate rows here, up rows 64 further on
      n_row = two_boxes ? (n0 / 2 / 64) * 128 + n0 / 2 % 64 : n0 + (bn / CG) * static_cast<int>(rank);
    };
    auto load_x = [&](int slot, int ks) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int kb = ks * kPer + i;
        if (kb < k_blocks) {
          const uint32_t dst = smem_base + slot * kStage + i * kBlock;
          if constexpr (CG == 1) tma_load_2d(dst, &tmX, full0 + 8 * slot, kb * 128, m_row, pol_x);
          else tma_load_2d_pair(dst, &tmX, full0 + 8 * slot, kb * 128, m_row, pol_x);
        }
      }
    };
    auto load_w = [&](int slot, int ks) {
      const int blocks = k_blocks - ks * kPer < kPer ? k_blocks - ks * kPer : kPer;
      if (rank == 0) mbar_arrive_expect_tx(bar_full + 8 * slot, CG * blocks * (kBlock - (128 - p.x_rows + (BN - bn) / CG) * 128));
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int kb = ks * kPer + i;
        if (kb < k_blocks) {
          const uint32_t dst = smem_base + slot * kStage + i * kBlock + 16384;
          if constexpr (CG == 1) {
            tma_load_2d(dst, &tmW, full0 + 8 * slot, kb * 128, n_row, pol_w);
            if (two_boxes) tma_load_2d(dst + BN / 2 * 128, &tmW, full0 + 8 * slot, kb * 128, n_row + 64, pol_w);
          } else {
            tma_load_2d_pair(dst, bn == BN ? &tmW : &tmNarrow, full0 + 8 * slot, kb * 128, n_row, pol_w);
          }
        }
      }
    };
    int s = 0, filled = 0;
    uint32_t ph = 1;  // the slots start out empty
    const int ahead = ks1 - ks0 < S ? ks1 - ks0 : S;  // of the first tile (there is one: no more groups than tiles)
    enter(group);
    if (one) {
      tma_prefetch_desc(&tmX);
      tma_prefetch_desc(&tmW);
      for (int i = 0; i < ahead; ++i) load_w(i, ks0 + i);
    }
    __syncwarp();
    griddep_wait();
    for (int t = group; t < tiles && !dead; t += groups) {
      if (t != group) enter(t);
      for (int ks = ks0; ks < ks1; ++ks) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar_empty + 8 * s, ph, kWaitBudgetNs))) {
          dead = true;
          break;
        }
        if (one) {
          if (filled >= ahead) load_w(s, ks);
          load_x(s, ks);
        }
        __syncwarp();
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
    if (dead && lane == 0) report();
    __syncwarp();
  } else if (warp == 5) {
    // ------------------------------------ MMA ------------------------------------
    if (rank == 0) {
      const bool one = elect_one();
      constexpr uint64_t desc = umma_smem_desc(0, 1, 64);
      int s = 0, n = 0;
      uint32_t ph = 0;
      for (int t = group; t < tiles && !dead; t += groups, ++n) {
        const uint32_t b = n & 1, use = n >> 1;
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar_acc_empty + 8 * b, (use & 1) ^ 1, kWaitBudgetNs))) {
          dead = true;
          break;
        }
        tc_fence_after_sync();
        const uint32_t acc = tmem_base + b * BN, idesc = umma_idesc_i8(128 * CG, width_of(t / p.tiles_m));
        for (int ks = ks0; ks < ks1; ++ks) {
          if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar_full + 8 * s, ph, kWaitBudgetNs))) {
            dead = true;
            break;
          }
          if (one) {
            const uint64_t at = desc | (((smem_base + s * kStage) >> 4) & 0x3FFFu);
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
              if (i == 0 || ks * kPer + i < k_blocks) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  gemm8_mma<CG>(acc, at + (i * kBlock / 16 + 2 * k), at + ((i * kBlock + 16384) / 16 + 2 * k), idesc,
                                ks != ks0 || i != 0 || k != 0);
              }
            }
            gemm8_commit<CG>(bar_empty + 8 * s);
          }
          __syncwarp();
          if (++s == S) {
            s = 0;
            ph ^= 1;
          }
        }
        if (!dead && one) gemm8_commit<CG>(bar_acc_full + 8 * b);
        __syncwarp();
      }
      if (dead && lane == 0) report();
    }
    __syncwarp();
  } else {
    // ------------------------------------ epilogue ------------------------------------
    const W8A8Params& q = p.out;
    int n = 0;
    for (int t = group; t < tiles; t += groups, ++n) {
      const int m = (t % p.tiles_m) * (128 * CG) + 128 * rank + 32 * warp + lane, n0 = first_of(t / p.tiles_m);
      const int bn = width_of(t / p.tiles_m);
      const uint32_t b = n & 1, use = n >> 1;
      const bool row = m < q.M;
      const float xs = row ? x_scale(q, m) : 0.f;
      named_bar_sync(1, 128);  // the previous tile's column values have been read
      for (int j = threadIdx.x; j < bn; j += 128) {
        int w = n0 + j;  // weight row of column j
        if (BN < 128 && gated) w = gate_row(n0 / 2 + j % (BN / 2)) + (j < BN / 2 ? 0 : 64);
        col_scale[j] = w < q.N && q.w_scales != nullptr ? __half2float(q.w_scales[w]) : 1.f;
        col_bias[j] = w < q.N && q.bias != nullptr ? __half2float(q.bias[w]) : 0.f;
      }
      named_bar_sync(1, 128);
      if (!dead && !__all_sync(0xffffffffu, mbar_wait_bounded(bar_acc_full + 8 * b, use & 1, 2 * kWaitBudgetNs))) {
        dead = true;
        if (lane == 0) report();
      }
      if (CG == 1 && splits > 1) break;  // the cluster's one tile: finished below, together
      if (dead) continue;
      tc_fence_after_sync();
      finish(n0, bn, m, row, xs, b, nullptr);
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if constexpr (CG == 1) mbar_arrive(bar_acc_empty + 8 * b);
        else mbar_arrive_cluster(map_to_rank(bar_acc_empty + 8 * b, 0));
      }
    }
  }

  if constexpr (CG == 1) {
    if (splits > 1) {
      // Partial sums meet in the leader's ring: [follower][column][128 rows].  First barrier: the leader's MMAs have read
      // everything that its copies brought.  Second: the followers' sums are there.
      tc_fence_before_sync();
      __syncwarp();
      cluster_sync();
      tc_fence_after_sync();
      const uint32_t sums = smem_base;
      if (warp < 4 && part > 0) {
        const uint32_t to = map_to_rank(sums, 0) + (((part - 1) * BN) * 128 + 32 * warp + lane) * 4;
#pragma unroll 1
        for (int c = 0; c < BN; c += kPiece) {
          uint32_t r[kPiece];
          load_sums(tmem_base + (static_cast<uint32_t>(warp * 32) << 16) + c, r);
#pragma unroll
          for (int j = 0; j < kPiece; ++j) st_cluster(to + (c + j) * 512, r[j]);
        }
      }
      __syncwarp();
      cluster_sync();
      if (warp < 4 && part == 0) {
        const int m = (group % p.tiles_m) * 128 + 32 * warp + lane;
        const bool row = m < p.out.M;
        tc_fence_after_sync();
        finish(group / p.tiles_m * BN, BN, m, row && !dead, row ? x_scale(p.out, m) : 0.f, 0, reinterpret_cast<const uint32_t*>(smem_gen) + 32 * warp + lane);
      }
    }
  }

  // ---- teardown: every MMA has completed (the epilogues have seen them) and the pair leaves together ----
  tc_fence_before_sync();
  __syncthreads();
  if (cluster > 1) cluster_sync();
  if (warp == 5) {
    tc_fence_after_sync();
    if constexpr (CG == 1) {
      tmem_dealloc(tmem_base, kCols);
    } else {
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kCols) : "memory");
    }
  }
  if (CG == 2) cluster_sync();
}

}  // namespace fg

// Attention over the paged 4-bit key/value cache (fg_kv_attention_int4); layout in fg_kv4.cuh.
//
//   s_t = softmax_scale * q . k_t     k_t = lowk_t + sk_t * ck_t     (ck_t: the codes, integers 0..15)
//       = softmax_scale * (sk_t * (q . ck_t) + lowk_t * sum(q))
//   o   = sum_t p_t v_t / sum_t p_t   = (sum_t (p_t sv_t) cv_t + sum_t p_t lowv_t) / sum_t p_t,   p_t = exp(s_t - m)
//
// so the matrix products run on bare codes and every scale is applied to a score or a weight, in 32 bits.
//
// The bytes of the cache are the floor: D + 8 of them per row and head, against 16 D bit operations' worth of
// unpacking.  What this kernel does about the second:
//   - A code's four bits, masked in place, ARE an fp16 number: bits 0-3 of a half are the subnormal code * 2^-24, bits 4-7
//     code * 2^-20.  The tensor core multiplies subnormals exactly, so unpacking is one AND per two codes (and one shift
//     per eight); the power of two comes out with the scale.  Low and high nibbles go to separate accumulators (keys) or
//     separate accumulator rows (values).
//   - Codes are the 16-row operand of mma.sync.m16n8k16 and the queries that share a key/value head its 8 columns, so a
//     group of up to eight query heads costs what one does.  S^T = K Q^T leaves P^T in the layout from which
//     movmatrix makes the second product's operand; nothing goes through shared memory but the cache itself.
//     (tcgen05.mma takes its operands from shared memory: the codes would have to be written back there as fp16, four
//     times the bytes that came in.)
//   - The softmax's running maximum moves only when a score exceeds it by more than 2^8 (a warp vote per 16 rows instead
//     of a reduction); weights then stay below 2^8 and exact sums are unchanged, since every term uses the same m.
//     The maximum is taken over log2(p_t sv_t), the weight that is rounded to fp16: its relative error is 2^-11 whatever
//     the scale of the values.
//
// Each warp streams its own blocks of 16 rows through its own ring (bulk copies by lane 0, one mbarrier per slot), so no
// warp waits for another inside a segment.  The rows of all (sequence, head, query tile) items form one list of 64-row
// units that is dealt out evenly to the CTAs whatever the lengths; an item that several CTAs share is joined by the last of
// them to finish, in CTA order (deterministic), from partial sums in the workspace.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/fastgate_b200.h"
#include "fg_host.h"
#include "fg_kv4.cuh"

namespace fg {
namespace {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kAttnStages = 4;             // ring slots of a warp
constexpr int kUnitRows = kAttnWarps * kKvBlock;
constexpr int kAttnMaxGrid = 1024;
constexpr int kAttnMinUnits = 4;           // units a CTA gets at least, so that joining stays cheap
constexpr float kLazyMax = 8.f;            // log2 of how far a weight may exceed the running maximum
constexpr unsigned long long kAttnWaitNs = 2000000000ull;
constexpr int kStatusAttnTimeout = 6;      // FG_ERR_TIMEOUT

// Workspace: [0,256) header, kAttnMaxGrid tickets (zero between launches), then two partials per CTA.
constexpr size_t kAttnTicketsOffset = 256;
constexpr size_t kAttnPartialsOffset = kAttnTicketsOffset + kAttnMaxGrid * 4;
constexpr int kAttnMaxCols = 16;
__host__ __device__ constexpr int partial_floats(int d, int cols) { return cols * (d + 4); }  // [cols][d] sums, [cols] maxima, [cols] norms, padding

struct AttnParams {
  const __half* q;        // [tokens, q_heads, D], token stride ldq
  long long ldq;
  __half* out;            // the same with ldo
  long long ldo;
  int q_heads, group;     // group = q_heads / kv.heads
  KvPages kv;
  const int* table;       // [batch, table_width], row stride ldt
  long long ldt;
  int table_width;
  const int* lens;        // [batch]
  const int* q_starts;    // [batch + 1], or nullptr: one query token per sequence
  int batch;
  long long tokens;       // rows of q
  float scale_log2;       // softmax scale * log2(e)
  unsigned int* tickets;
  float* partials;
  int* status;            // may be nullptr
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
               "r"(bytes), "r"(bar)
               : "memory");
}
__device__ __forceinline__ uint32_t movmatrix_trans(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float lg2(float x) {
  float r;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <int BYTES>
__device__ __forceinline__ void lds_words(uint32_t addr, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES == 16) lds_v4(addr, w[0], w[1], w[2], w[3]);
  else if constexpr (BYTES == 8) lds_v2(addr, w[0], w[1]);
  else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[0]) : "r"(addr));
}
__device__ __forceinline__ float2 lds_half2(uint32_t addr) {
  uint32_t w;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(addr));
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

// What of the work list belongs to sequence b.
struct Sequence {
  int len;       // rows that its queries may see at most
  int q0, nq;    // its query tokens
  int tiles;     // query tiles per key/value head
  int units;     // units per item, at least one
  __device__ long long total(int kv_heads) const { return static_cast<long long>(tiles) * kv_heads * units; }
};

template <int COLS>
__device__ __forceinline__ Sequence sequence(const AttnParams& p, int b, bool report) {
  Sequence s;
  bool bad = false;
  s.len = p.lens[b];
  const long long room = static_cast<long long>(p.table_width) * p.kv.page_size;
  if (s.len < 0 || s.len > room) {
    bad = true;
    s.len = 0;  // its outputs become zeros
  }
  s.q0 = p.q_starts ? p.q_starts[b] : b;
  s.nq = p.q_starts ? p.q_starts[b + 1] - s.q0 : 1;
  if (s.q0 < 0 || s.nq < 0 || s.q0 + static_cast<long long>(s.nq) > p.tokens) {
    bad = true;
    s.q0 = s.nq = 0;  // nothing is read or written for it
  }
  if (bad && report && p.status != nullptr) atomicExch(p.status, kStatusIndex);
  s.tiles = static_cast<int>((static_cast<long long>(s.nq) * p.group + COLS - 1) / COLS);
  s.units = s.len > 0 ? (s.len + kUnitRows - 1) / kUnitRows : 1;
  return s;
}

template <int D, int NQ>
__global__ void __launch_bounds__(kAttnThreads, NQ == 1 ? 4 : 3) fg_kv_attention_kernel(const AttnParams p) {
  constexpr int COLS = 8 * NQ;          // query columns of an item
  constexpr int KW = D / 32;            // 32-bit words of a key row per lane
  constexpr int VW = D / 64;            // 32-bit words of a value row per lane
  constexpr int MT = D / 16;            // 16-channel accumulator tiles
  constexpr int SB = kv_block_bytes(D);
  constexpr int kRing = kAttnStages * SB;
  constexpr int kWarpBytes = (kRing > COLS * (D + 4) * 4 ? kRing : COLS * (D + 4) * 4);  // a warp's sums are parked in its ring
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kAttnWarps * kAttnStages];
  __shared__ long long scan[kAttnWarps + 1];
  __shared__ long long start_before;
  __shared__ int start_b;
  __shared__ unsigned int ticket;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  uint8_t* my_smem = smem + warp * kWarpBytes;
  const uint32_t ring = smem_u32(my_smem);
  const uint32_t bar = smem_u32(bars + warp * kAttnStages);
  if (lane < kAttnStages) mbar_init(bar + 8 * lane, 1);
  fence_mbar_init();
  fence_proxy_async();
  griddep_launch_dependents();
  griddep_wait();

  // ---- this CTA's share [ub, ue) of the work list ----
  const int per = (p.batch + kAttnThreads - 1) / kAttnThreads;
  const int b_lo = min(p.batch, tid * per), b_hi = min(p.batch, b_lo + per);
  long long mine = 0;
  for (int b = b_lo; b < b_hi; ++b) mine += sequence<COLS>(p, b, blockIdx.x == 0).total(p.kv.heads);
  long long incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const long long v = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += v;
  }
  if (lane == 31) scan[warp] = incl;
  __syncthreads();
  long long before = incl - mine, total = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
  }
  const long long want = (total + kAttnMinUnits - 1) / kAttnMinUnits;
  const long long G = want < gridDim.x ? want : gridDim.x;
  if (static_cast<long long>(blockIdx.x) >= G) return;
  const long long cta = blockIdx.x;
  const long long ub = cta * total / G, ue = (cta + 1) * total / G;
  if (mine > 0 && ub >= before && ub < before + mine) {
    int b = b_lo;
    for (;; ++b) {
      const long long t = sequence<COLS>(p, b, false).total(p.kv.heads);
      if (ub < before + t) break;
      before += t;
    }
    start_b = b;
    start_before = before;
  }
  __syncthreads();
  int b = start_b;
  long long b_before = start_before;  // units before sequence b
  Sequence sq = sequence<COLS>(p, b, false);

  uint32_t phase = 0;  // one bit per ring slot
  bool dead = false;
  long long u = ub;
  while (u < ue) {
    while (u >= b_before + sq.total(p.kv.heads)) {
      b_before += sq.total(p.kv.heads);
      sq = sequence<COLS>(p, ++b, false);
    }
    // ---- the segment: units [seg0, seg0 + seg_len) of item (b, head, tile) ----
    const long long item = (u - b_before) / sq.units;
    const long long item_u0 = b_before + item * sq.units;
    const int seg0 = static_cast<int>(u - item_u0);
    const int seg_len = static_cast<int>(min(static_cast<long long>(sq.units - seg0), ue - u));
    const int head = static_cast<int>(item / sq.tiles), tile = static_cast<int>(item - static_cast<long long>(head) * sq.tiles);
    const int cols = min(COLS, sq.nq * p.group - tile * COLS);

    // ---- queries into fragments, their sums, the last row that each column sees ----
    uint32_t qf[NQ][KW][4];
    float qs[NQ][2];
    int limit[NQ][2], min_limit = 0x7fffffff;
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int col = n * 8 + g;
      float sum = 0.f;
      uint4 raw[KW];
#pragma unroll
      for (int w = 0; w < KW; ++w) raw[w] = make_uint4(0, 0, 0, 0);
      if (col < cols) {
        const int flat = tile * COLS + col;
        const __half* src = p.q + static_cast<long long>(sq.q0 + flat / p.group) * p.ldq +
                            static_cast<long long>(head * p.group + flat % p.group) * D + c * (8 * KW);
#pragma unroll
        for (int w = 0; w < KW; ++w) raw[w] = *reinterpret_cast<const uint4*>(src + 8 * w);
      }
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        // channels (0,4), (2,6) meet the low nibbles' pairs, (1,5), (3,7) the high ones'
        qf[n][w][0] = prmt(raw[w].x, raw[w].z, 0x5410);
        qf[n][w][1] = prmt(raw[w].y, raw[w].w, 0x5410);
        qf[n][w][2] = prmt(raw[w].x, raw[w].z, 0x7632);
        qf[n][w][3] = prmt(raw[w].y, raw[w].w, 0x7632);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[n][w][i]));
          sum += f.x + f.y;
        }
      }
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int my = n * 8 + 2 * c + i;
        qs[n][i] = __shfl_sync(0xffffffffu, sum, (2 * c + i) * 4) * p.scale_log2;
        limit[n][i] = my < cols ? sq.len - sq.nq + (tile * COLS + my) / p.group : sq.len - 1;
      }
    }
    min_limit = min(sq.len - 1, sq.len - sq.nq + (tile * COLS) / p.group);  // column 0 sees least

    float oacc[NQ][MT][4], mref[NQ][2], lsum[NQ][2], zsum[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mref[n][i] = -INFINITY;
        lsum[n][i] = zsum[n][i] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) oacc[n][t][i] = 0.f;
    }

    // ---- this warp's blocks: seg0 * 4 + warp, + 4, ... ----
    const int blocks_per_page = p.kv.page_size / kKvBlock;
    const int all_blocks = (sq.len + kKvBlock - 1) / kKvBlock;
    const int blk0 = seg0 * kAttnWarps + warp;
    const int blk_end = min(all_blocks, (seg0 + seg_len) * kAttnWarps);
    const int n_blk = blk_end > blk0 && !dead ? (blk_end - blk0 + kAttnWarps - 1) / kAttnWarps : 0;
    const int* trow = p.table + static_cast<long long>(b) * p.ldt;
    // lane i holds the page of this warp's block 32 k + i; `pages_next` the 32 after those
    auto fetch_pages = [&](int k) {
      const int blk = blk0 + (32 * k + lane) * kAttnWarps;
      int page = -1;
      if (blk < blk_end) {
        page = __ldg(trow + blk / blocks_per_page);
        if (page < 0 || page >= p.kv.pages) {
          if (p.status != nullptr) atomicExch(p.status, kStatusIndex);
          page = -1;
        }
      }
      return page;
    };
    int pages_now = fetch_pages(0), pages_next = fetch_pages(1);
    uint32_t skipped = 0;  // bit s: the block in slot s has no page and is left out
    auto issue = [&](int j) {  // whole warp; block j of this warp into slot j % stages
      if (j >= n_blk) return;
      const int page = __shfl_sync(0xffffffffu, (j & 32) ? pages_next : pages_now, j & 31);
      const int s = j % kAttnStages;
      if (page < 0) {
        skipped |= 1u << s;
        return;
      }
      skipped &= ~(1u << s);
      if (lane == 0) {
        const int blk = blk0 + j * kAttnWarps;
        mbar_arrive_expect_tx(bar + 8 * s, SB);
        bulk_load(ring + s * SB, kv_block_ptr(p.kv, D, page, head, blk % blocks_per_page), SB, bar + 8 * s);
      }
    };
    for (int j = 0; j < kAttnStages; ++j) issue(j);

    // key row g of a 16-row operand is row kmap(g) of the block's half: rows 2i and 2i + 1 of an operand then lie in
    // different halves of the shared-memory banks
    const int ka = (g & 1) ? 4 + ((g >> 1) ^ 1) : g >> 1;
    const int v0 = c, v1 = 4 + (c ^ 1);
    for (int j = 0; j < n_blk && !dead; ++j) {
      const int s = j % kAttnStages;
      const bool skip = (skipped >> s) & 1u;
      if (!skip) {
        if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar + 8 * s, (phase >> s) & 1u, kAttnWaitNs))) {
          dead = true;
          if (lane == 0 && p.status != nullptr) atomicExch(p.status, kStatusAttnTimeout);
          break;
        }
        phase ^= 1u << s;
        const uint32_t base = ring + s * SB;
        const int row0 = (blk0 + j * kAttnWarps) * kKvBlock;

        // S^T = K Q^T on the codes
        uint32_t wa[KW], wb[KW];
        lds_words<4 * KW>(base + kv_codes_offset(D, 0, ka) + c * (4 * KW), wa);
        lds_words<4 * KW>(base + kv_codes_offset(D, 0, ka + 8) + c * (4 * KW), wb);
        float slo[NQ][4], shi[NQ][4];
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) slo[n][i] = shi[n][i] = 0.f;
#pragma unroll
        for (int w = 0; w < KW; ++w) {
          const uint32_t xa = wa[w] >> 8, xb = wb[w] >> 8;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            mma_16816(slo[n], wa[w] & 0x000F000Fu, wb[w] & 0x000F000Fu, xa & 0x000F000Fu, xb & 0x000F000Fu, qf[n][w][0], qf[n][w][1]);
            mma_16816(shi[n], wa[w] & 0x00F000F0u, wb[w] & 0x00F000F0u, xa & 0x00F000F0u, xb & 0x00F000F0u, qf[n][w][2], qf[n][w][3]);
          }
        }

        float2 kp[2], vp[2];  // (scale, low) of rows ka and ka + 8
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          kp[i] = lds_half2(base + kv_params_offset(D, 0, ka + 8 * i));
          vp[i] = lds_half2(base + kv_params_offset(D, 1, ka + 8 * i));
        }
        const bool masked = row0 + kKvBlock - 1 > min_limit;
        float sk[2], lv[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          sk[i] = kp[i].x * (p.scale_log2 * 16777216.f);
          lv[i] = lg2(fmaxf(vp[i].x, 5.9604644775390625e-8f));
        }
        float s2[NQ][4];  // log2 of the weights before the values' scales
        bool up = false;
#pragma unroll
        for (int n = 0; n < NQ; ++n)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i >> 1, q = i & 1;
            s2[n][i] = fmaf(fmaf(shi[n][i], 0.0625f, slo[n][i]), sk[r], kp[r].y * qs[n][q]);
            if (masked && row0 + ka + 8 * r > limit[n][q]) s2[n][i] = -INFINITY;
            up |= s2[n][i] + lv[r] > mref[n][q] + kLazyMax;
          }
        if (__any_sync(0xffffffffu, up)) {
          // a new maximum: the largest of the old one and this block's, and everything so far brought to it
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float m = fmaxf(s2[n][q] + lv[0], s2[n][2 + q] + lv[1]);
#pragma unroll
              for (int off = 4; off <= 16; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
              m = fmaxf(m, mref[n][q]);
              const float f = m == -INFINITY ? 1.f : ex2(mref[n][q] - m);
              mref[n][q] = m;
              lsum[n][q] *= f;
              zsum[n][q] *= f;
#pragma unroll
              for (int t = 0; t < MT; ++t) {
                oacc[n][t][q] *= f;
                oacc[n][t][2 + q] *= f;
              }
            }
        }
        uint32_t pb[NQ][2];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float wgt[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i >> 1, q = i & 1;
            const float m = mref[n][q] == -INFINITY ? 0.f : mref[n][q];
            const float e = ex2(s2[n][i] - m);
            lsum[n][q] += e;
            if (masked && s2[n][i] == -INFINITY) {
              wgt[i] = 0.f;  // whatever the row's parameters hold
            } else {
              zsum[n][q] = fmaf(e, vp[r].y, zsum[n][q]);
              wgt[i] = e * vp[r].x;
            }
          }
          const __half2 h0 = __floats2half2_rn(wgt[0], wgt[1]), h1 = __floats2half2_rn(wgt[2], wgt[3]);
          pb[n][0] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&h0));
          pb[n][1] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&h1));
        }

        // O^T += V^T P^T on the codes: lane g owns channels 8 VW g.., operand columns are rows (v0, v1) and (v0, v1) + 8
        uint32_t r0[VW], r1[VW], r2[VW], r3[VW];
        lds_words<4 * VW>(base + kv_codes_offset(D, 1, v0) + g * (4 * VW), r0);
        lds_words<4 * VW>(base + kv_codes_offset(D, 1, v1) + g * (4 * VW), r1);
        lds_words<4 * VW>(base + kv_codes_offset(D, 1, v0 + 8) + g * (4 * VW), r2);
        lds_words<4 * VW>(base + kv_codes_offset(D, 1, v1 + 8) + g * (4 * VW), r3);
#pragma unroll
        for (int w = 0; w < VW; ++w)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t xa = prmt(r0[w], r1[w], hf ? 0x7632 : 0x5410), xb = prmt(r2[w], r3[w], hf ? 0x7632 : 0x5410);
#pragma unroll
            for (int by = 0; by < 2; ++by) {
#pragma unroll
              for (int n = 0; n < NQ; ++n)
                mma_16816(oacc[n][w * 4 + hf * 2 + by], xa & 0x000F000Fu, xa & 0x00F000F0u, xb & 0x000F000Fu, xb & 0x00F000F0u, pb[n][0], pb[n][1]);
              xa >>= 8;
              xb >>= 8;
            }
          }
      }
      __syncwarp();  // every lane has read the slot
      if (((j + kAttnStages) & 31) == 0) {
        // the block to be issued next is the first of a new set of 32 page numbers
        const int k = (j + kAttnStages) >> 5;
        if (k & 1) pages_now = fetch_pages(k + 1);
        else pages_next = fetch_pages(k + 1);
      }
      issue(j + kAttnStages);
    }

    // ---- the four warps' sums meet in shared memory (each parks its own in its ring, which is empty now) ----
    float* park = reinterpret_cast<float*>(my_smem);
    __syncwarp();
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float l = lsum[n][q], z = zsum[n][q];
#pragma unroll
        for (int off = 4; off <= 16; off <<= 1) {
          l += __shfl_xor_sync(0xffffffffu, l, off);
          z += __shfl_xor_sync(0xffffffffu, z, off);
        }
        const int col = n * 8 + 2 * c + q;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          // accumulator row g holds the even channel (low nibble), row g + 8 the odd one
          const float2 v = make_float2(fmaf(oacc[n][t][q], 16777216.f, z), fmaf(oacc[n][t][2 + q], 1048576.f, z));
          *reinterpret_cast<float2*>(park + col * D + g * (8 * VW) + 2 * t) = v;
        }
        if (g == 0) {
          park[COLS * D + col] = mref[n][q];
          park[COLS * D + COLS + col] = dead ? NAN : l;
        }
      }
    __syncthreads();
    const bool whole = seg_len == sq.units;
    float* part = p.partials + (cta * 2 + (u == ub ? 0 : 1)) * partial_floats(D, COLS);
    // thread: four channels of every (kAttnThreads / (D / 4))th column
    constexpr int TPC = D / 4;
    const int d4 = (tid % TPC) * 4;
    auto write_out = [&](int col, float4 v, float l) {
      if (col >= cols) return;
      const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing gives zeros
      const int flat = tile * COLS + col;
      const __half2 h0 = __floats2half2_rn(v.x * inv, v.y * inv), h1 = __floats2half2_rn(v.z * inv, v.w * inv);
      *reinterpret_cast<uint2*>(p.out + static_cast<long long>(sq.q0 + flat / p.group) * p.ldo +
                                static_cast<long long>(head * p.group + flat % p.group) * D + d4) =
          make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
    };
#pragma unroll 1
    for (int col = tid / TPC; col < COLS; col += kAttnThreads / TPC) {
      float m = -INFINITY, l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      float mw[kAttnWarps];
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        mw[w] = reinterpret_cast<const float*>(smem + w * kWarpBytes)[COLS * D + col];
        m = fmaxf(m, mw[w]);
      }
#pragma unroll
      for (int w = 0; w < kAttnWarps; ++w) {
        const float* src = reinterpret_cast<const float*>(smem + w * kWarpBytes);
        const float f = m == -INFINITY ? 1.f : ex2(mw[w] - m);
        const float4 a = *reinterpret_cast<const float4*>(src + col * D + d4);
        l = fmaf(f, src[COLS * D + COLS + col], l);
        v.x = fmaf(f, a.x, v.x);
        v.y = fmaf(f, a.y, v.y);
        v.z = fmaf(f, a.z, v.z);
        v.w = fmaf(f, a.w, v.w);
      }
      if (whole) {
        write_out(col, v, l);
      } else {
        __stcg(reinterpret_cast<float4*>(part + col * D + d4), v);
        if (d4 == 0) {
          __stcg(part + COLS * D + col, m);
          __stcg(part + COLS * D + COLS + col, l);
        }
      }
    }
    if (!whole) {
      // ---- an item of several CTAs: the last of them to get here joins the partials in CTA order ----
      const long long last_u = item_u0 + sq.units - 1;
      auto cta_of = [&](long long unit) {  // the CTA whose share holds `unit`
        long long x = unit * G / total;
        while (x + 1 < G && (x + 1) * total / G <= unit) ++x;
        while (x > 0 && x * total / G > unit) --x;
        return x;
      };
      const long long c_first = cta_of(item_u0), c_last = cta_of(last_u);
      __syncthreads();
      if (tid == 0) {
        __threadfence();
        const unsigned int t = atomicAdd(p.tickets + c_first, 1u);
        fence_acq_rel_gpu();
        ticket = t;
      }
      __syncthreads();
      if (ticket == static_cast<unsigned int>(c_last - c_first)) {
        // only the first contributor can have begun its share in an earlier item
        const int first_slot = c_first * total / G < item_u0 ? 1 : 0;
        auto part_of = [&](long long x) {
          const int slot = x == c_first ? first_slot : 0;
          return p.partials + (x * 2 + slot) * partial_floats(D, COLS);
        };
#pragma unroll 1
        for (int col = tid / TPC; col < cols; col += kAttnThreads / TPC) {
          float m = -INFINITY, l = 0.f;
          float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
          for (long long x = c_first; x <= c_last; ++x) m = fmaxf(m, __ldcg(part_of(x) + COLS * D + col));
#pragma unroll 4
          for (long long x = c_first; x <= c_last; ++x) {
            const float* src = part_of(x);
            const float mx = __ldcg(src + COLS * D + col);
            const float f = m == -INFINITY ? 1.f : ex2(mx - m);
            const float4 a = __ldcg(reinterpret_cast<const float4*>(src + col * D + d4));
            l = fmaf(f, __ldcg(src + COLS * D + COLS + col), l);
            v.x = fmaf(f, a.x, v.x);
            v.y = fmaf(f, a.y, v.y);
            v.z = fmaf(f, a.z, v.z);
            v.w = fmaf(f, a.w, v.w);
          }
          write_out(col, v, l);
        }
        if (tid == 0) p.tickets[c_first] = 0;  // ready for the next launch
      }
    }
    __syncthreads();          // the parked sums have been read
    fence_proxy_async();      // ... and the copies of the next segment may overwrite them
    u += seg_len;
  }
  if (dead) {
    // a wait gave up: copies that are still in flight get time to land before the shared memory goes away
    for (int s = 0; s < kAttnStages; ++s) mbar_wait_bounded(bar + 8 * s, (phase >> s) & 1u, kAttnWaitNs / 10);
  }
}

}  // namespace
}  // namespace fg

extern "C" size_t fg_kv_attention_workspace_bytes(void) {
  return fg::kAttnPartialsOffset + static_cast<size_t>(fg::kAttnMaxGrid) * 2 * fg::partial_floats(128, fg::kAttnMaxCols) * sizeof(float);
}

extern "C" int fg_kv_attention_workspace_init(void* ws, size_t ws_bytes, fg_stream_t stream) {
  if (ws == nullptr || !fg::host::aligned(ws, 256) || ws_bytes < fg_kv_attention_workspace_bytes()) return FG_ERR_WORKSPACE;
  const cudaError_t e = cudaMemsetAsync(ws, 0, fg::kAttnPartialsOffset, reinterpret_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? FG_OK : (fg::host::launched(e), FG_ERR_CUDA);
}

extern "C" int fg_kv_attention_int4(const void* q, long long ldq, void* out, long long ldo, long long tokens, int q_heads, int kv_heads,
                                    int d, const void* pages, long long num_pages, int page_size, const int* block_table,
                                    long long ldt, int table_width, const int* seq_lens, const int* q_starts, int batch, float scale,
                                    int* status_dev, void* ws, size_t ws_bytes, fg_stream_t stream) {
  using namespace fg;
  if (q == nullptr || out == nullptr || pages == nullptr || block_table == nullptr || seq_lens == nullptr) return FG_ERR_NULL;
  if ((d != 64 && d != 128) || num_pages < 1 || kv_heads < 1 || page_size < kKvBlock || (page_size % kKvBlock) != 0) return FG_ERR_SHAPE;
  if (q_heads < 1 || (q_heads % kv_heads) != 0 || batch < 1 || tokens < 1 || table_width < 1 || ldt < table_width) return FG_ERR_SHAPE;
  if (q_starts == nullptr && tokens != batch) return FG_ERR_SHAPE;
  if (tokens > 0x7fffffffLL / q_heads || static_cast<long long>(table_width) * page_size > 0x7fffffffLL - 2 * kUnitRows) return FG_ERR_SHAPE;
  if (ldq < static_cast<long long>(q_heads) * d || ldo < static_cast<long long>(q_heads) * d || (ldq % 8) != 0 || (ldo % 8) != 0) return FG_ERR_SHAPE;
  if (!(scale > 0.f) || !(scale <= 3.0e38f)) return FG_ERR_SHAPE;
  if (!host::aligned(q, 16) || !host::aligned(out, 16) || !host::aligned(pages, 16) || !host::aligned(block_table, 4) ||
      !host::aligned(seq_lens, 4) || !host::aligned(q_starts, 4) || !host::aligned(status_dev, 4))
    return FG_ERR_ALIGN;
  if (ws == nullptr || !host::aligned(ws, 256) || ws_bytes < fg_kv_attention_workspace_bytes()) return FG_ERR_WORKSPACE;
  host::Device dev;
  int st = host::current_device(&dev);
  if (st != FG_OK) return st;
  AttnParams p = {};
  p.q = static_cast<const __half*>(q);
  p.ldq = ldq;
  p.out = static_cast<__half*>(out);
  p.ldo = ldo;
  p.q_heads = q_heads;
  p.group = q_heads / kv_heads;
  p.kv = {const_cast<uint8_t*>(static_cast<const uint8_t*>(pages)), num_pages, kv_heads, page_size};
  p.table = block_table;
  p.ldt = ldt;
  p.table_width = table_width;
  p.lens = seq_lens;
  p.q_starts = q_starts;
  p.batch = batch;
  p.tokens = tokens;
  p.scale_log2 = scale * 1.4426950408889634f;
  p.tickets = reinterpret_cast<unsigned int*>(static_cast<uint8_t*>(ws) + kAttnTicketsOffset);
  p.partials = reinterpret_cast<float*>(static_cast<uint8_t*>(ws) + kAttnPartialsOffset);
  p.status = status_dev;
  // One column tile of eight where a sequence's queries of one key/value head fit it, else sixteen.
  const long long per_seq = (tokens + batch - 1) / batch * p.group;
  const bool wide = per_seq > 8;
  void (*kern)(const AttnParams) = d == 128 ? (wide ? fg_kv_attention_kernel<128, 2> : fg_kv_attention_kernel<128, 1>)
                                            : (wide ? fg_kv_attention_kernel<64, 2> : fg_kv_attention_kernel<64, 1>);
  const int cols = wide ? 16 : 8;
  const int ring = kAttnStages * kv_block_bytes(d), park = cols * (d + 4) * 4;
  const int smem = kAttnWarps * (ring > park ? ring : park);
  if ((st = host::opt_in_smem(reinterpret_cast<const void*>(kern), smem)) != FG_OK) return st;
  const int grid = min(kAttnMaxGrid, dev.sm_count * (wide ? 3 : 4));
  return host::launch(kern, dim3(grid), dim3(kAttnThreads), smem, reinterpret_cast<cudaStream_t>(stream), true, p);
}

// Attention over the paged 4-bit key/value cache (fg_kv_attention_int4); layout in fg_kv4.cuh.
//
//   s_t = softmax_scale * q . k_t     k_t = lowk_t + sk_t * ck_t     (ck_t: the codes, integers 0..15)
//       = softmax_scale * (sk_t * (q . ck_t) + lowk_t * sum(q))
//   o   = sum_t p_t v_t / sum_t p_t   = (sum_t (p_t sv_t) cv_t + sum_t p_t lowv_t) / sum_t p_t,   p_t = exp(s_t - m)
//
// so the matrix products run on bare codes and every scale is applied to a score or a weight, in 32 bits.
//
// The bytes of the cache are the floor: D + 8 of them per row and head, against 16 D bit operations' worth of
// unpacking.  Measured on B200 (64 / 8 heads of 128 channels): 64 sequences of up to 8000 rows 93.6 us, 4.2 TB/s.  Of the 500
// cycles that a scheduler spends on 16 rows the tensor pipe is busy 192 and the integer pipe 220, and the two hardly overlap: more
// warps do not help (twelve an SM 97 us; ten, three of them on one scheduler, 110).  One sequence of 5000 rows (32 / 8 heads)
// 10.9 us: lengths, table, rows, partial sums, ticket, join, each a trip to L2 or memory.
// What this kernel does about the unpacking:
//   - A code's four bits, masked in place, ARE an fp16 number: bits 0-3 of a half are the subnormal code * 2^-24, bits 4-7
//     code * 2^-20.  The tensor core multiplies subnormals exactly, so unpacking is one AND per two codes (and one shift
//     per eight); the power of two comes out with the scale.  Low and high nibbles go to separate accumulators (keys) or
//     separate accumulator rows (values).
//   - Codes are the 16-row operand of mma.sync.m16n8k16 and the queries that share a key/value head its 8 columns, so a
//     group of up to eight query heads costs what one does.  S^T = K Q^T leaves P^T in the layout from which
//     movmatrix makes the second product's operand; nothing goes through shared memory but the cache itself.
//     (tcgen05.mma could take unpacked codes from tensor memory, written there from registers, and pays where many columns share
//     them; a few query columns do not, and a kernel for prompts was not built.  6000 new tokens of one sequence, 32 / 8 heads of
//     128 channels, take 4.3 ms here, 69 TFLOP/s: every eight columns load and unpack the rows again, and units that an item's
//     last row does not see are still gone through.)
//   - The softmax's running maximum moves only when a weight exceeds it by more than 2^8 (a warp vote per 32 or 64 rows instead
//     of a reduction); weights then stay below 2^8 and exact sums are unchanged, since every term uses the same m.
//     The maximum is taken over log2(p_t sv_t), the weight that is rounded to fp16: its relative error is 2^-11 whatever
//     the scale of the values.
//   - The fp16 weights alone would leave the output's error at 2.7 times that of an exact result rounded to fp16 (codes are never
//     negative, so errors of weights meet codes at their full size).  What the rounding of a weight leaves over, again in fp16, is
//     a second operand of the same product: 1.00 to 1.2 times then.  (64 sequences of up to 8000 rows: 95 us against 86
//     without; the weights' errors on codes about their middle, which costs 88, still give 1.4 to 1.55; now 93.6.)
//   - The tensor core cuts off, towards zero, what does not fit below a 32-bit accumulator; over thousands of rows of
//     codes that are never negative that adds up (3.3 times the rounding of the output).  Every kDriftSlots slots one more product
//     takes 7.5 times the weights of those slots off all accumulators, halfway, and its exact amount goes to the 32-bit sums:
//     the accumulators stay small, and are below zero as often as above.
//
// Each warp streams its own slots of four blocks through its own ring (bulk copies, one mbarrier per slot), so no
// warp waits for another inside a segment.  The rows of all (sequence, head, query tile) items form one list of 256-row
// units that is dealt out evenly to the CTAs whatever the lengths; an item that several CTAs share is joined by the last of
// them to finish, in CTA order (deterministic), from partial sums in the workspace.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <type_traits>

#include "../../include/fastgate_b200.h"
#include "fg_host.h"
#include "fg_kv4.cuh"

namespace fg {
namespace {

constexpr int kAttnWarps = 4;
constexpr int kAttnThreads = kAttnWarps * 32;
constexpr int kPairRows = 2 * kKvBlock;       // rows of one masked step of the softmax
constexpr int kSlotBlocks = 4;                // blocks of a ring slot
constexpr int kSlotRows = kSlotBlocks * kKvBlock;
constexpr int kUnitRows = kAttnWarps * kSlotRows;
constexpr int kAttnMaxGrid = 1024;
constexpr int kDriftSlots = 4;                // slots of a warp per correction (8 gave up to 1.4 times the output's rounding)
constexpr float kLazyMax = 8.f;               // log2 of how far a weight may exceed the running maximum
constexpr float kNoMax = -1e30f;              // stands for the maximum of no rows (scores stay far above it)
constexpr float kMaxScale = 1048576.f;        // largest softmax scale: |scores| < 2^20 * 128 * 2^36
constexpr unsigned long long kAttnWaitNs = 2000000000ull;
constexpr int kStatusAttnTimeout = 6;         // FG_ERR_TIMEOUT

// Workspace: [0,256) header, kAttnMaxGrid tickets (zero between launches), then two partials per CTA.
constexpr size_t kAttnTicketsOffset = 256;
constexpr size_t kAttnPartialsOffset = kAttnTicketsOffset + kAttnMaxGrid * 4;
__host__ __device__ constexpr int partial_floats(int d, int cols) { return cols * (d + 4); }  // [cols][d] sums, [cols] maxima, [cols] norms, padding
__host__ __device__ constexpr int attn_stages(int d) { return (d == 128 ? 8 : 12) / kSlotBlocks; }  // ring slots of a warp
__host__ __device__ constexpr int attn_slot_bytes(int d, int cols) {                          // a warp's sums are parked in the slot it has emptied last
  return kSlotBlocks * kv_block_bytes(d) > cols * d * 4 ? kSlotBlocks * kv_block_bytes(d) : cols * d * 4;
}
__host__ __device__ constexpr int attn_smem_bytes(int d, int cols) { return kAttnWarps * attn_stages(d) * attn_slot_bytes(d, cols); }
// (Measured with eight columns, two CTAs that take four blocks a step / three that have registers for two: 64 sequences of up to
// 8000 rows 95 / 99 us, one of 5000 11.1 / 13.7.  A third ring slot changes neither.  Sixteen columns, 24 x 3000 rows of 64
// channels, two / three / four CTAs: 20.6 / 22.9 / 28.4, before the second operand of the weights.)
constexpr int kAttnCtasPerSm = 2;
constexpr int kAttnMostFloats = partial_floats(64, 16);  // of a partial; eight columns of 128 channels take less
static_assert(partial_floats(128, 8) <= kAttnMostFloats, "workspace");

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
__device__ __forceinline__ uint32_t add_release(unsigned int* p, unsigned int v) {
  uint32_t r;
  asm volatile("atom.add.release.gpu.global.u32 %0, [%1], %2;" : "=r"(r) : "l"(p), "r"(v) : "memory");
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
// Words of a shared-memory row (ordinary loads: the compiler may place them).
template <int BYTES>
__device__ __forceinline__ void lds_words(const uint8_t* p, uint32_t (&w)[BYTES / 4]) {
  if constexpr (BYTES == 16) {
    const uint4 v = *reinterpret_cast<const uint4*>(p);
    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
  } else if constexpr (BYTES == 8) {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    w[0] = v.x; w[1] = v.y;
  } else {
    w[0] = *reinterpret_cast<const uint32_t*>(p);
  }
}
__device__ __forceinline__ float2 lds_half2(const uint8_t* p) { return __half22float2(*reinterpret_cast<const __half2*>(p)); }
// D(16x8, f32) = A(16x16, f16, row) B(16x8, f16, col) + C
__device__ __forceinline__ void mma_codes(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1,
                                          float c0, float c1, float c2, float c3) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%11,%12,%13};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c0), "f"(c1), "f"(c2), "f"(c3));
}

// What of the work list belongs to sequence b.
struct Sequence {
  int len;         // its rows in the cache
  int q0, nq;      // its query tokens
  uint32_t tiles;  // query tiles per key/value head
  uint32_t units;  // units per item, at least one
  __device__ uint32_t total(int kv_heads) const { return tiles * kv_heads * units; }  // < 2^31: the host has checked
};

template <int COLS>
__device__ __forceinline__ Sequence sequence(const AttnParams& p, int b, bool report) {
  Sequence s;
  bool bad = false;
  s.len = p.lens[b];
  if (s.len < 0 || s.len > p.table_width * p.kv.page_size) {
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
  s.tiles = (static_cast<uint32_t>(s.nq) * p.group + COLS - 1) / COLS;
  s.units = s.len > 0 ? (s.len + kUnitRows - 1) / kUnitRows : 1;
  return s;
}

// A place in the work list.
struct Walk {
  int b;            // sequence
  uint32_t before;  // units before it
  Sequence sq;
};
struct Segment {
  uint32_t item_u0;     // first unit of the item
  int first, len;       // units of the item
  int head, tile;
};

// An item of which this CTA has left a partial: joined at the CTA's end if it was the last to leave one.
struct Pending {
  uint32_t first, parts;  // the CTAs that share the item
  uint32_t first_slot;    // which of its two partials the first one's is
  uint32_t ticket;        // how many had left theirs before
  int cols, tile, head, q0;
};

template <int D, int NQ>
__global__ void __launch_bounds__(kAttnThreads, kAttnCtasPerSm) fg_kv_attention_kernel(const AttnParams p) {
  constexpr int COLS = 8 * NQ;          // query columns of an item
  constexpr int KW = D / 32;            // 32-bit words of a key row per lane
  constexpr int VW = D / 64;            // 32-bit words of a value row per lane
  constexpr int MT = D / 16;            // 16-channel accumulator tiles
  constexpr int SB = kv_block_bytes(D);
  constexpr int S = attn_stages(D);
  constexpr int kSlot = attn_slot_bytes(D, COLS);
  constexpr uint32_t kNoBlock = 0xffffffffu, kSlotMask = (1u << kSlotBlocks) - 1;
  constexpr int kSet = 32 / kSlotBlocks;  // slots whose blocks the lanes of a warp hold
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ __align__(8) unsigned long long bars[kAttnWarps * S];
  __shared__ uint32_t scan[kAttnWarps], scan_rough[kAttnWarps], start_before;
  __shared__ int start_b;
  __shared__ Pending pending[2];
  __shared__ float warp_max[kAttnWarps][COLS], warp_norm[kAttnWarps][COLS];
  __shared__ const float* warp_sums[kAttnWarps];

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, c = lane & 3;
  uint8_t* ring = smem + warp * (S * kSlot);
  const uint32_t ring_u32 = smem_u32(ring);
  const uint32_t bar = smem_u32(bars + warp * S);
  if (lane < S) mbar_init(bar + 8 * lane, 1);
  fence_mbar_init();
  fence_proxy_async();
  griddep_wait();
  griddep_launch_dependents();

  // ---- this CTA's share [ub, ue) of the work list: equal runs of `chunk` units ----
  const int kv_heads = p.kv.heads;
  const int per = (p.batch + kAttnThreads - 1) / kAttnThreads;
  const int b_lo = min(p.batch, tid * per), b_hi = min(p.batch, b_lo + per);
  unsigned long long sum = 0;
  for (int b = b_lo; b < b_hi; ++b) sum += sequence<COLS>(p, b, blockIdx.x == 0).total(kv_heads);
  const uint32_t mine = static_cast<uint32_t>(min(sum, 0x80000000ull));
  uint32_t incl = mine;
#pragma unroll
  for (int off = 1; off < 32; off <<= 1) {
    const uint32_t v = __shfl_up_sync(0xffffffffu, incl, off);
    if (lane >= off) incl += v;
  }
  const uint32_t rough = __reduce_add_sync(0xffffffffu, mine >> 12);
  if (lane == 31) {
    scan[warp] = incl;
    scan_rough[warp] = rough;
  }
  __syncthreads();
  uint32_t before = incl - mine, total = 0, all_rough = 0;
#pragma unroll
  for (int w = 0; w < kAttnWarps; ++w) {
    if (w < warp) before += scan[w];
    total += scan[w];
    all_rough += scan_rough[w];
  }
  if (all_rough >= 0x80000u - kAttnThreads) {  // about 2^31 units, more than q has rows for: q_starts overlap
    if (tid == 0 && blockIdx.x == 0 && p.status != nullptr) atomicExch(p.status, kStatusIndex);
    return;
  }
  const uint32_t chunk = (total + gridDim.x - 1) / gridDim.x;
  const uint32_t cta = blockIdx.x, ub = cta * chunk, ue = min(total, ub + chunk);
  if (ub >= total) return;
  if (ub >= before && ub - before < mine) {
    int b = b_lo;
    for (;; ++b) {
      const uint32_t t = sequence<COLS>(p, b, false).total(kv_heads);
      if (ub < before + t) break;
      before += t;
    }
    start_b = b;
    start_before = before;
  }
  __syncthreads();
  auto settle = [&](Walk& w, uint32_t u) {  // to the sequence that holds unit u
    while (u >= w.before + w.sq.total(kv_heads)) {
      w.before += w.sq.total(kv_heads);
      w.sq = sequence<COLS>(p, ++w.b, false);
    }
  };
  auto segment_at = [&](const Walk& w, uint32_t u) {  // from unit u to the end of its item or of the share
    Segment s;
    const uint32_t item = (u - w.before) / w.sq.units;
    s.item_u0 = w.before + item * w.sq.units;
    s.first = static_cast<int>(u - s.item_u0);
    s.len = static_cast<int>(min(w.sq.units - s.first, ue - u));
    s.head = static_cast<int>(item / w.sq.tiles);
    s.tile = static_cast<int>(item - s.head * w.sq.tiles);
    return s;
  };
  // slots that this warp takes of a segment: warp, warp + 4, ... counted from its first row
  auto slots_of = [&](const Walk& w, const Segment& s) {
    const int first = s.first * kAttnWarps + warp, end = min((w.sq.len + kSlotRows - 1) / kSlotRows, (s.first + s.len) * kAttnWarps);
    return end > first ? (end - first + kAttnWarps - 1) / kAttnWarps : 0;
  };

  // ---- copies: a cursor that runs up to S slots ahead of the rows being used, across segments ----
  const int blocks_per_page = p.kv.page_size / kKvBlock;
  Walk cw = {start_b, start_before, sequence<COLS>(p, start_b, false)};
  uint32_t cu = ub;                  // where the cursor's segment begins
  int c_slots = 0, c_next = 0;       // its slots of this warp, and the next one to be copied
  int c_first = 0, c_head = 0, c_slot = 0;
  uint32_t now_at, now_bytes, now_none, next_at, next_bytes, next_none;
  uint32_t gone = 0;                 // a bit per block of the ring: those that are not there
  // Lane kSlotBlocks i + k holds block k of the i-th of kSet slots: its number, and how many bytes to copy from it (neighbouring blocks
  // of a slot that lie side by side in the pool are one copy).  `none`: which of the 32 are absent.
  auto fetch = [&](int set, uint32_t& at, uint32_t& bytes, uint32_t& none) {
    const int i = kSet * set + lane / kSlotBlocks, blk = (c_first + i * kAttnWarps) * kSlotBlocks + lane % kSlotBlocks;
    at = kNoBlock;
    if (i < c_slots && blk * kKvBlock < cw.sq.len) {
      const int nth = blk / blocks_per_page, page = p.table[static_cast<long long>(cw.b) * p.ldt + nth];
      if (page >= 0 && page < p.kv.pages)
        at = (static_cast<uint32_t>(page) * kv_heads + c_head) * blocks_per_page + (blk - nth * blocks_per_page);
      else if (p.status != nullptr)
        atomicExch(p.status, kStatusIndex);
    }
    const uint32_t left = __shfl_up_sync(0xffffffffu, at, 1);
    const bool follows = lane % kSlotBlocks != 0 && at != kNoBlock && left != kNoBlock && at == left + 1;
    const uint32_t chain = __ballot_sync(0xffffffffu, follows);
    none = __ballot_sync(0xffffffffu, at == kNoBlock);
    const int run = lane == 31 ? 1 : __ffs(~(chain >> (lane + 1)));  // 1 + the blocks that follow
    bytes = at != kNoBlock && !follows ? run * SB : 0;
  };
  auto open = [&](uint32_t u) {  // the cursor enters the segment that begins at u, or the first after it with rows for this warp
    for (cu = u; cu < ue;) {
      settle(cw, cu);
      const Segment s = segment_at(cw, cu);
      c_slots = slots_of(cw, s);
      c_next = 0;
      cu += s.len;
      if (c_slots > 0) {
        c_first = s.first * kAttnWarps + warp;
        c_head = s.head;
        fetch(0, now_at, now_bytes, now_none);
        if (c_slots > kSet) fetch(1, next_at, next_bytes, next_none);
        return;
      }
    }
    c_slots = c_next = 0;
  };
  auto copy_next = [&]() {  // whole warp: the next slot of the stream into the ring
    if (c_next == c_slots) {
      if (c_slots == 0 && cu >= ue) return;
      open(cu);
      if (c_slots == 0) return;
    }
    const int i = c_next % kSet;
    const uint32_t missing = (now_none >> (kSlotBlocks * i)) & kSlotMask;
    gone = (gone & ~(kSlotMask << (kSlotBlocks * c_slot))) | (missing << (kSlotBlocks * c_slot));
    if (lane / kSlotBlocks == i) {
      const uint32_t full = bar + 8 * c_slot;
      if (lane % kSlotBlocks == 0) mbar_arrive_expect_tx(full, SB * (kSlotBlocks - __popc(missing)));
      if (now_bytes != 0)
        bulk_load(ring_u32 + c_slot * kSlot + (lane % kSlotBlocks) * SB, p.kv.base + static_cast<size_t>(now_at) * SB, now_bytes, full);
    }
    __syncwarp();
    c_slot = c_slot + 1 == S ? 0 : c_slot + 1;
    ++c_next;
    if (c_next % kSet == 0 && c_next < c_slots) {
      now_at = next_at;
      now_bytes = next_bytes;
      now_none = next_none;
      if (c_next + kSet < c_slots) fetch(c_next / kSet + 1, next_at, next_bytes, next_none);
    }
  };
  // Output: a thread has four channels of every (kAttnThreads / (D / 4))th column.
  constexpr int TPC = D / 4;
  const int d4 = (tid % TPC) * 4;
  auto write_out = [&](int flat, int head, int q0, float4 v, float l) {
    const float inv = l == 0.f ? 0.f : 1.f / l;  // a row that sees nothing gives zeros
    const __half2 h0 = __floats2half2_rn(v.x * inv, v.y * inv), h1 = __floats2half2_rn(v.z * inv, v.w * inv);
    *reinterpret_cast<uint2*>(p.out + static_cast<long long>(q0 + flat / p.group) * p.ldo +
                              static_cast<long long>(head * p.group + flat % p.group) * D + d4) =
        make_uint2(*reinterpret_cast<const uint32_t*>(&h0), *reinterpret_cast<const uint32_t*>(&h1));
  };

  // ---- queries: 16-byte pieces of a segment's columns, fetched ahead of their use ----
  uint4 raw[NQ][KW];
  auto load_queries = [&](const Sequence& sq, const Segment& seg) {
    const int cols = min(COLS, sq.nq * p.group - seg.tile * COLS);
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const int col = n * 8 + g, flat = seg.tile * COLS + col;
      const __half* src = p.q + static_cast<long long>(sq.q0 + flat / p.group) * p.ldq +
                          static_cast<long long>(seg.head * p.group + flat % p.group) * D + c * (8 * KW);
#pragma unroll
      for (int i = 0; i < KW; ++i) raw[n][i] = col < cols ? *reinterpret_cast<const uint4*>(src + 8 * i) : make_uint4(0, 0, 0, 0);
    }
  };
  Walk w = cw;
  settle(w, ub);
  Segment seg = segment_at(w, ub);
  load_queries(w.sq, seg);
  open(ub);
  for (int i = 0; i < S; ++i) copy_next();

  uint32_t phase = 0;  // one bit per ring slot
  int slot = 0, n_pending = 0;
  bool dead = false;
  for (uint32_t u = ub; u < ue;) {
    const Sequence sq = w.sq;
    const int head = seg.head, tile = seg.tile;
    const int cols = min(COLS, sq.nq * p.group - tile * COLS);
    const int n_slots = dead ? 0 : slots_of(w, seg);

    // ---- queries as fragments, their sums, the last row that each column sees ----
    uint32_t qf[NQ][KW][4];
    float qs[NQ][2];
    int limit[NQ][2];
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        // channels (0,4), (2,6) meet the low nibbles' pairs, (1,5), (3,7) the high ones'
        qf[n][i][0] = prmt(raw[n][i].x, raw[n][i].z, 0x5410);
        qf[n][i][1] = prmt(raw[n][i].y, raw[n][i].w, 0x5410);
        qf[n][i][2] = prmt(raw[n][i].x, raw[n][i].z, 0x7632);
        qf[n][i][3] = prmt(raw[n][i].y, raw[n][i].w, 0x7632);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&qf[n][i][k]));
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
    const int min_limit = sq.len - sq.nq + (tile * COLS) / p.group;  // column 0 sees least

    float oacc[NQ][MT][4], mref[NQ][2], lsum[NQ][2], zsum[NQ][2];
    __half2 drift[NQ];  // weights of up to kDriftSlots slots: 2^8 * 2 * 16 at most
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      drift[n] = __float2half2_rn(0.f);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        mref[n][i] = 0.f;
        lsum[n][i] = zsum[n][i] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < MT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) oacc[n][t][i] = 0.f;
    }

    // Operand row g of a 16-row block is its row ka, operand row g + 8 its row ka + 8: rows 2i and 2i + 1 of an operand then
    // lie in different halves of the shared-memory banks.
    const int ka = (g & 1) ? 4 + ((g >> 1) ^ 1) : g >> 1;
    const int v0 = c, v1 = 4 + (c ^ 1);
    bool fresh = true;  // no rows yet: the first ones set the maximum, whatever its size
    // NB blocks.  MASKED: some column does not see all of their rows, or a block is absent.
    auto consume = [&](const uint8_t* base, int row0, uint32_t absent, auto masked_tag, auto blocks_tag) {
      constexpr bool MASKED = decltype(masked_tag)::value;
      constexpr int NB = decltype(blocks_tag)::value;
      float t[NB][NQ][4];          // log2 of the weights over the values' scales, less the running maximum
      float sv[NB][2], lv[NB][2];  // the value rows' scale and low end
      bool up = fresh;
#pragma unroll
      for (int h = 0; h < NB; ++h) {
        const uint8_t* blk = base + h * SB;
        // S^T = K Q^T on the codes
        uint32_t wa[KW], wb[KW];
        lds_words<4 * KW>(blk + kv_codes_offset(D, 0, ka) + c * (4 * KW), wa);
        lds_words<4 * KW>(blk + kv_codes_offset(D, 0, ka + 8) + c * (4 * KW), wb);
        float slo[NQ][4], shi[NQ][4];
#pragma unroll
        for (int i = 0; i < KW; ++i) {
          const uint32_t xa = wa[i] >> 8, xb = wb[i] >> 8;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            float *l = slo[n], *u = shi[n];
            mma_codes(slo[n], wa[i] & 0x000F000Fu, wb[i] & 0x000F000Fu, xa & 0x000F000Fu, xb & 0x000F000Fu, qf[n][i][0], qf[n][i][1],
                      i ? l[0] : 0.f, i ? l[1] : 0.f, i ? l[2] : 0.f, i ? l[3] : 0.f);
            mma_codes(shi[n], wa[i] & 0x00F000F0u, wb[i] & 0x00F000F0u, xa & 0x00F000F0u, xb & 0x00F000F0u, qf[n][i][2], qf[n][i][3],
                      i ? u[0] : 0.f, i ? u[1] : 0.f, i ? u[2] : 0.f, i ? u[3] : 0.f);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const float2 kp = lds_half2(blk + kv_params_offset(D, 0, ka + 8 * r)), vp = lds_half2(blk + kv_params_offset(D, 1, ka + 8 * r));
          const float sk = kp.x * (p.scale_log2 * 16777216.f);
          sv[h][r] = vp.x;
          lv[h][r] = vp.y;
          const float most = kLazyMax - lg2(fmaxf(vp.x, 5.9604644775390625e-8f));  // weight * scale <= 2^kLazyMax
#pragma unroll
          for (int n = 0; n < NQ; ++n)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float v = fmaf(fmaf(shi[n][2 * r + q], 0.0625f, slo[n][2 * r + q]), sk, fmaf(kp.y, qs[n][q], -mref[n][q]));
              if (MASKED && (row0 + 16 * h + ka + 8 * r > limit[n][q] || ((absent >> h) & 1u))) v = -INFINITY;
              t[h][n][2 * r + q] = v;
              up |= v > most;
            }
        }
      }
      if (__any_sync(0xffffffffu, up)) {
        // a new maximum: the largest of the old one and these rows', and everything so far brought to it
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          drift[n] = __float2half2_rn(0.f);  // what they added has just shrunk
#pragma unroll
          for (int q = 0; q < 2; ++q) {
            float m = fresh ? -INFINITY : 0.f;  // relative to the old one
#pragma unroll
            for (int h = 0; h < NB; ++h)
#pragma unroll
              for (int r = 0; r < 2; ++r) m = fmaxf(m, t[h][n][2 * r + q] + lg2(fmaxf(sv[h][r], 5.9604644775390625e-8f)));
#pragma unroll
            for (int off = 4; off <= 16; off <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, off));
            if (m == -INFINITY) m = 0.f;  // a column that sees none of them (nor, then, any later row)
            const float f = fresh ? 1.f : ex2(-m);
            mref[n][q] += m;
            lsum[n][q] *= f;
            zsum[n][q] *= f;
#pragma unroll
            for (int h = 0; h < NB; ++h) {
              t[h][n][q] -= m;
              t[h][n][2 + q] -= m;
            }
#pragma unroll
            for (int i = 0; i < MT; ++i) {
              oacc[n][i][q] *= f;
              oacc[n][i][2 + q] *= f;
            }
          }
        }
        if (absent != (1u << NB) - 1) fresh = false;
      }
#pragma unroll
      for (int h = 0; h < NB; ++h) {
        const uint8_t* blk = base + h * SB;
        uint32_t pb[NQ][2], pl[NQ][2];  // the weights' fp16, and what it leaves over
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          float wgt[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int r = i >> 1, q = i & 1;
            const float e = ex2(t[h][n][i]);
            lsum[n][q] += e;
            if (MASKED && t[h][n][i] == -INFINITY) {
              wgt[i] = 0.f;  // whatever the row's parameters hold
            } else {
              zsum[n][q] = fmaf(e, lv[h][r], zsum[n][q]);
              wgt[i] = e * sv[h][r];
            }
          }
          const __half2 h0 = __floats2half2_rn(wgt[0], wgt[1]), h1 = __floats2half2_rn(wgt[2], wgt[3]);
          const float2 f0 = __half22float2(h0), f1 = __half22float2(h1);
          const __half2 l0 = __floats2half2_rn(wgt[0] - f0.x, wgt[1] - f0.y), l1 = __floats2half2_rn(wgt[2] - f1.x, wgt[3] - f1.y);
          drift[n] = __hadd2(drift[n], __hadd2(h0, h1));
          pb[n][0] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&h0));
          pb[n][1] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&h1));
          pl[n][0] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&l0));
          pl[n][1] = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&l1));
        }
        // O^T += V^T P^T on the codes: lane g owns channels 8 VW g.., operand columns are rows (v0, v1) and (v0, v1) + 8
        uint32_t r0[VW], r1[VW], r2[VW], r3[VW];
        lds_words<4 * VW>(blk + kv_codes_offset(D, 1, v0) + g * (4 * VW), r0);
        lds_words<4 * VW>(blk + kv_codes_offset(D, 1, v1) + g * (4 * VW), r1);
        lds_words<4 * VW>(blk + kv_codes_offset(D, 1, v0 + 8) + g * (4 * VW), r2);
        lds_words<4 * VW>(blk + kv_codes_offset(D, 1, v1 + 8) + g * (4 * VW), r3);
#pragma unroll
        for (int i = 0; i < VW; ++i)
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            // row g: the even channel's code; row g + 8: the whole byte, even + 16 odd (an exact fp16 too), which takes no
            // second mask: the odd channel's sum is the difference, once at the end
            const uint32_t xa = prmt(r0[i], r1[i], hf ? 0x7632 : 0x5410), xb = prmt(r2[i], r3[i], hf ? 0x7632 : 0x5410);
            const uint32_t ya[2] = {xa & 0x00FF00FFu, prmt(xa, 0u, 0x4341)}, yb[2] = {xb & 0x00FF00FFu, prmt(xb, 0u, 0x4341)};
#pragma unroll
            for (int part = 0; part < 2; ++part)
#pragma unroll
              for (int by = 0; by < 2; ++by)
#pragma unroll
                for (int n = 0; n < NQ; ++n) {
                  float* o = oacc[n][i * 4 + hf * 2 + by];
                  mma_codes(oacc[n][i * 4 + hf * 2 + by], ya[by] & 0x000F000Fu, ya[by], yb[by] & 0x000F000Fu, yb[by],
                            part ? pl[n][0] : pb[n][0], part ? pl[n][1] : pb[n][1], o[0], o[1], o[2], o[3]);
                }
          }
      }
    };

    constexpr int kStep = 4 / NQ;  // blocks of one softmax step, as registers allow
    int row0 = (seg.first * kAttnWarps + warp) * kSlotRows;
    for (int j = 0; j < n_slots; ++j, row0 += kUnitRows) {
      if (!__all_sync(0xffffffffu, mbar_wait_bounded(bar + 8 * slot, (phase >> slot) & 1u, kAttnWaitNs))) {
        dead = true;
        if (lane == 0 && p.status != nullptr) atomicExch(p.status, kStatusAttnTimeout);
        break;
      }
      phase ^= 1u << slot;
      const uint8_t* base = ring + slot * kSlot;
      const uint32_t absent = (gone >> (kSlotBlocks * slot)) & kSlotMask;
      if (row0 + kSlotRows - 1 <= min_limit && absent == 0) {
#pragma unroll
        for (int h = 0; h < kSlotBlocks; h += kStep) consume(base + h * SB, 0, 0u, std::false_type{}, std::integral_constant<int, kStep>{});
      } else {
#pragma unroll 1
        for (int h = 0; h < kSlotBlocks / 2; ++h)
          if (row0 + h * kPairRows < sq.len) consume(base + h * (2 * SB), row0 + h * kPairRows, (absent >> (2 * h)) & 3u, std::true_type{}, std::integral_constant<int, 2>{});
      }
      __syncwarp();  // every lane has read the slot
      if (j % kDriftSlots == kDriftSlots - 1) {
#pragma unroll
        for (int n = 0; n < NQ; ++n) drift[n] = __float2half2_rn(0.f);
      }
      if (j % kDriftSlots == kDriftSlots / 2 - 1) {  // for what these two slots have added and as much that is to come
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          const __half2 off = __hneg2(drift[n]);  // times code 15 of either nibble
          const float2 f = __half22float2(off);
          zsum[n][0] = fmaf(-15.f, f.x, zsum[n][0]);
          zsum[n][1] = fmaf(-15.f, f.y, zsum[n][1]);
          const uint32_t b = movmatrix_trans(*reinterpret_cast<const uint32_t*>(&off));
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            float* o = oacc[n][t];
            mma_codes(oacc[n][t], 0x000F000Fu, 0x00FF00FFu, 0u, 0u, b, 0u, o[0], o[1], o[2], o[3]);
          }
        }
      }
      if (j + 1 < n_slots) copy_next();  // (the last one's is parked in first)
      slot = slot + 1 == S ? 0 : slot + 1;
    }

    // ---- the next segment: its first rows are on their way already, its queries are asked for now ----
    const uint32_t u_next = u + seg.len;
    const Segment here = seg;
    if (u_next < ue) {
      settle(w, u_next);
      seg = segment_at(w, u_next);
      load_queries(w.sq, seg);
    }

    // ---- the four warps' sums meet in shared memory ----
    float* park = reinterpret_cast<float*>(ring + (slot == 0 ? S - 1 : slot - 1) * kSlot);
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
        if (n_slots > 0) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            // accumulator row g holds the even channel (low nibble), row g + 8 even + 16 odd
            const float2 v = make_float2(fmaf(oacc[n][t][q], 16777216.f, z), fmaf(oacc[n][t][2 + q] - oacc[n][t][q], 1048576.f, z));
            *reinterpret_cast<float2*>(park + col * D + g * (8 * VW) + 2 * t) = v;
          }
        }
        if (g == 0) {
          warp_max[warp][col] = n_slots == 0 || l == 0.f ? kNoMax : mref[n][q];
          warp_norm[warp][col] = dead ? NAN : l;
        }
      }
    if (lane == 0) warp_sums[warp] = n_slots > 0 ? park : nullptr;
    __syncthreads();
    const bool whole = here.len == static_cast<int>(sq.units);
    float* part = p.partials + static_cast<size_t>(cta * 2 + (u == ub ? 0 : 1)) * partial_floats(D, COLS);
#pragma unroll 1
    for (int col = tid / TPC; col < cols; col += kAttnThreads / TPC) {
      float m = kNoMax, l = 0.f;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int i = 0; i < kAttnWarps; ++i) m = fmaxf(m, warp_max[i][col]);
#pragma unroll
      for (int i = 0; i < kAttnWarps; ++i) {
        const float f = ex2(warp_max[i][col] - m);
        l = fmaf(f, warp_norm[i][col], l);
        if (warp_sums[i] != nullptr) {
          const float4 a = *reinterpret_cast<const float4*>(warp_sums[i] + col * D + d4);
          v.x = fmaf(f, a.x, v.x);
          v.y = fmaf(f, a.y, v.y);
          v.z = fmaf(f, a.z, v.z);
          v.w = fmaf(f, a.w, v.w);
        }
      }
      if (whole) {
        write_out(tile * COLS + col, head, sq.q0, v, l);
      } else {
        __stcg(reinterpret_cast<float4*>(part + col * D + d4), v);
        if (d4 == 0) {
          __stcg(part + COLS * D + col, m);
          __stcg(part + COLS * D + COLS + col, l);
        }
      }
    }
    fence_proxy_async();  // the parked sums have been read before copies overwrite them
    __syncthreads();
    if (n_slots > 0 && !dead) copy_next();
    if (!whole) {
      // Publish the partial and go on; who was last is looked at when the share is done.
      if (tid == 0) {
        Pending& q = pending[n_pending];
        q.first = here.item_u0 / chunk;
        q.parts = (here.item_u0 + sq.units - 1) / chunk - q.first + 1;
        q.first_slot = q.first * chunk < here.item_u0 ? 1 : 0;  // only the first CTA can have begun its share in an earlier item
        q.cols = cols;
        q.tile = tile;
        q.head = head;
        q.q0 = sq.q0;
        q.ticket = add_release(p.tickets + q.first, 1u);  // the other threads' stores too: the barrier has ordered them before
      }
      ++n_pending;
    }
    u = u_next;
  }

  // ---- items of several CTAs: the last of them to get here joins the partials in CTA order ----
  if (n_pending > 0) {
    // The thread that took the tickets acquires what the other CTAs released with theirs, the barrier carries it to all threads.
    if (tid == 0) fence_acq_rel_gpu();
    __syncthreads();
  }
  for (int k = 0; k < n_pending; ++k) {
    const Pending q = pending[k];
    if (q.ticket != q.parts - 1) continue;
    const float* first = p.partials + static_cast<size_t>(q.first * 2) * partial_floats(D, COLS);
    auto part_of = [&](uint32_t x) { return first + static_cast<size_t>(2 * x + (x == 0 ? q.first_slot : 0)) * partial_floats(D, COLS); };
    // With L2 most of a microsecond away it is the number of dependent passes that counts: a thread asks for 24 partials of its
    // column at once, maxima included, or for 8 of each of two columns where there are more than one per thread (one sequence of
    // 5000 rows in 20 parts, before dependents were signalled after the wait: 10.4 us, with 8 at once 11.2).
    constexpr int kStep = kAttnThreads / TPC;
    auto join = [&](auto columns) {
      constexpr int Y = decltype(columns)::value;
      constexpr uint32_t kParts = Y == 1 ? 24 : 8;
#pragma unroll 1
      for (int col0 = tid / TPC; col0 < q.cols; col0 += Y * kStep) {
        float m[Y], l[Y];
        float4 v[Y];
#pragma unroll
        for (int y = 0; y < Y; ++y) {
          m[y] = kNoMax;
          l[y] = 0.f;
          v[y] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll 1
        for (uint32_t x0 = 0; x0 < q.parts; x0 += kParts) {
          float4 a[kParts][Y];
          float mx[kParts][Y], lx[kParts][Y];
#pragma unroll
          for (uint32_t i = 0; i < kParts; ++i)
#pragma unroll
            for (int y = 0; y < Y; ++y)
              if (x0 + i < q.parts && col0 + y * kStep < q.cols) {
                const float* src = part_of(x0 + i);
                const int col = col0 + y * kStep;
                a[i][y] = __ldcg(reinterpret_cast<const float4*>(src + col * D + d4));
                mx[i][y] = __ldcg(src + COLS * D + col);
                lx[i][y] = __ldcg(src + COLS * D + COLS + col);
              } else {
                a[i][y] = make_float4(0.f, 0.f, 0.f, 0.f);
                mx[i][y] = kNoMax;
                lx[i][y] = 0.f;
              }
#pragma unroll
          for (int y = 0; y < Y; ++y) {
            float top = m[y];
#pragma unroll
            for (uint32_t i = 0; i < kParts; ++i) top = fmaxf(top, mx[i][y]);
            const float back = ex2(m[y] - top);
            m[y] = top;
            l[y] *= back;
            v[y].x *= back;
            v[y].y *= back;
            v[y].z *= back;
            v[y].w *= back;
#pragma unroll
            for (uint32_t i = 0; i < kParts; ++i) {
              const float f = ex2(mx[i][y] - top);
              l[y] = fmaf(f, lx[i][y], l[y]);
              v[y].x = fmaf(f, a[i][y].x, v[y].x);
              v[y].y = fmaf(f, a[i][y].y, v[y].y);
              v[y].z = fmaf(f, a[i][y].z, v[y].z);
              v[y].w = fmaf(f, a[i][y].w, v[y].w);
            }
          }
        }
#pragma unroll
        for (int y = 0; y < Y; ++y)
          if (col0 + y * kStep < q.cols) write_out(q.tile * COLS + col0 + y * kStep, q.head, q.q0, v[y], l[y]);
      }
    };
    if (q.cols <= kStep) join(std::integral_constant<int, 1>{});
    else join(std::integral_constant<int, 2>{});
    if (tid == 0) p.tickets[q.first] = 0;  // ready for the next launch
  }
  if (dead) {
    // a wait gave up: copies that are still in flight get time to land before the shared memory goes away
    for (int i = 0; i < S; ++i) mbar_wait_bounded(bar + 8 * i, (phase >> i) & 1u, kAttnWaitNs / 10);
  }
}

}  // namespace
}  // namespace fg

extern "C" size_t fg_kv_attention_workspace_bytes(void) {
  return fg::kAttnPartialsOffset + static_cast<size_t>(fg::kAttnMaxGrid) * 2 * fg::kAttnMostFloats * sizeof(float);
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
  if (!(scale > 0.f) || !(scale <= kMaxScale)) return FG_ERR_SHAPE;
  // work units and block numbers are 32-bit in the kernel; an upper bound of both, whatever the lengths turn out to be
  const long long group = q_heads / kv_heads;
  const double most_units = (static_cast<double>(tokens) * group / 8 + batch) * kv_heads * (static_cast<double>(table_width) * page_size / kUnitRows + 1);
  if (most_units >= 2146900000.0 || static_cast<double>(num_pages) * kv_heads * (page_size / kKvBlock) >= 4294967295.0) return FG_ERR_SHAPE;
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
  // Sixteen columns where a sequence has more than eight queries of a key/value head and a head 64 channels: half the unpacking
  // (24 x 3000 rows, 16 columns a sequence: 24.7 us, with eight 29.2; 48 columns: 39.2 / 43.5; thirty-two columns leave too
  // few registers).  With 128 channels the registers spill and eight are as good or better (16 columns 38.1 / 38.6, 48 columns
  // 61.3 / 60.0, 64 x 500 rows 62.1 / 56.1).
  const long long per_seq = (tokens + batch - 1) / batch * p.group;
  const int cols = d == 64 && per_seq > 8 ? 16 : 8;
  void (*kern)(const AttnParams) =
      d == 128 ? fg_kv_attention_kernel<128, 1> : cols == 16 ? fg_kv_attention_kernel<64, 2> : fg_kv_attention_kernel<64, 1>;
  const int smem = attn_smem_bytes(d, cols);
  if ((st = host::opt_in_smem(reinterpret_cast<const void*>(kern), smem)) != FG_OK) return st;
  const int grid = min(kAttnMaxGrid, dev.sm_count * kAttnCtasPerSm);
  return host::launch(kern, dim3(grid), dim3(kAttnThreads), smem, reinterpret_cast<cudaStream_t>(stream), true, p);
}

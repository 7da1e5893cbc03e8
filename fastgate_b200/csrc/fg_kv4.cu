// Rows into and out of the 4-bit key/value cache (fg_kv_append_int4, fg_kv_read_int4); layout in fg_kv4.cuh.
//
// append, per row x of D channels (keys and queries turned first, x' = (a cos - b sin, b cos + a sin) on each pair):
//     low = fp16(min x), scale = max(fp16((max x - low) / 15), 2^-24), code = clamp(rint((x - low) / scale), 0, 15)
// The codes are taken against the parameters as they are stored, so low + scale * code is the nearest value that the
// format has.  2^-24 is the smallest positive fp16: a constant row gets it instead of a division by zero.
//
// Both kernels move each byte once.  Measured on B200: read 40000 rows of 8 heads of 128 channels 37.2 us (5.6 TB/s, nearly four
// fifths of it stores), append 6001 tokens of 48 heads of 64 channels 16.9 us (3.9 TB/s: each lane waits for its slot, then for
// its rows; issue slots are half full), and 64 tokens 2.2, 500 rows read 1.75 us, which is a launch and those latencies.
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "../../include/fastgate_b200.h"
#include "fg_host.h"
#include "fg_kv4.cuh"

namespace fg {
namespace {

constexpr int kKvThreads = 128;  // (6001 tokens appended: 16.6 us, with 256 17.1, with 384 17.8)

struct AppendParams {
  const __half *q, *k, *v;       // token strides ldq, ldk, ldv; heads dense
  long long ldq, ldk, ldv;
  __half* q_out;                 // [T, q_heads, D], token stride ldqo
  long long ldqo;
  int q_heads;                   // 0: no queries
  const float* cos_sin;          // [positions_len, D] or nullptr: no rotation
  long long positions_len;
  IndexArray positions, slots;
  int interleaved;
  KvPages kv;
  int* status;
  long long tokens;
};

__device__ __forceinline__ void unpack8(const uint4& q, float (&v)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  uint4 q;
  uint32_t* w = reinterpret_cast<uint32_t*>(&q);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return q;
}

// Codes of four values as 16 bits: clamped, rounded to integers by adding and taking away 1.5 * 2^23 (to nearest, ties to
// even), and put together as c0 + 16 c1 + 256 c2 + 4096 c3, which 32 bits hold exactly.
// The quotient is the product with 1 / scale and one step of iterative refinement from its remainder: fp16 values often lie
// exactly between two codes, where the bare product would pick either.
__device__ __forceinline__ uint32_t codes4(const float* x, float low, float scale, float inv) {
  float c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float y = x[i] - low;
    float v = y * inv;
    v = fmaf(fmaf(-v, scale, y), inv, v);
    v = fminf(fmaxf(v, 0.f), 15.f);  // NaN: 0
    c[i] = __fsub_rn(__fadd_rn(v, 12582912.f), 12582912.f);
  }
  return static_cast<uint32_t>(__float2int_rn(fmaf(fmaf(fmaf(c[3], 16.f, c[2]), 16.f, c[1]), 16.f, c[0])));
}

// D/16 lanes take a row: lane i the channels 8i.. of its lower half and the matching 8 of its upper half, so that both
// kinds of rotation pair channels within one lane (i with i + D/2, or 2i with 2i + 1).  blockIdx.y picks HPT consecutive
// heads of the list queries, keys, values: whether a row is only turned or also quantised is the same for a whole CTA, and
// one token's heads in a lane have their loads in flight together and share its angles.
template <int D, int HPT>
__global__ void __launch_bounds__(kKvThreads) fg_kv_append_kernel(const AppendParams p) {
  constexpr int LPR = D / 16;  // lanes per row
  const int lane = threadIdx.x % LPR;
  const int heads = p.q_heads + 2 * p.kv.heads, turned = p.q_heads + p.kv.heads;  // head numbers below `turned` are rotated
  const long long token = static_cast<long long>(blockIdx.x) * (kKvThreads / LPR) + threadIdx.x / LPR;
  const int head0 = blockIdx.y * HPT;
  griddep_wait();
  griddep_launch_dependents();

  // A padding token (negative slot) is left out whole; an index out of range too, and reported.
  const bool there = token < p.tokens;
  const long long slot = there ? p.slots[token] : -1;
  const long long pos = there && p.cos_sin != nullptr ? p.positions[token] : 0;
  const bool placed = p.cos_sin == nullptr || (pos >= 0 && pos < p.positions_len);
  const bool go = slot >= 0 && slot < p.kv.pages * p.kv.page_size && placed;
  if (slot >= 0 && !go && lane == 0 && p.status != nullptr) atomicExch(p.status, kStatusIndex);
  uint4 raw[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = head0 + i;
    raw[i][0] = raw[i][1] = make_uint4(0, 0, 0, 0);
    // One head: the row is asked for without waiting for its slot, also a padding token's (64 tokens: 2.3 us, else 2.5).  Four
    // heads: after the slot (6001 tokens of 48 heads, 256 threads: 17.1 us, else 19.2).
    if ((HPT == 1 ? there : go) && h < heads) {
      const __half* src = h < p.q_heads ? p.q + token * p.ldq + static_cast<long long>(h) * D
                          : h < turned  ? p.k + token * p.ldk + static_cast<long long>(h - p.q_heads) * D
                                        : p.v + token * p.ldv + static_cast<long long>(h - turned) * D;
      raw[i][0] = *reinterpret_cast<const uint4*>(src + 8 * lane);
      raw[i][1] = *reinterpret_cast<const uint4*>(src + D / 2 + 8 * lane);
    }
  }
  const bool rotate = p.cos_sin != nullptr && head0 < turned;
  float cs[8], sn[8];
  if (rotate && there && placed) {
    const float* t = p.cos_sin + pos * D;
    // pairs (i, i + D/2): angles 8 lane..; pairs (2i, 2i + 1): angles 4 lane.. of the lower and of the upper half
    const int a0 = p.interleaved ? 4 * lane : 8 * lane, a1 = p.interleaved ? D / 4 + 4 * lane : 8 * lane + 4;
    const float4 c0 = *reinterpret_cast<const float4*>(t + a0), c1 = *reinterpret_cast<const float4*>(t + a1);
    const float4 s0 = *reinterpret_cast<const float4*>(t + D / 2 + a0), s1 = *reinterpret_cast<const float4*>(t + D / 2 + a1);
    cs[0] = c0.x; cs[1] = c0.y; cs[2] = c0.z; cs[3] = c0.w; cs[4] = c1.x; cs[5] = c1.y; cs[6] = c1.z; cs[7] = c1.w;
    sn[0] = s0.x; sn[1] = s0.y; sn[2] = s0.z; sn[3] = s0.w; sn[4] = s1.x; sn[5] = s1.y; sn[6] = s1.z; sn[7] = s1.w;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      cs[j] = 1.f;
      sn[j] = 0.f;
    }
  }

#pragma unroll
  for (int i = 0; i < HPT; ++i) {
    const int h = head0 + i;
    if (h >= heads) break;
    float lo[8], hi[8];
    unpack8(raw[i][0], lo);
    unpack8(raw[i][1], hi);
    if (rotate && h < turned) {
      if (p.interleaved) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float a = lo[2 * j], b = lo[2 * j + 1], c = hi[2 * j], d = hi[2 * j + 1];
          lo[2 * j] = a * cs[j] - b * sn[j];
          lo[2 * j + 1] = b * cs[j] + a * sn[j];
          hi[2 * j] = c * cs[4 + j] - d * sn[4 + j];
          hi[2 * j + 1] = d * cs[4 + j] + c * sn[4 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float a = lo[j], b = hi[j];
          lo[j] = a * cs[j] - b * sn[j];
          hi[j] = b * cs[j] + a * sn[j];
        }
      }
    }
    if (h < p.q_heads) {
      if (go) {
        __half* dst = p.q_out + token * p.ldqo + static_cast<long long>(h) * D;
        *reinterpret_cast<uint4*>(dst + 8 * lane) = pack8(lo);
        *reinterpret_cast<uint4*>(dst + D / 2 + 8 * lane) = pack8(hi);
      }
      continue;
    }
    // every lane of the warp takes part in the row reductions; rows that store nothing are reduced too
    float mn = fminf(lo[0], hi[0]), mx = fmaxf(lo[0], hi[0]), bad = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      mn = fminf(mn, fminf(lo[j], hi[j]));
      mx = fmaxf(mx, fmaxf(lo[j], hi[j]));
      bad = fmaf(lo[j], 0.f, fmaf(hi[j], 0.f, bad));  // 0, or NaN after an infinity or a NaN
    }
#pragma unroll
    for (int off = LPR / 2; off >= 1; off >>= 1) {
      mn = fminf(mn, __shfl_xor_sync(0xffffffffu, mn, off));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
      bad += __shfl_xor_sync(0xffffffffu, bad, off);
    }
    if (go) {
      const int which = h >= turned ? 1 : 0, kv_head = h - p.q_heads - which * p.kv.heads;
      const __half low_h = __float2half_rn(mn);
      const float low = __half2float(low_h);
      __half scale_h = __float2half_rn(__fdiv_rn(mx - low, 15.f));
      if (!(__half2float(scale_h) >= 5.9604644775390625e-8f)) scale_h = __ushort_as_half(1);
      if (bad != 0.f) scale_h = __ushort_as_half(0x7e00);  // the whole row reads back as NaN
      const float scale = __half2float(scale_h), inv = __frcp_rn(scale);
      const uint32_t w0 = codes4(lo, low, scale, inv) | (codes4(lo + 4, low, scale, inv) << 16);
      const uint32_t w1 = codes4(hi, low, scale, inv) | (codes4(hi + 4, low, scale, inv) << 16);
      const long long page = slot / p.kv.page_size;
      const int in_page = static_cast<int>(slot - page * p.kv.page_size), row = in_page % kKvBlock;
      uint8_t* blk = kv_block_ptr(p.kv, D, page, kv_head, in_page / kKvBlock);
      uint8_t* codes = blk + kv_codes_offset(D, which, row);
      *reinterpret_cast<uint32_t*>(codes + 4 * lane) = w0;
      *reinterpret_cast<uint32_t*>(codes + D / 4 + 4 * lane) = w1;
      if (lane == 0) *reinterpret_cast<__half2*>(blk + kv_params_offset(D, which, row)) = __halves2half2(scale_h, low_h);
    }
  }
}

struct ReadParams {
  KvPages kv;
  IndexArray slots;
  __half *k, *v;  // [T, heads, D] dense
  int* status;
  long long tokens;
};

// D/8 lanes take a row, eight channels each: a 4-byte load of codes becomes one 16-byte store, so that a warp's stores
// cover whole rows of the output, which is nine tenths of the traffic.  blockIdx.y picks HPT consecutive heads; neighbouring
// lane groups take neighbouring tokens, whose rows lie side by side in a block.
template <int D, int HPT>
__global__ void __launch_bounds__(kKvThreads) fg_kv_read_kernel(const ReadParams p) {
  constexpr int LPR = D / 8;
  const int lane = threadIdx.x % LPR;
  const long long token = static_cast<long long>(blockIdx.x) * (kKvThreads / LPR) + threadIdx.x / LPR;
  const int head0 = blockIdx.y * HPT;
  griddep_wait();  // (no early launch of the next kernel: these rows may be what a linear takes for its weight, which it reads at once)
  if (token >= p.tokens) return;
  const long long slot = p.slots[token];
  if (slot < 0) return;
  if (slot >= p.kv.pages * p.kv.page_size) {
    if (lane == 0 && p.status != nullptr) atomicExch(p.status, kStatusIndex);
    return;
  }
  const long long page = slot / p.kv.page_size;
  const int in_page = static_cast<int>(slot - page * p.kv.page_size);
  const int row = in_page % kKvBlock;
  uint32_t w[HPT][2];
  __half2 par[HPT][2];
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (head0 + i < p.kv.heads) {
      const uint8_t* blk = kv_block_ptr(p.kv, D, page, head0 + i, in_page / kKvBlock);
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        w[i][which] = *reinterpret_cast<const uint32_t*>(blk + kv_codes_offset(D, which, row) + 4 * lane);
        par[i][which] = *reinterpret_cast<const __half2*>(blk + kv_params_offset(D, which, row));
      }
    }
#pragma unroll
  for (int i = 0; i < HPT; ++i)
    if (head0 + i < p.kv.heads) {
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        const float scale = __low2float(par[i][which]), low = __high2float(par[i][which]);
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          // at the ends of fp16's range the rounded scale may carry the top code past 65504: it saturates (NaN stays NaN)
          const float f = fmaf(static_cast<float>((w[i][which] >> (4 * j)) & 15u), scale, low);
          v[j] = f > 65504.f ? 65504.f : f;
        }
        __half* dst = (which ? p.v : p.k) + (token * p.kv.heads + head0 + i) * D + 8 * lane;
        *reinterpret_cast<uint4*>(dst) = pack8(v);
      }
    }
}

int check_pages(const void* pages, long long num_pages, int heads, int page_size, int d) {
  if (pages == nullptr) return FG_ERR_NULL;
  if ((d != 64 && d != 128) || num_pages < 1 || heads < 1 || page_size < kKvBlock || (page_size % kKvBlock) != 0) return FG_ERR_SHAPE;
  if (!host::aligned(pages, 16)) return FG_ERR_ALIGN;
  return FG_OK;
}

}  // namespace
}  // namespace fg

extern "C" int fg_kv_append_int4(const void* k, long long ldk, const void* v, long long ldv, long long tokens, int kv_heads,
                                 int d, void* pages, long long num_pages, int page_size, const void* slots, int slots_64,
                                 const float* cos_sin, long long positions_len, const void* positions, int positions_64,
                                 const void* q, long long ldq, void* q_out, long long ldqo, int q_heads, int interleaved,
                                 int* status_dev, fg_stream_t stream) {
  using namespace fg;
  int st = check_pages(pages, num_pages, kv_heads, page_size, d);
  if (st != FG_OK) return st;
  if (k == nullptr || v == nullptr || slots == nullptr) return FG_ERR_NULL;
  if ((q == nullptr) != (q_out == nullptr) || (cos_sin == nullptr) != (positions == nullptr)) return FG_ERR_NULL;
  if (q != nullptr && cos_sin == nullptr) return FG_ERR_NULL;
  if (tokens < 1 || (q != nullptr) != (q_heads > 0) || q_heads < 0 || q_heads > 16384 || kv_heads > 16384) return FG_ERR_SHAPE;
  if (cos_sin != nullptr && positions_len < 1) return FG_ERR_SHAPE;
  if (ldk < static_cast<long long>(kv_heads) * d || ldv < static_cast<long long>(kv_heads) * d || (ldk % 8) != 0 || (ldv % 8) != 0)
    return FG_ERR_SHAPE;
  if (q != nullptr && (ldq < static_cast<long long>(q_heads) * d || ldqo < static_cast<long long>(q_heads) * d || (ldq % 8) != 0 || (ldqo % 8) != 0))
    return FG_ERR_SHAPE;
  if (!host::aligned(k, 16) || !host::aligned(v, 16) || !host::aligned(q, 16) || !host::aligned(q_out, 16) || !host::aligned(cos_sin, 16) ||
      !host::aligned(slots, slots_64 ? 8 : 4) || !host::aligned(positions, positions_64 ? 8 : 4) || !host::aligned(status_dev, 4))
    return FG_ERR_ALIGN;
  host::Device dev;
  if ((st = host::current_device(&dev)) != FG_OK) return st;
  AppendParams p = {};
  p.q = static_cast<const __half*>(q);
  p.k = static_cast<const __half*>(k);
  p.v = static_cast<const __half*>(v);
  p.ldq = ldq;
  p.ldk = ldk;
  p.ldv = ldv;
  p.q_out = static_cast<__half*>(q_out);
  p.ldqo = ldqo;
  p.q_heads = q_heads;
  p.cos_sin = cos_sin;
  p.positions_len = positions_len;
  p.positions = {positions, positions_64};
  p.slots = {slots, slots_64};
  p.interleaved = interleaved;
  p.kv = {static_cast<uint8_t*>(pages), num_pages, kv_heads, page_size};
  p.status = status_dev;
  p.tokens = tokens;
  // Few rows: one a lane group, for latency; enough rows for four CTAs' worth a SM with four: four (6001 tokens of 48 heads of
  // 64 channels: 16.6 us, with one 21.6; 64 tokens: 2.3 us, with four 4.7).
  const long long heads = q_heads + 2LL * kv_heads, rows_per_cta = kKvThreads / (d / 16);
  const bool many = tokens * heads >= 4 * 8 * rows_per_cta * dev.sm_count;
  const long long gx = (tokens + rows_per_cta - 1) / rows_per_cta, gy = (heads + (many ? 3 : 0)) / (many ? 4 : 1);
  if (gx > 0x7fffffffLL || gy > 65535) return FG_ERR_SHAPE;
  void (*kern)(const AppendParams) = d == 128 ? (many ? fg_kv_append_kernel<128, 4> : fg_kv_append_kernel<128, 1>)
                                              : (many ? fg_kv_append_kernel<64, 4> : fg_kv_append_kernel<64, 1>);
  return host::launch(kern, dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), dim3(kKvThreads), 0,
                      reinterpret_cast<cudaStream_t>(stream), true, p);
}

extern "C" int fg_kv_read_int4(const void* pages, long long num_pages, int page_size, int kv_heads, int d, const void* slots,
                               int slots_64, long long tokens, void* k_out, void* v_out, int* status_dev, fg_stream_t stream) {
  using namespace fg;
  int st = check_pages(pages, num_pages, kv_heads, page_size, d);
  if (st != FG_OK) return st;
  if (slots == nullptr || k_out == nullptr || v_out == nullptr) return FG_ERR_NULL;
  if (tokens < 1 || kv_heads > 16384) return FG_ERR_SHAPE;
  if (!host::aligned(k_out, 16) || !host::aligned(v_out, 16) || !host::aligned(slots, slots_64 ? 8 : 4) || !host::aligned(status_dev, 4))
    return FG_ERR_ALIGN;
  host::Device dev;
  if ((st = host::current_device(&dev)) != FG_OK) return st;
  ReadParams p = {};
  p.kv = {const_cast<uint8_t*>(static_cast<const uint8_t*>(pages)), num_pages, kv_heads, page_size};
  p.slots = {slots, slots_64};
  p.k = static_cast<__half*>(k_out);
  p.v = static_cast<__half*>(v_out);
  p.status = status_dev;
  p.tokens = tokens;
  const long long rows_per_cta = kKvThreads / (d / 8), gx = (tokens + rows_per_cta - 1) / rows_per_cta;
  const bool many = tokens * kv_heads >= 4 * 16 * rows_per_cta * dev.sm_count;  // 40000 rows: 38 us, with one head a thread 47
  const long long gy = (kv_heads + (many ? 3 : 0)) / (many ? 4 : 1);
  if (gx > 0x7fffffffLL || gy > 65535) return FG_ERR_SHAPE;
  void (*kern)(const ReadParams) = d == 128 ? (many ? fg_kv_read_kernel<128, 4> : fg_kv_read_kernel<128, 1>)
                                            : (many ? fg_kv_read_kernel<64, 4> : fg_kv_read_kernel<64, 1>);
  return host::launch(kern, dim3(static_cast<unsigned>(gx), static_cast<unsigned>(gy)), dim3(kKvThreads), 0,
                      reinterpret_cast<cudaStream_t>(stream), true, p);
}

// Layout of the paged key/value cache held in 4 bits, shared by its three kernels.
//
// A page holds `page_size` rows (a multiple of 16) of every key/value head.  Inside a page a head's rows lie in
// blocks of 16, each one contiguous piece that a single bulk copy brings in:
//
//   [16][D/2] key codes | [16][D/2] value codes | [16] key parameters | [16] value parameters
//
// 16 (D + 8) bytes in all.  Codes: two per byte, low nibble = even channel (the packing of fg_quantize_rows_w4);
// parameters: a (scale, low) pair of fp16; a stored row is low + scale * code.
#pragma once
#include <cuda_fp16.h>
#include <stdint.h>

#include "fg_ptx.cuh"

namespace fg {

constexpr int kKvBlock = 16;  // rows of a block
__host__ __device__ constexpr int kv_block_bytes(int d) { return kKvBlock * (d + 8); }
__host__ __device__ constexpr int kv_codes_offset(int d, int which, int row) { return (which * kKvBlock + row) * (d / 2); }
__host__ __device__ constexpr int kv_params_offset(int d, int which, int row) {
  return kKvBlock * d + (which * kKvBlock + row) * 4;
}

struct KvPages {
  uint8_t* base;
  long long pages;
  int heads;      // key/value heads
  int page_size;  // rows of a page, a multiple of 16
};

// Block `block` (of 16 rows) of head `head` in page `page`.
__device__ __forceinline__ uint8_t* kv_block_ptr(const KvPages& kv, int d, long long page, int head, int block) {
  return kv.base + ((page * kv.heads + head) * (kv.page_size / kKvBlock) + block) * kv_block_bytes(d);
}

// A device array of 32- or 64-bit indices.
struct IndexArray {
  const void* p;
  int is64;
  __device__ __forceinline__ long long operator[](long long i) const {
    return is64 ? static_cast<const long long*>(p)[i] : static_cast<long long>(static_cast<const int*>(p)[i]);
  }
};

constexpr int kStatusIndex = 9;  // FG_ERR_INDEX

}  // namespace fg

// kv_mx4.h - the KV cache held in 4 bits (OCP MXFP4): its layout, shared by
// kv_mx4_cache.hip (quantising, reading back) and kv_mx4_attention.hip, and
// the host checks both make.  Not installed; not part of the C ABI.
//
// A chunk (the tokens of one block of one half of one layer, T tokens, H
// heads, D elements a head) is
//   [head][token][D / 2]     code bytes, element 2i in the low half of byte i
//   [head][D / 32][token]    scale bytes, one for 32 neighbouring elements
// so a head's codes and scales of a block are two contiguous runs: attention
// reads a head's tokens as whole cache lines, and the scales of neighbouring
// tokens are one load.  T is a multiple of 16, so a chunk is a multiple of 272
// bytes and a 16-token tile lies within one block.
//
// Element code c = sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3,
// 4, 6 and their negatives.  Scale byte b stands for 2^(b - 127), 255 for NaN.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv_device.h"
#include "kv_internal.h"

namespace fkv_detail {
#pragma GCC visibility push(hidden)

constexpr int kMx4Group = 32;        // elements that share a scale
constexpr int kMx4TokenTile = 16;    // tokens_per_block is a multiple of this
constexpr int kMx4MaxTokens = 4096;  // tokens_per_block at most
constexpr int kMx4MaxHeads = 1024;
constexpr int kMx4MaxHeadSize = 1024;

inline int64_t mx4_chunk_bytes(int64_t tokens, int64_t heads, int64_t dim) {
  return tokens * heads * (dim / kMx4Group) * 17;
}

// tokens_per_block, num_heads, head_size of a 4-bit cache
inline int mx4_check_shape(int tokens, int heads, int dim) {
  if (tokens < kMx4TokenTile || tokens > kMx4MaxTokens || tokens % kMx4TokenTile)
    return fail(kInval, "tokens_per_block must be a multiple of %d up to %d in a 4-bit cache, "
                "got %d", kMx4TokenTile, kMx4MaxTokens, tokens);
  if (heads < 1 || heads > kMx4MaxHeads)
    return fail(kInval, "num_heads must be in [1, %d], got %d", kMx4MaxHeads, heads);
  if (dim < kMx4Group || dim > kMx4MaxHeadSize || dim % kMx4Group)
    return fail(kInval, "head_size must be a multiple of %d up to %d in a 4-bit cache, got %d",
                kMx4Group, kMx4MaxHeadSize, dim);
  return 0;
}

inline int64_t dtype_bytes(int dtype) { return dtype == FKV_DTYPE_FP32 ? 4 : 2; }

inline int mx4_check_dtype(int dtype) {
  if (dtype < FKV_DTYPE_BF16 || dtype > FKV_DTYPE_FP32)
    return fail(kInval, "dtype must be FKV_DTYPE_BF16, _FP16 or _FP32, got %d", dtype);
  return 0;
}

// One layer of a 4-bit cache on the device: half k of block b at
// ptr + k * kv_stride + b * block_stride.  Every block lies inside the
// allocation of ptr.
inline int mx4_check_layer(const void* ptr, int64_t kv_stride, int64_t block_stride,
                           int64_t num_blocks, int halves, int64_t chunk) {
  if (!ptr) return fail(kInval, "null 4-bit cache pointer");
  if (num_blocks < 1 || num_blocks > INT32_MAX)
    return fail(kInval, "num_mx_blocks must be in [1, 2^31), got %lld", (long long)num_blocks);
  if (kv_stride < 0 || block_stride < 0 || kv_stride % 16 || block_stride % 16 ||
      reinterpret_cast<uintptr_t>(ptr) % 16)
    return fail(kInval, "the 4-bit cache's pointer and strides must be non-negative multiples of "
                "16 bytes (kv %lld, block %lld)", (long long)kv_stride, (long long)block_stride);
  PtrInfo info;
  if (query_ptr(ptr, &info) != 0 || !info.device)
    return fail(kInval, "the 4-bit cache %p is not device memory", ptr);
  const __int128 hi = static_cast<__int128>(halves - 1) * kv_stride +
                      static_cast<__int128>(num_blocks - 1) * block_stride + chunk;
  if (!range_inside(static_cast<const char*>(ptr), 0, hi, info))
    return fail(kInval, "%lld blocks of the 4-bit cache reach outside its allocation (%zu bytes)",
                (long long)num_blocks, info.size);
  return 0;
}

#pragma GCC visibility pop
}  // namespace fkv_detail

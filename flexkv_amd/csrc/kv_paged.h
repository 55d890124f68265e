// kv_paged.h - one layer of a paged KV cache as the operators on it take it (fkv_paged_layer),
// shared by kv_paged_cache.hip and kv_paged_attention.hip: the host checks, and where a
// token's row lies.  Not installed; not part of the C ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv_device.h"
#include "kv_internal.h"
#include "kv_overlap.h"

namespace fkv_detail {
#pragma GCC visibility push(hidden)

inline int64_t paged_element_bytes(int dtype) { return dtype == FKV_DTYPE_FP32 ? 4 : 2; }

inline int paged_check_sizes(const fkv_paged_layer& c) {
  if (c.tokens_per_block < 1 || c.tokens_per_block > (1 << 20))
    return fail(kInval, "tokens_per_block must be in [1, 2^20], got %d", c.tokens_per_block);
  if (c.num_heads < 1 || c.num_heads > 1024)
    return fail(kInval, "num_heads must be in [1, 1024], got %d", c.num_heads);
  if (c.dtype < FKV_DTYPE_BF16 || c.dtype > FKV_DTYPE_FP32)
    return fail(kInval, "dtype must be FKV_DTYPE_BF16, _FP16 or _FP32, got %d", c.dtype);
  if (c.head_size < 1 || c.head_size > 1024 || c.head_size * paged_element_bytes(c.dtype) % 16)
    return fail(kInval, "head_size must be a multiple of 16 bytes up to 1024 elements, got %d",
                c.head_size);
  if (c.num_blocks < 1 || c.num_blocks > INT32_MAX)
    return fail(kInval, "num_blocks must be in [1, 2^31), got %lld", (long long)c.num_blocks);
  return 0;
}

// Every row of every block lies inside the allocation of its pointer.  A null `value` is a
// cache of one half.
inline int paged_check_layer(const fkv_paged_layer& c) {
  int rc;
  if ((rc = paged_check_sizes(c))) return rc;
  const char* const p[2] = {static_cast<const char*>(c.key), static_cast<const char*>(c.value)};
  const int64_t s[2][3] = {{c.key_block_stride_bytes, c.key_token_stride_bytes,
                            c.key_head_stride_bytes},
                           {c.value_block_stride_bytes, c.value_token_stride_bytes,
                            c.value_head_stride_bytes}};
  if (!p[0]) return fail(kInval, "null cache pointer");
  const int halves = p[1] ? 2 : 1;
  auto name_of = [](int k) { return k ? "value" : "key"; };
  for (int k = 0; k < halves; ++k) {
    const char* const name = name_of(k);
    for (int64_t v : s[k])
      if (v < 0 || v % 16)
        return fail(kInval, "the %s cache's strides must be non-negative multiples of 16 bytes "
                    "(block %lld, token %lld, head %lld)", name, (long long)s[k][0],
                    (long long)s[k][1], (long long)s[k][2]);
    if (reinterpret_cast<uintptr_t>(p[k]) % 16)
      return fail(kInval, "the %s cache's pointer must be a multiple of 16 bytes", name);
  }
  PtrInfo info;
  for (int k = 0; k < halves; ++k) {
    const char* const name = name_of(k);
    const __int128 hi = static_cast<__int128>(c.num_blocks - 1) * s[k][0] +
                        static_cast<__int128>(c.tokens_per_block - 1) * s[k][1] +
                        static_cast<__int128>(c.num_heads - 1) * s[k][2] +
                        c.head_size * paged_element_bytes(c.dtype);
    // K and V are often views of one allocation
    if (k && info.device && range_inside(p[k], 0, hi, info)) continue;
    if (query_ptr(p[k], &info) != 0 || !info.device)
      return fail(kInval, "the %s cache %p is not device memory", name, (const void*)p[k]);
    if (!range_inside(p[k], 0, hi, info))
      return fail(kInval, "%lld blocks of the %s cache reach outside its allocation (%zu bytes)",
                  (long long)c.num_blocks, name, info.size);
  }
  return 0;
}

// Of a layer that is written to no two rows share memory: what two of them got would be a mixture.
inline int paged_check_written(const fkv_paged_layer& c) {
  const int64_t counts[3] = {c.num_blocks, c.tokens_per_block, c.num_heads};
  const int64_t bytes = c.head_size * paged_element_bytes(c.dtype);
  const RowSet k(c.key, bytes,
                 {c.key_block_stride_bytes, c.key_token_stride_bytes, c.key_head_stride_bytes},
                 counts);
  if (!rows_apart(k)) return fail(kInval, "rows of the key cache overlap");
  if (!c.value) return 0;
  const RowSet v(c.value, bytes,
                 {c.value_block_stride_bytes, c.value_token_stride_bytes,
                  c.value_head_stride_bytes},
                 counts);
  if (!rows_apart(v)) return fail(kInval, "rows of the value cache overlap");
  if (rows_meet(k, v)) return fail(kInval, "the key and value caches overlap");
  return 0;
}

// One half of a layer.
struct Half {
  char* p;
  int64_t block, token, head;     // strides in bytes
};
inline Half key_half(const fkv_paged_layer& c) {
  return {static_cast<char*>(c.key), c.key_block_stride_bytes, c.key_token_stride_bytes,
          c.key_head_stride_bytes};
}
inline Half value_half(const fkv_paged_layer& c) {
  return {static_cast<char*>(c.value), c.value_block_stride_bytes, c.value_token_stride_bytes,
          c.value_head_stride_bytes};
}

#pragma GCC visibility pop
}  // namespace fkv_detail

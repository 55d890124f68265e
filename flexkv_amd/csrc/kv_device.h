// kv_device.h - small pieces that the kernels with arithmetic share.  Not installed;
// not part of the C ABI.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace fkv_detail {
#pragma GCC visibility push(hidden)

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 as one wide multiplication.
struct FastDiv {
  uint32_t d = 1, mul = 1u << 31, shift = 31;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(div) {
    uint32_t s = 0;
    while ((uint64_t(1) << s) < div) ++s;
    mul = static_cast<uint32_t>(((uint64_t(1) << (31 + s)) + div - 1) / div);
    shift = 31 + s;
  }
  __host__ __device__ uint32_t div(uint32_t n) const {
    return static_cast<uint32_t>((static_cast<uint64_t>(n) * mul) >> shift);
  }
};

__device__ inline float bits_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ inline uint32_t f32_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
__device__ inline uint32_t pack_bf16(float a, float b) {
  v2bf r;
  r[0] = static_cast<__bf16>(a);
  r[1] = static_cast<__bf16>(b);
  return __builtin_bit_cast(uint32_t, r);
}

#pragma GCC visibility pop
}  // namespace fkv_detail

// kv_mx4_cache.hip - quantising the KV cache to 4 bits and reading it back
// (layout and format in kv_mx4.h).
//
// A group x[0..31] of a row with a = max |x| gets the scale s = 2^(E - 2),
// E = floor(log2 a), one more where a's mantissa is over 1.75 (those would round
// past 6, the largest element, to 8); element i becomes the nearest of 0, 0.5, 1,
// 1.5, 2, 3, 4, 6 to |x_i| / s with its sign, ties to the even code.  Dividing by
// a power of two is exact, so a code is one rounding of the input and every
// element is within s of it.  E is at most 127 (biased 254), where elements over 7 s
// saturate at 6 s, and s at least 2^-127.  A group that holds an infinity or a
// NaN gets scale byte 255 and reads back as NaN.
//
// Both directions move bytes: 2 (4 for fp32) and 17/32 bytes an element, no
// reuse, a handful of operations each (gfx950 rounds two elements to 4 bits in
// one instruction), so memory bounds them.  Four neighbouring lanes hold a
// group, 8 elements each, of every fourth of 16 tokens: 16-byte accesses on the wide
// side, a dword of codes on the narrow one, where neighbouring quads' tokens and so
// their bytes are neighbours, a scale byte a lane, and two swaps within the quad for
// the group's maximum.  With four tokens in a row to a quad the pieces were 64 bytes,
// which the link to a pinned 4-bit cache minds: 128 blocks of Llama-3-8B's shape to
// it 1320 us for 1800 (54 GB/s of the link's 57), and from it 1260 for 1440; a latent
// of 576 elements 1160 for 1015 and 885 for 965.  On the device both measured alike.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <cstring>
#include <exception>

#include "kv_mx4.h"

using namespace fkv_detail;

namespace {

constexpr int kThreads = 256;
constexpr int kTokensPerUnit = 4;     // tokens whose group one quad of lanes handles, as many apart
constexpr int kInlinePairs = 256;     // id pairs in the kernel arguments
constexpr int64_t kUnitsPerLaunch = int64_t(1) << 28;

struct Bf16 {};
struct Fp16 {};
struct Fp32 {};
template <class T>
constexpr int kBytes = 2;
template <>
constexpr int kBytes<Fp32> = 4;

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

__device__ inline float bits_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ inline uint32_t f32_bits(float f) { return __builtin_bit_cast(uint32_t, f); }

// 8 neighbouring elements as they lie in memory
template <class T>
struct Raw {
  uint4 v;
};
template <>
struct Raw<Fp32> {
  uint4 v, w;
};
template <class T>
__device__ inline Raw<T> load_raw(const char* p) {
  Raw<T> r;
  r.v = *reinterpret_cast<const uint4*>(p);
  if constexpr (kBytes<T> == 4) r.w = *reinterpret_cast<const uint4*>(p + 16);
  return r;
}
// Blocks pass through once, so they are not to displace what the caches hold: MI355X,
// 1024 blocks of 2 MB each way 1024 us for 1072 with plain accesses, 173 blocks of 0.7 MB
// read back 24 for 29.  (New tokens, just computed, are read from the caches: 8191 of
// them 12.5 us, 16 by this.)
__device__ inline uint4 load_once(const char* p) {
  return __builtin_bit_cast(uint4, __builtin_nontemporal_load(reinterpret_cast<const v4u*>(p)));
}
__device__ inline void store_once(char* p, const uint4& v) {
  __builtin_nontemporal_store(__builtin_bit_cast(v4u, v), reinterpret_cast<v4u*>(p));
}
template <class T>
__device__ inline Raw<T> load_raw_once(const char* p) {
  Raw<T> r;
  r.v = load_once(p);
  if constexpr (kBytes<T> == 4) r.w = load_once(p + 16);
  return r;
}
template <class T>
__device__ inline void store_raw_once(char* p, const Raw<T>& r) {
  store_once(p, r.v);
  if constexpr (kBytes<T> == 4) store_once(p + 16, r.w);
}

__device__ inline void widen(const Raw<Bf16>& r, float (&x)[8]) {
  const uint32_t u[4] = {r.v.x, r.v.y, r.v.z, r.v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = bits_f32(u[i] << 16);
    x[2 * i + 1] = bits_f32(u[i] & 0xffff0000u);
  }
}
__device__ inline void widen(const Raw<Fp16>& r, float (&x)[8]) {
  const v8h h = __builtin_bit_cast(v8h, r.v);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(h[i]);
}
__device__ inline void widen(const Raw<Fp32>& r, float (&x)[8]) {
  const uint32_t u[8] = {r.v.x, r.v.y, r.v.z, r.v.w, r.w.x, r.w.y, r.w.z, r.w.w};
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = bits_f32(u[i]);
}

// A group's scale byte and this lane's 8 codes; the 4 lanes of an aligned
// quad hold the group.
__device__ inline uint32_t encode(const float (&x)[8], uint32_t* scale_byte) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, f32_bits(x[i]) & 0x7fffffffu);
  a = max(a, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(a, 0xB1, 0xf, 0xf, true)));
  a = max(a, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(a, 0x4E, 0xf, 0xf, true)));
  // as integers the magnitudes are ordered, NaN above infinity above the rest;
  // the addition carries into the exponent where the mantissa is over 1.75
  const uint32_t e = max(min((a + 0x1fffffu) >> 23, 254u), 2u) - 2u;
  const float s = bits_f32(e << 23);     // the conversions read the exponent alone: 0 is 2^-127
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[0], x[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[2], x[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[4], x[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, x[6], x[7], s, 3);
  const bool lost = a >= 0x7f800000u;
  *scale_byte = lost ? 255u : e;
  return lost ? 0u : c;
}

// 8 codes and their scale byte as values; one beyond the type's largest
// finite value is that value.
template <class T>
__device__ inline Raw<T> decode(uint32_t c, uint32_t scale_byte) {
  const float s = bits_f32(scale_byte << 23);
  const v2f p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0),
                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1),
                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2),
                    __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3)};
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = p[i / 2][i & 1];
  if (scale_byte == 255) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = bits_f32(0x7fc00000u);
  }
  Raw<T> r;
  if constexpr (kBytes<T> == 4) {
    uint32_t u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u[i] = f32_bits(x[i]);
      if ((u[i] & 0x7fffffffu) == 0x7f800000u) u[i] -= 1;
    }
    r.v = make_uint4(u[0], u[1], u[2], u[3]);
    r.w = make_uint4(u[4], u[5], u[6], u[7]);
  } else if constexpr (__is_same(T, Bf16)) {
    // two significant bits: bf16 holds every value but those past its largest
    uint32_t u[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t lo = f32_bits(x[2 * i]), hi = f32_bits(x[2 * i + 1]);
      if ((lo & 0x7fffffffu) == 0x7f800000u) lo -= 0x10000u;
      if ((hi & 0x7fffffffu) == 0x7f800000u) hi -= 0x10000u;
      u[i] = (lo >> 16) | (hi & 0xffff0000u);
    }
    r.v = make_uint4(u[0], u[1], u[2], u[3]);
  } else {
    v8h h;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      // a comparison, so that a NaN stays one
      const float m = x[i] > 65504.f ? 65504.f : x[i] < -65504.f ? -65504.f : x[i];
      h[i] = static_cast<_Float16>(m);
    }
    r.v = __builtin_bit_cast(uint4, h);
  }
  return r;
}

struct BlockArgs {
  char* mx;                 // 4-bit cache at the launch's first layer
  int64_t gks, gbs;         // wide cache: half and block strides
  int64_t mks, mls, mbs;    // 4-bit cache: half, layer and block strides
  const int64_t* pairs;     // null: inline_pairs; else (gpu id, 4-bit id) on the device
  uint32_t units;           // of the launch
  int halves_log2;          // 1 for K and V, 0 for one latent half
  int heads, tokens, dim;
  FastDiv per_chunk, per_head, groups, layers;
  uint64_t layer_ptrs[kMaxLayersPerLaunch];
  int32_t inline_pairs[2 * kInlinePairs];
};

// The addresses of unit `u`'s group: `wide` its elements of the first of its four
// tokens, `codes` and `scales` (a token's a byte apart).
struct Unit {
  char* wide;
  char* codes;
  char* scales;
};
template <class T>
__device__ inline Unit locate(const BlockArgs& a, uint32_t u) {
  const uint32_t c = a.per_chunk.div(u), r = u - c * a.per_chunk.d;
  const uint32_t h = a.per_head.div(r), r2 = r - h * a.per_head.d;
  const uint32_t t = a.groups.div(r2), g = r2 - t * a.groups.d;
  const uint32_t k = a.halves_log2 ? c & 1 : 0, bl = c >> a.halves_log2;
  const uint32_t i = a.layers.div(bl), l = bl - i * a.layers.d;
  int64_t gid, mid;
  if (a.pairs) {
    gid = a.pairs[2 * i], mid = a.pairs[2 * i + 1];
  } else {
    gid = a.inline_pairs[2 * i], mid = a.inline_pairs[2 * i + 1];
  }
  char* const chunk = a.mx + l * a.mls + k * a.mks + mid * a.mbs;
  const uint32_t tok = t / 4 * 16 + t % 4;
  Unit at;
  at.wide = reinterpret_cast<char*>(a.layer_ptrs[l]) + k * a.gks + gid * a.gbs +
            (static_cast<int64_t>(tok * a.heads + h) * a.dim + kMx4Group * g) * kBytes<T>;
  at.codes = chunk + static_cast<int64_t>(h * a.tokens + tok) * (a.dim / 2) + 16 * g;
  at.scales = chunk + static_cast<int64_t>(a.heads) * a.tokens * (a.dim / 2) +
              static_cast<int64_t>(h * a.groups.d + g) * a.tokens + tok;
  return at;
}

template <class T, bool to_mx>
__global__ __launch_bounds__(kThreads) void mx4_blocks_kernel(const BlockArgs a) {
  const uint32_t thread = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t u = thread / 4, s = thread % 4;
  if (u >= a.units) return;    // whole quads at a time
  const Unit at = locate<T>(a, u);
  const int64_t wide_step = static_cast<int64_t>(a.heads) * a.dim * kBytes<T> * kTokensPerUnit;
  const int64_t code_step = a.dim / 2 * kTokensPerUnit;
  char* const wide = at.wide + 8 * s * kBytes<T>;
  char* const codes = at.codes + 4 * s;
  if constexpr (to_mx) {
    Raw<T> raw[kTokensPerUnit];
#pragma unroll
    for (int j = 0; j < kTokensPerUnit; ++j) raw[j] = load_raw_once<T>(wide + j * wide_step);
    uint32_t scale = 0;      // of token s of the four
#pragma unroll
    for (int j = 0; j < kTokensPerUnit; ++j) {
      float x[8];
      widen(raw[j], x);
      uint32_t b;
      const uint32_t c = encode(x, &b);
      __builtin_nontemporal_store(c, reinterpret_cast<uint32_t*>(codes + j * code_step));
      if (s == j) scale = b;
    }
    *reinterpret_cast<uint8_t*>(at.scales + kTokensPerUnit * s) = static_cast<uint8_t>(scale);
  } else {
    uint32_t c[kTokensPerUnit];
#pragma unroll
    for (int j = 0; j < kTokensPerUnit; ++j)
      c[j] = *reinterpret_cast<const uint32_t*>(codes + j * code_step);
    const int scale = *reinterpret_cast<const uint8_t*>(at.scales + kTokensPerUnit * s);
    const int scales[kTokensPerUnit] = {
        __builtin_amdgcn_mov_dpp(scale, 0x00, 0xf, 0xf, true),    // of the quad's lane 0 to 3
        __builtin_amdgcn_mov_dpp(scale, 0x55, 0xf, 0xf, true),
        __builtin_amdgcn_mov_dpp(scale, 0xAA, 0xf, 0xf, true),
        __builtin_amdgcn_mov_dpp(scale, 0xFF, 0xf, 0xf, true)};
#pragma unroll
    for (int j = 0; j < kTokensPerUnit; ++j)
      store_raw_once<T>(wide + j * wide_step, decode<T>(c[j], static_cast<uint32_t>(scales[j])));
  }
}

// The id pairs from the pinned buffer to device memory, so that the
// workgroups do not read them across the host link.
__global__ __launch_bounds__(kThreads) void mx4_pairs_kernel(const int64_t* in, int64_t* out,
                                                             int n) {
  const int i = blockIdx.x * kThreads + static_cast<int>(threadIdx.x);
  if (i < n) out[i] = in[i];
}

struct TokenArgs {
  const char* rows[2];      // K, V
  int64_t token_stride[2], head_stride[2];
  char* mx;
  int64_t mks, mbs;
  const void* slots;
  int64_t num_slots;        // of the cache
  uint32_t units;
  int heads, tokens, dim, slots64;
  FastDiv per_half, per_token, groups;
};

// New tokens into their slots: a quad of lanes takes one group of one row.
template <class T>
__global__ __launch_bounds__(kThreads) void mx4_tokens_kernel(const TokenArgs a) {
  const uint32_t thread = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t u = thread / 4, s = thread % 4;
  if (u >= a.units) return;
  const uint32_t k = a.per_half.div(u), r = u - k * a.per_half.d;
  const uint32_t n = a.per_token.div(r), r2 = r - n * a.per_token.d;
  const uint32_t h = a.groups.div(r2), g = r2 - h * a.groups.d;
  const int64_t slot = a.slots64 ? static_cast<const int64_t*>(a.slots)[n]
                                 : static_cast<const int32_t*>(a.slots)[n];
  if (slot < 0 || slot >= a.num_slots) return;    // uniform in the quad: padding
  const int64_t block = slot / a.tokens;
  const int64_t t = slot - block * a.tokens;
  float x[8];
  widen(load_raw<T>(a.rows[k] + n * a.token_stride[k] + h * a.head_stride[k] +
                    (kMx4Group * g + 8 * s) * kBytes<T>), x);
  uint32_t b;
  const uint32_t c = encode(x, &b);
  char* const chunk = a.mx + k * a.mks + block * a.mbs;
  *reinterpret_cast<uint32_t*>(chunk + (static_cast<int64_t>(h) * a.tokens + t) * (a.dim / 2) +
                               16 * g + 4 * s) = c;
  if (s == 0)
    *reinterpret_cast<uint8_t*>(chunk + static_cast<int64_t>(a.heads) * a.tokens * (a.dim / 2) +
                                (static_cast<int64_t>(h) * a.groups.d + g) * a.tokens + t) = b;
}

// ---------------------------------------------------------------------------
// Host side

struct BlockCall {
  int num_blocks, start_layer, num_layers, halves;
  const int64_t* gids;
  const int64_t* mids;
  void* const* layer_ptrs;
  int64_t gks, gbs, mks, mls, mbs;
  char* mx;
  PtrInfo mx_info;
  int tokens, heads, dim, dtype;
  bool wide_ids;       // some id needs 64 bits

  int64_t wide_chunk() const {
    return static_cast<int64_t>(tokens) * heads * dim * dtype_bytes(dtype);
  }
  int64_t mx_chunk() const { return mx4_chunk_bytes(tokens, heads, dim); }
};

int check_blocks(BlockCall& c) {
  if (c.num_blocks < 0 || c.num_layers < 0 || c.start_layer < 0)
    return fail(kInval, "negative count: num_blocks=%d num_layers=%d start_layer_id=%d",
                c.num_blocks, c.num_layers, c.start_layer);
  if (!c.gids || !c.mids || !c.layer_ptrs || !c.mx) return fail(kInval, "null pointer argument");
  int rc;
  if ((rc = mx4_check_shape(c.tokens, c.heads, c.dim)) || (rc = mx4_check_dtype(c.dtype)))
    return rc;
  const int64_t strides[] = {c.gks, c.gbs, c.mks, c.mls, c.mbs};
  for (int64_t v : strides)
    if (v < 0 || v % 16)
      return fail(kInval, "strides must be non-negative multiples of 16 bytes (gkv=%lld gblk=%lld "
                  "mxkv=%lld mxlayer=%lld mxblk=%lld)", (long long)c.gks, (long long)c.gbs,
                  (long long)c.mks, (long long)c.mls, (long long)c.mbs);
  if (reinterpret_cast<uintptr_t>(c.mx) % 16) return fail(kInval, "mx_ptr is not 16-byte aligned");
  int64_t gmin = INT64_MAX, gmax = -1, mmin = INT64_MAX, mmax = -1;
  for (int i = 0; i < c.num_blocks; ++i) {
    const int64_t a = c.gids[i], b = c.mids[i];
    if (a < 0 || b < 0)
      return fail(kInval, "negative block id at position %d (gpu %lld, 4-bit %lld)", i,
                  (long long)a, (long long)b);
    gmin = std::min(gmin, a), gmax = std::max(gmax, a);
    mmin = std::min(mmin, b), mmax = std::max(mmax, b);
  }
  c.wide_ids = std::max(gmax, mmax) > INT32_MAX;
  if (query_ptr(c.mx, &c.mx_info) != 0)
    return fail(kInval, "mx_ptr %p is not pinned host or device memory known to HIP", c.mx);
  const __int128 lo = static_cast<__int128>(c.start_layer) * c.mls +
                      static_cast<__int128>(mmin) * c.mbs;
  const __int128 hi = static_cast<__int128>(c.start_layer + int64_t(c.num_layers) - 1) * c.mls +
                      static_cast<__int128>(c.halves - 1) * c.mks +
                      static_cast<__int128>(mmax) * c.mbs + c.mx_chunk();
  if (!range_inside(c.mx, lo, hi, c.mx_info))
    return fail(kInval, "4-bit block ids [%lld, %lld] with layers [%d, %lld) address bytes outside "
                "the 4-bit cache's allocation (%zu bytes)", (long long)mmin, (long long)mmax,
                c.start_layer, c.start_layer + (long long)c.num_layers, c.mx_info.size);
  const __int128 glo = static_cast<__int128>(gmin) * c.gbs;
  const __int128 ghi = static_cast<__int128>(c.halves - 1) * c.gks +
                       static_cast<__int128>(gmax) * c.gbs + c.wide_chunk();
  PtrInfo pi;
  for (int l = 0; l < c.num_layers; ++l) {
    const char* p = static_cast<const char*>(c.layer_ptrs[l]);
    if (!p) return fail(kInval, "gpu layer pointer %d is null", l);
    if (reinterpret_cast<uintptr_t>(p) % 16)
      return fail(kInval, "gpu layer pointer %d is not 16-byte aligned", l);
    if (!(pi.device && p >= pi.base && p < pi.base + pi.size)) {
      pi = PtrInfo();
      if (query_ptr(p, &pi) != 0) pi.device = false;
    }
    if (!pi.device)
      return fail(kInval, "gpu layer pointer %d (%p) is not device memory", l, p);
    if (!range_inside(p, glo, ghi, pi))
      return fail(kInval, "gpu block ids [%lld, %lld] address bytes outside the allocation of "
                  "layer pointer %d (%zu bytes)", (long long)gmin, (long long)gmax, l, pi.size);
  }
  return 0;
}

template <class T>
void launch_blocks(const BlockArgs& a, bool to_mx, hipStream_t s) {
  const dim3 grid((static_cast<int64_t>(a.units) * 4 + kThreads - 1) / kThreads);
  if (to_mx)
    hipLaunchKernelGGL((mx4_blocks_kernel<T, true>), grid, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((mx4_blocks_kernel<T, false>), grid, dim3(kThreads), 0, s, a);
}

int run_blocks(const BlockCall& c, hipStream_t s, int dev, bool to_mx) {
  IdLease host;          // before the drain: freed after it
  DevIdLease table;
  DrainOnError drain{s};
  ProfRecorder prof;
  hipEvent_t ev = nullptr;
  int rc;
  BlockArgs a;
  a.gks = c.gks, a.gbs = c.gbs, a.mks = c.mks, a.mls = c.mls, a.mbs = c.mbs;
  a.halves_log2 = c.halves - 1;
  a.heads = c.heads, a.tokens = c.tokens, a.dim = c.dim;
  const uint32_t groups = c.dim / kMx4Group;
  a.groups = FastDiv(groups);
  a.per_head = FastDiv(groups * (c.tokens / kTokensPerUnit));
  a.per_chunk = FastDiv(a.per_head.d * c.heads);
  (void)hipGetLastError();  // a stale error from elsewhere must not be blamed on these launches
  const int64_t* pairs = nullptr;
  if (c.num_blocks > kInlinePairs || c.wide_ids) {
    const size_t bytes = static_cast<size_t>(c.num_blocks) * 16;
    if ((rc = ids_acquire(bytes, &host.buf))) return rc;
    for (int i = 0; i < c.num_blocks; ++i) {
      host.buf.host[2 * i] = c.gids[i];
      host.buf.host[2 * i + 1] = c.mids[i];
    }
    table.dev = dev;
    if ((rc = dev_ids_acquire(dev, bytes, &table.buf))) return rc;
    int64_t* out = reinterpret_cast<int64_t*>(table.buf.dev);
    // at most 2^30 pairs fit the launch's int counts (num_blocks is an int)
    const int64_t n = 2 * static_cast<int64_t>(c.num_blocks);
    for (int64_t i = 0; i < n; i += int64_t(1) << 30) {
      const int part = static_cast<int>(std::min<int64_t>(n - i, int64_t(1) << 30));
      hipLaunchKernelGGL(mx4_pairs_kernel, dim3((part + kThreads - 1) / kThreads), dim3(kThreads),
                         0, s, reinterpret_cast<const int64_t*>(host.buf.dev) + i, out + i, part);
      FKV_HIP(hipGetLastError());
    }
    pairs = out;
  }
  const int64_t chunk_units = a.per_chunk.d;     // at most 2^25
  for (int l0 = 0; l0 < c.num_layers; l0 += kMaxLayersPerLaunch) {
    int nl = std::min(c.num_layers - l0, kMaxLayersPerLaunch);
    // windows of fewer layers where one block alone has too many units
    while (nl > 1 && chunk_units * c.halves * nl > kUnitsPerLaunch) nl = (nl + 1) / 2;
    for (int l1 = l0; l1 < std::min(l0 + kMaxLayersPerLaunch, c.num_layers); l1 += nl) {
      const int n = std::min({nl, l0 + kMaxLayersPerLaunch - l1, c.num_layers - l1});
      a.mx = c.mx_info.dev_ptr + static_cast<int64_t>(c.start_layer + l1) * c.mls;
      a.layers = FastDiv(n);
      for (int l = 0; l < n; ++l) a.layer_ptrs[l] = reinterpret_cast<uint64_t>(c.layer_ptrs[l1 + l]);
      const int64_t block_units = chunk_units * c.halves * n;
      const int64_t step = std::max<int64_t>(1, kUnitsPerLaunch / block_units);
      for (int64_t b = 0; b < c.num_blocks; b += step) {
        const int nb = static_cast<int>(std::min<int64_t>(step, c.num_blocks - b));
        a.units = static_cast<uint32_t>(block_units * nb);
        a.pairs = pairs ? pairs + 2 * b : nullptr;
        if (!pairs)
          for (int i = 0; i < nb; ++i) {
            a.inline_pairs[2 * i] = static_cast<int32_t>(c.gids[b + i]);
            a.inline_pairs[2 * i + 1] = static_cast<int32_t>(c.mids[b + i]);
          }
        if ((rc = prof.begin(s, &ev))) return rc;
        if (c.dtype == FKV_DTYPE_BF16) launch_blocks<Bf16>(a, to_mx, s);
        else if (c.dtype == FKV_DTYPE_FP16) launch_blocks<Fp16>(a, to_mx, s);
        else launch_blocks<Fp32>(a, to_mx, s);
        FKV_HIP(hipGetLastError());
        if ((rc = prof.end(s, ev, nb * c.halves * n * (c.wide_chunk() + c.mx_chunk()), 0, false)))
          return rc;
      }
    }
  }
  FKV_HIP(hipStreamSynchronize(s));
  drain.armed = false;
  prof.flush();
  return 0;
}

int blocks_entry(int num_blocks, int start_layer_id, int num_layers, const int64_t* gpu_block_ids,
                 void* const* gpu_layer_ptrs, int64_t gks, int64_t gbs,
                 const int64_t* mx_block_ids, void* mx_ptr, int64_t mks, int64_t mls, int64_t mbs,
                 int tokens, int heads, int dim, int dtype, fkv_stream_t stream, int is_mla,
                 bool to_mx) {
  try {
    last_error().clear();
    last_unsafe_host_blocks().clear();
    if (num_blocks == 0 || num_layers == 0) return 0;
    BlockCall c{num_blocks, start_layer_id, num_layers, is_mla ? 1 : 2, gpu_block_ids,
                mx_block_ids, gpu_layer_ptrs, gks, gbs, mks, mls, mbs,
                static_cast<char*>(mx_ptr), PtrInfo(), tokens, heads, dim, dtype, false};
    int rc = check_blocks(c);
    if (rc) return rc;
    hipStream_t s = static_cast<hipStream_t>(stream);
    // synchronous, and the ids are read on the host: a captured call could not replay
    hipStreamCaptureStatus cap = hipStreamCaptureStatusNone;
    if (s) FKV_HIP(hipStreamIsCapturing(s, &cap));
    if (cap != hipStreamCaptureStatusNone)
      return fail(static_cast<int>(hipErrorStreamCaptureUnsupported),
                  "blocks cannot be quantised or read back on a stream under HIP graph capture "
                  "(the call synchronises the stream and reads its ids on the host)");
    int dev = 0;
    DeviceGuard guard;
    if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
    return run_blocks(c, s, dev, to_mx);
  } catch (const std::exception& e) {
    return fail(static_cast<int>(hipErrorUnknown), "exception: %s", e.what());
  } catch (...) {
    return fail(static_cast<int>(hipErrorUnknown), "unknown exception");
  }
}

}  // namespace

extern "C" {

int fkv_quantize_kv_blocks(int num_blocks, int start_layer_id, int num_layers,
                           const int64_t* gpu_block_ids, void* const* gpu_layer_ptrs,
                           int64_t gpu_kv_stride_bytes, int64_t gpu_block_stride_bytes,
                           const int64_t* mx_block_ids, void* mx_ptr, int64_t mx_kv_stride_bytes,
                           int64_t mx_layer_stride_bytes, int64_t mx_block_stride_bytes,
                           int tokens_per_block, int num_heads, int head_size, int dtype,
                           fkv_stream_t stream, int is_mla) {
  return blocks_entry(num_blocks, start_layer_id, num_layers, gpu_block_ids, gpu_layer_ptrs,
                      gpu_kv_stride_bytes, gpu_block_stride_bytes, mx_block_ids, mx_ptr,
                      mx_kv_stride_bytes, mx_layer_stride_bytes, mx_block_stride_bytes,
                      tokens_per_block, num_heads, head_size, dtype, stream, is_mla, true);
}

int fkv_dequantize_kv_blocks(int num_blocks, int start_layer_id, int num_layers,
                             const int64_t* gpu_block_ids, void* const* gpu_layer_ptrs,
                             int64_t gpu_kv_stride_bytes, int64_t gpu_block_stride_bytes,
                             const int64_t* mx_block_ids, const void* mx_ptr,
                             int64_t mx_kv_stride_bytes, int64_t mx_layer_stride_bytes,
                             int64_t mx_block_stride_bytes, int tokens_per_block, int num_heads,
                             int head_size, int dtype, fkv_stream_t stream, int is_mla) {
  return blocks_entry(num_blocks, start_layer_id, num_layers, gpu_block_ids, gpu_layer_ptrs,
                      gpu_kv_stride_bytes, gpu_block_stride_bytes, mx_block_ids,
                      const_cast<void*>(mx_ptr), mx_kv_stride_bytes, mx_layer_stride_bytes,
                      mx_block_stride_bytes, tokens_per_block, num_heads, head_size, dtype, stream,
                      is_mla, false);
}

int fkv_quantize_kv_tokens(int num_tokens, const void* key, int64_t key_token_stride_bytes,
                           int64_t key_head_stride_bytes, const void* value,
                           int64_t value_token_stride_bytes, int64_t value_head_stride_bytes,
                           const void* slots, int slots_are_64bit, void* mx_ptr,
                           int64_t mx_kv_stride_bytes, int64_t mx_block_stride_bytes,
                           int64_t num_mx_blocks, int tokens_per_block, int num_heads,
                           int head_size, int dtype, fkv_stream_t stream) {
  try {
    last_error().clear();
    if (num_tokens < 0) return fail(kInval, "negative count: num_tokens=%d", num_tokens);
    const int halves = value ? 2 : 1;
    int rc;
    if ((rc = mx4_check_shape(tokens_per_block, num_heads, head_size)) ||
        (rc = mx4_check_dtype(dtype)))
      return rc;
    // less than 2^32 threads, in whole workgroups
    const int64_t groups = head_size / kMx4Group, per_token = groups * num_heads;
    if (per_token * num_tokens * halves > (int64_t(1) << 30) - kThreads / 4)
      return fail(kInval, "%d tokens of %d heads of %d are too many for one call", num_tokens,
                  num_heads, head_size);
    if ((rc = mx4_check_layer(mx_ptr, mx_kv_stride_bytes, mx_block_stride_bytes, num_mx_blocks,
                              halves, mx4_chunk_bytes(tokens_per_block, num_heads, head_size))))
      return rc;
    if (num_tokens == 0) return 0;
    if (!key || !slots) return fail(kInval, "null pointer argument");
    TokenArgs a;
    a.rows[0] = static_cast<const char*>(key);
    a.rows[1] = static_cast<const char*>(value);
    a.token_stride[0] = key_token_stride_bytes, a.head_stride[0] = key_head_stride_bytes;
    a.token_stride[1] = value_token_stride_bytes, a.head_stride[1] = value_head_stride_bytes;
    for (int k = 0; k < halves; ++k)
      if (reinterpret_cast<uintptr_t>(a.rows[k]) % 16 || a.token_stride[k] % 16 ||
          a.head_stride[k] % 16)
        return fail(kInval, "%s's pointer and strides must be multiples of 16 bytes (token %lld, "
                    "head %lld)", k ? "value" : "key", (long long)a.token_stride[k],
                    (long long)a.head_stride[k]);
    a.mx = static_cast<char*>(mx_ptr);
    a.mks = mx_kv_stride_bytes, a.mbs = mx_block_stride_bytes;
    a.slots = slots, a.slots64 = slots_are_64bit;
    a.num_slots = num_mx_blocks * tokens_per_block;
    a.heads = num_heads, a.tokens = tokens_per_block, a.dim = head_size;
    a.groups = FastDiv(groups);
    a.per_token = FastDiv(per_token);
    a.per_half = FastDiv(per_token * num_tokens);
    a.units = static_cast<uint32_t>(per_token * num_tokens * halves);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int dev = 0;
    DeviceGuard guard;
    if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
    const dim3 grid((static_cast<int64_t>(a.units) * 4 + kThreads - 1) / kThreads);
    (void)hipGetLastError();
    if (dtype == FKV_DTYPE_BF16)
      hipLaunchKernelGGL(mx4_tokens_kernel<Bf16>, grid, dim3(kThreads), 0, s, a);
    else if (dtype == FKV_DTYPE_FP16)
      hipLaunchKernelGGL(mx4_tokens_kernel<Fp16>, grid, dim3(kThreads), 0, s, a);
    else
      hipLaunchKernelGGL(mx4_tokens_kernel<Fp32>, grid, dim3(kThreads), 0, s, a);
    FKV_HIP(hipGetLastError());
    return 0;
  } catch (const std::exception& e) {
    return fail(static_cast<int>(hipErrorUnknown), "exception: %s", e.what());
  } catch (...) {
    return fail(static_cast<int>(hipErrorUnknown), "unknown exception");
  }
}

}  // extern "C"

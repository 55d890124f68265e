// kv_mx4_attention.hip - attention over a paged KV cache held in 4 bits (layout
// and format in kv_mx4.h): for query i of head hq in a sequence,
//
//   o = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q . k_t - max),   t <= its own position
//
// with K/V head hq / group.  The queries of a group and of neighbouring positions
// are the rows of one tile (row = position * group + head in the group), 16 rows
// being the columns of a matrix instruction, so K and V are read once for all.
//
// K's codes go into the scaled matrix instruction (16x16x128) as they lie in memory: a
// lane's operand is 32 neighbouring elements of one token, which is one scale
// group, 16 bytes and one scale byte.  The queries are the other operand, as sums
// of two e4m3 parts (bf16: 4 + 4 significant bits, exact) or three (fp16), one
// scale a row; parts of elements 2^13 below the row's largest lose bits under
// 2^-21 of it.  S comes out with 4 tokens of one row in a lane.  Those lanes are
// the layout of the second product's operand if its 32 tokens are taken in the
// order (quad * 4 + i of one tile, then of the next), so P never leaves its lane.
// V's codes become bf16 in registers (exact: 2 significant bits), two tokens to a
// register by byte permutes.
//
// Softmax: one pass, running maximum and sum per row in 32 bits, in units of log2.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>

#include "kv_mx4.h"

using namespace fkv_detail;

namespace {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kRows = 16;          // rows of a tile: columns of a matrix instruction
constexpr int kStep = 32;          // tokens of a step: two tiles of 16, k of the second product
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ inline float bits_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ inline uint32_t f32_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ inline uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ inline int64_t uniform64(int64_t v) {
  const uint64_t u = static_cast<uint64_t>(v);
  const uint64_t lo = static_cast<uint32_t>(uniform(static_cast<int>(u)));
  const uint64_t hi = static_cast<uint32_t>(uniform(static_cast<int>(u >> 32)));
  return static_cast<int64_t>(hi << 32 | lo);
}
// the larger of a lane's value and those 16, 32 and 48 lanes away
__device__ inline float max_over_quads(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ inline float sum_over_quads(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

struct Args {
  const char* q;
  char* out;
  float* lse;                        // null: not asked for
  int64_t q_row, q_head, out_row, out_head;   // bytes
  int64_t lse_row, lse_head;         // elements
  const char* mx;
  int64_t mks, mbs;                  // 4-bit cache: half and block strides
  const void* table;
  const void* lens;
  const void* starts;                // null: one query a sequence
  int64_t table_row;                 // elements
  int index64;                       // table, lens and starts are int64
  int num_blocks, width;             // of the cache; of a table row
  int batch, heads, group, queries;
  int tokens;                        // of a block
  int causal;
  float scale_log2;
  FastDiv tiles_per_block, group_div;
};

__device__ inline int64_t index_at(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i]
              : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

struct Seq {
  int first, count;   // its queries
  int keys;           // -1: more than its table row can hold
};
__device__ inline Seq sequence(const Args& a, int b) {
  Seq s;
  if (a.starts) {
    const int64_t lo = index_at(a.starts, b, a.index64), hi = index_at(a.starts, b + 1, a.index64);
    const int64_t n = a.queries;
    s.first = static_cast<int>(lo < 0 ? 0 : lo > n ? n : lo);
    const int64_t end = hi < s.first ? s.first : hi > n ? n : hi;
    s.count = static_cast<int>(end) - s.first;
  } else {
    s.first = b;
    s.count = 1;
  }
  const int64_t k = index_at(a.lens, b, a.index64);
  s.keys = k < 0 ? 0 : k > static_cast<int64_t>(a.width) * a.tokens ? -1 : static_cast<int>(k);
  return s;
}

// Row tiles are numbered so that sequence b's start at first(b) * group / kRows + b,
// which leaves room for its last, partly filled one, and needs no lengths
// but its own: tile `t` belongs to the last sequence that starts at or before it.
__device__ inline int tile_base(const Args& a, int b) {
  if (!a.starts) return b * ((a.group + kRows - 1) / kRows);
  int64_t lo = index_at(a.starts, b, a.index64);
  lo = lo < 0 ? 0 : lo > a.queries ? a.queries : lo;
  return static_cast<int>(lo * a.group / kRows) + b;
}

// The queries of one row as e4m3 parts: operand registers for each part and
// 128-element step, and the scale bytes.
template <int D, int PARTS>
struct Query {
  static constexpr int kSteps = (D + 127) / 128;
  v8i part[PARTS][kSteps];
  int scale[PARTS];
};

template <class T>
__device__ inline void load_16(const char* p, float (&x)[16]) {
  const uint4 r[2] = {reinterpret_cast<const uint4*>(p)[0], reinterpret_cast<const uint4*>(p)[1]};
  if constexpr (__is_same(T, __bf16)) {
    uint32_t u[8];
    __builtin_memcpy(u, r, 32);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[2 * i] = bits_f32(u[i] << 16);
      x[2 * i + 1] = bits_f32(u[i] & 0xffff0000u);
    }
  } else {
    v8h h[2];
    __builtin_memcpy(h, r, 32);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = static_cast<float>(h[i / 8][i % 8]);
  }
}

// Lane (row, quad) holds elements 16 quad .. + 15 and 64 + 16 quad .. + 15 of each
// 128: the order of the instruction's 8-bit operand.
template <class T, int D, int PARTS>
__device__ inline void load_query(const char* row, bool valid, int quad, bool negate,
                                  Query<D, PARTS>& q) {
  constexpr int kSteps = Query<D, PARTS>::kSteps;
  constexpr int kHalves = D >= 128 ? 2 : 1;
  float x[kSteps][kHalves][16];
  uint32_t top = 0;
#pragma unroll
  for (int s = 0; s < kSteps; ++s)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      if (valid) {
        load_16<T>(row + (128 * s + 64 * h + 16 * quad) * 2, x[s][h]);
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) x[s][h][i] = 0.f;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) top = max(top, f32_bits(x[s][h][i]) & 0x7fffffffu);
    }
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 16)));
  top = max(top, static_cast<uint32_t>(__shfl_xor(static_cast<int>(top), 32)));
  // the largest lies in [2^7, 2^8) of the first part, whose elements reach 448; each
  // further part has a scale 2^4 smaller.  A row with an infinity or NaN: scale NaN.
  const bool lost = top >= 0x7f800000u;
  const int e = max(static_cast<int>(top >> 23) - 7, 4 * (PARTS - 1));
  const float up = lost ? 0.f : bits_f32(static_cast<uint32_t>(254 - e) << 23);
#pragma unroll
  for (int p = 0; p < PARTS; ++p) q.scale[p] = lost ? 255 : e - 4 * p;
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          float v = 0.f;
          if (h < kHalves) v = lost ? 0.f : x[s][h < kHalves ? h : 0][4 * w + i] * up;
          r[i] = negate ? -v : v;
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          int c = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
          c = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], c, true);
          q.part[p][s][4 * h + w] = c;
          const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
          const v2f hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
          r[0] = (r[0] - lo[0]) * 16.f;
          r[1] = (r[1] - lo[1]) * 16.f;
          r[2] = (r[2] - hi[0]) * 16.f;
          r[3] = (r[3] - hi[1]) * 16.f;
        }
      }
    }
  }
}

// What a lane loads of one 16-token tile.
template <int D>
struct Tile {
  static constexpr int kSteps = (D + 127) / 128;
  static constexpr int kWords = D >= 128 ? D / 128 : 1;   // of V a token: D / 16 codes
  uint4 k[kSteps];
  int k_scale[kSteps];
  uint32_t v[4][kWords];
  uint32_t v_scale;     // of 4 tokens
};

// Where a lane's parts of a tile lie, from the head's codes and scales on.
template <int D>
struct Lanes {
  uint32_t k_code, k_scale, v_code, v_scale;
};
template <int D>
__device__ inline Lanes<D> lane_offsets(int lane, int tokens) {
  const int c = lane & 15, quad = lane >> 4;
  Lanes<D> o;
  // D = 64: quads 2 and 3 repeat what 0 and 1 load; their queries are zero
  const int block = D >= 128 ? quad : quad & 1;
  o.k_code = c * (D / 2) + 16 * block;
  o.k_scale = block * tokens + c;
  o.v_code = quad * 4 * (D / 2) + c * (D / 32);
  o.v_scale = (c * (D / 16) / 32) * tokens + quad * 4;
  return o;
}

template <int D>
__device__ inline void load_tile(const Args& a, const Lanes<D>& o, int64_t block, int head,
                                 int offset, int quad, Tile<D>& t) {
  const int64_t plane = static_cast<int64_t>(a.heads) * a.tokens * (D / 2);
  const char* const k = a.mx + block * a.mbs;
  const char* const kc = k + (static_cast<int64_t>(head) * a.tokens + offset) * (D / 2);
  const char* const ks = k + plane + static_cast<int64_t>(head) * (D / 32) * a.tokens + offset;
  const char* const vc = kc + a.mks;
  const char* const vs = ks + a.mks;
#pragma unroll
  for (int s = 0; s < Tile<D>::kSteps; ++s) {
    t.k[s] = *reinterpret_cast<const uint4*>(kc + o.k_code + 64 * s);
    t.k_scale[s] = *reinterpret_cast<const uint8_t*>(ks + o.k_scale + 4 * s * a.tokens);
    if (D == 64 && quad >= 2) t.k_scale[s] = 127;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (D == 64) {
      t.v[i][0] = *reinterpret_cast<const uint16_t*>(vc + o.v_code + i * (D / 2));
    } else if constexpr (D == 128) {
      t.v[i][0] = *reinterpret_cast<const uint32_t*>(vc + o.v_code + i * (D / 2));
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(vc + o.v_code + i * (D / 2));
      t.v[i][0] = w.x;
      t.v[i][1] = w.y;
    }
  }
  t.v_scale = *reinterpret_cast<const uint32_t*>(vs + o.v_scale);
}

__device__ inline uint32_t cvt_bf16(uint32_t codes, float scale, int byte) {
  v2bf r;
  switch (byte) {
    case 0: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0); break;
    case 1: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1); break;
    case 2: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2); break;
    default: r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3); break;
  }
  return __builtin_bit_cast(uint32_t, r);
}

__device__ inline uint32_t pack_bf16(float a, float b) {
  v2bf r;
  r[0] = static_cast<__bf16>(a);
  r[1] = static_cast<__bf16>(b);
  return __builtin_bit_cast(uint32_t, r);
}

// A row tile's state: lane (row, quad) holds row `lane & 15`.
template <int D>
struct State {
  v4f o[D / 16];   // o[j][i]: element (D / 16) * (quad * 4 + i) + j
  float m, l;      // l: of this lane's tokens
};

// Two tiles of 16 tokens from token `at` on.  MASKED: some row does not see
// all of them.  `visible`: the keys this lane's row sees; `keys`: those there are.
// P of bf16 has 8 significant bits, as flash attention's has; where the output has
// 11 (SPLIT_P) the rest of P is a second bf16 operand.
template <int D, int PARTS, bool MASKED, bool SPLIT_P>
__device__ inline void attend(const Query<D, PARTS>& q, Tile<D> (&t)[2], int at, int visible,
                              int keys, float scale_log2, int quad, State<D>& st) {
  constexpr int NT = D / 16;
  float s[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    v4f acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < Query<D, PARTS>::kSteps; ++k) {
      v8i kc = {static_cast<int>(t[h].k[k].x), static_cast<int>(t[h].k[k].y),
                static_cast<int>(t[h].k[k].z), static_cast<int>(t[h].k[k].w), 0, 0, 0, 0};
#pragma unroll
      for (int p = PARTS - 1; p >= 0; --p)
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
            kc, q.part[p][k], acc, 4, 0, 0, t[h].k_scale[k], 0, q.scale[p]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[h][i] = acc[i] * scale_log2;
      if (MASKED && at + 16 * h + quad * 4 + i >= visible) s[h][i] = -INFINITY;
    }
  }
  float top = s[0][0];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) top = fmaxf(top, s[h][i]);
  top = max_over_quads(top);
  const float m = fmaxf(st.m, top);
  const float ref = m == -INFINITY ? 0.f : m;     // a row that sees nothing yet
  const float fade = __builtin_amdgcn_exp2f(st.m - ref);
  st.m = m;
  st.l *= fade;
#pragma unroll
  for (int j = 0; j < NT; ++j) st.o[j] *= fade;
  uint32_t p_hi[4], p_lo[4];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float p[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[i] = __builtin_amdgcn_exp2f(s[h][i] - ref);
      st.l += p[i];
    }
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const uint32_t u = pack_bf16(p[2 * w], p[2 * w + 1]);
      p_hi[2 * h + w] = u;
      if constexpr (SPLIT_P)
        p_lo[2 * h + w] = pack_bf16(p[2 * w] - bits_f32(u << 16),
                                    p[2 * w + 1] - bits_f32(u & 0xffff0000u));
    }
  }
  // V: masked tokens hold nothing, whatever their bytes are
  bool any_lost = false;
  uint32_t lost[2] = {0, 0};     // byte i: 255 where token i's group is NaN
  float vs[2][4];
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t b = (t[h].v_scale >> (8 * i)) & 255u;
      if constexpr (MASKED) {
        const bool there = at + 16 * h + quad * 4 + i < keys;
        const bool nan = there && b == 255u;
        if (nan) lost[h] |= 255u << (8 * i);
        any_lost |= nan;
        if (!there || nan) {
          b = 127;
#pragma unroll
          for (int w = 0; w < Tile<D>::kWords; ++w) t[h].v[i][w] = 0;
        }
      }
      vs[h][i] = bits_f32(b << 23);
    }
  const v8bf ph = __builtin_bit_cast(v8bf, make_uint4(p_hi[0], p_hi[1], p_hi[2], p_hi[3]));
  v8bf pl;
  if constexpr (SPLIT_P)
    pl = __builtin_bit_cast(v8bf, make_uint4(p_lo[0], p_lo[1], p_lo[2], p_lo[3]));
#pragma unroll
  for (int j = 0; j < NT; j += 2) {
    uint32_t w[2][4];     // elements j, j + 1 of each token
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        w[h][i] = cvt_bf16(t[h].v[i][D >= 128 ? j / 8 : 0], vs[h][i], (j / 2) % 4);
    uint4 even, odd;
    even.x = perm(w[0][1], w[0][0], 0x05040100u);
    even.y = perm(w[0][3], w[0][2], 0x05040100u);
    even.z = perm(w[1][1], w[1][0], 0x05040100u);
    even.w = perm(w[1][3], w[1][2], 0x05040100u);
    odd.x = perm(w[0][1], w[0][0], 0x07060302u);
    odd.y = perm(w[0][3], w[0][2], 0x07060302u);
    odd.z = perm(w[1][1], w[1][0], 0x07060302u);
    odd.w = perm(w[1][3], w[1][2], 0x07060302u);
    const v8bf ve = __builtin_bit_cast(v8bf, even), vo = __builtin_bit_cast(v8bf, odd);
    st.o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, ph, st.o[j], 0, 0, 0);
    st.o[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, ph, st.o[j + 1], 0, 0, 0);
    if constexpr (SPLIT_P) {
      st.o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ve, pl, st.o[j], 0, 0, 0);
      st.o[j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vo, pl, st.o[j + 1], 0, 0, 0);
    }
  }
  if constexpr (MASKED) {
    // A NaN group of V that some rows see and others do not: 0 x NaN must not
    // reach those that do not, so the product took zeros, and the rows that see
    // it become NaN here.
    if (__any(any_lost)) {
      const int row = (threadIdx.x & 15);
      (void)row;
#pragma unroll
      for (int h = 0; h < 2; ++h)
        for (int tok = 0; tok < 16; ++tok)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const uint32_t f = static_cast<uint32_t>(
                __shfl(static_cast<int>(lost[h]), (tok / 4) * 16 + quad * 4 + i));
            if (((f >> (8 * (tok % 4))) & 255u) && at + 16 * h + tok < visible) {
#pragma unroll
              for (int j = 0; j < NT; ++j) st.o[j][i] = bits_f32(0x7fc00000u);
            }
          }
    }
  }
}

template <class T>
__device__ inline uint32_t narrow2(float a, float b) {
  if constexpr (__is_same(T, __bf16)) return pack_bf16(a, b);
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  v2h r;
  r[0] = static_cast<_Float16>(a);
  r[1] = static_cast<_Float16>(b);
  return __builtin_bit_cast(uint32_t, r);
}

// One wavefront for a row tile of one K/V head.
template <class T, int D>
__global__ __launch_bounds__(64) void mx4_attention_kernel(const Args a) {
  constexpr int PARTS = __is_same(T, __bf16) ? 2 : 3;
  constexpr bool SPLIT_P = !__is_same(T, __bf16);
  constexpr int NT = D / 16;
  const int head = blockIdx.x % a.heads;
  const int tile = blockIdx.x / a.heads;
  int lo = 0, hi = a.batch;        // the last sequence whose tiles start at or before `tile`
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (tile_base(a, mid) <= tile) lo = mid;
    else hi = mid;
  }
  const int b = uniform(lo);
  const Seq seq = sequence(a, b);
  const int first = (tile - tile_base(a, b)) * kRows;
  const int rows = min(kRows, seq.count * a.group - first);
  if (rows <= 0) return;
  const int lane = threadIdx.x, quad = lane >> 4;
  const int r = first + min(lane & 15, rows - 1);
  const int pos = a.group_div.div(r), in_group = r - pos * a.group;
  const bool valid = (lane & 15) < rows;
  const int keys = max(seq.keys, 0);
  const int visible = a.causal ? max(0, keys - seq.count + pos + 1) : keys;
  // of the tile's rows, in order: the first sees the fewest, the last the most
  const int fewest = __shfl(visible, 0), most = uniform(__shfl(visible, rows - 1));
  const int64_t q_at = static_cast<int64_t>(seq.first + pos);
  const int64_t hq = static_cast<int64_t>(head) * a.group + in_group;
  Query<D, PARTS> q;
  load_query<T, D, PARTS>(a.q + q_at * a.q_row + hq * a.q_head, valid, quad, a.scale_log2 < 0.f, q);
  State<D> st;
  st.m = -INFINITY;
  st.l = 0.f;
#pragma unroll
  for (int j = 0; j < NT; ++j) st.o[j] = {0.f, 0.f, 0.f, 0.f};
  const Lanes<D> o = lane_offsets<D>(lane, a.tokens);
  const float scale_log2 = fabsf(a.scale_log2);
  bool bad = seq.keys < 0;
  const int last_tile = (most - 1) / kMx4TokenTile;
  for (int at = 0; at < most; at += kStep) {
    Tile<D> t[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      // past the last tile: that one again, masked as a whole
      const int i = min(at / kMx4TokenTile + h, last_tile);
      const int page = a.tiles_per_block.div(i);
      int64_t block = index_at(a.table, b * a.table_row + page, a.index64);
      if (block < 0 || block >= a.num_blocks) {
        bad = true;
        block = 0;
      }
      block = uniform64(block);
      const int offset = (i - page * static_cast<int>(a.tiles_per_block.d)) * kMx4TokenTile;
      load_tile<D>(a, o, block, head, offset, quad, t[h]);
    }
    if (at + kStep <= fewest)
      attend<D, PARTS, false, SPLIT_P>(q, t, at, visible, keys, scale_log2, quad, st);
    else
      attend<D, PARTS, true, SPLIT_P>(q, t, at, visible, keys, scale_log2, quad, st);
  }
  const float l = bad ? bits_f32(0x7fc00000u) : sum_over_quads(st.l);
  if (!valid) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  char* const out = a.out + q_at * a.out_row + hq * a.out_head + quad * 4 * NT * 2;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t w[NT / 2];
#pragma unroll
    for (int j = 0; j < NT; j += 2) w[j / 2] = narrow2<T>(st.o[j][i] * inv, st.o[j + 1][i] * inv);
#pragma unroll
    for (int x = 0; x < NT / 2; x += 2)
      *reinterpret_cast<uint2*>(out + (i * NT + 2 * x) * 2) = make_uint2(w[x], w[x + 1]);
  }
  if (a.lse && quad == 0)
    a.lse[q_at * a.lse_row + hq * a.lse_head] =
        l == 0.f ? -INFINITY : (st.m + __builtin_amdgcn_logf(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// Host side

int check_attention(const fkv_mx4_attention_args& c) {
  int rc;
  if (c.batch < 0 || c.num_queries < 0)
    return fail(kInval, "negative count: batch=%d num_queries=%d", c.batch, c.num_queries);
  if ((rc = mx4_check_shape(c.tokens_per_block, c.num_heads, c.head_size))) return rc;
  if (c.head_size != 64 && c.head_size != 128 && c.head_size != 256)
    return fail(kInval, "attention over a 4-bit cache takes a head_size of 64, 128 or 256, got %d",
                c.head_size);
  if (c.dtype != FKV_DTYPE_BF16 && c.dtype != FKV_DTYPE_FP16)
    return fail(kInval, "attention over a 4-bit cache takes bf16 or fp16 queries, got dtype %d",
                c.dtype);
  if (c.group_size < 1 || c.group_size > 1024)
    return fail(kInval, "group_size must be in [1, 1024], got %d", c.group_size);
  if (!std::isfinite(c.scale)) return fail(kInval, "scale must be finite");
  if (c.table_width < 0 ||
      static_cast<int64_t>(c.table_width) * c.tokens_per_block > (int64_t(1) << 28))
    return fail(kInval, "table_width must be non-negative and hold at most 2^28 tokens, got %d "
                "blocks of %d", c.table_width, c.tokens_per_block);
  if (static_cast<int64_t>(c.num_queries) * c.group_size >= int64_t(1) << 30)
    return fail(kInval, "%d queries of %d heads a K/V head are too many for one call",
                c.num_queries, c.group_size);
  if (c.batch == 0 || c.num_queries == 0) return 0;
  if (!c.query_starts && c.num_queries < c.batch)
    return fail(kInval, "%d sequences of one query each, but %d queries", c.batch, c.num_queries);
  if (!c.query || !c.out || !c.seq_lens || (!c.block_table && c.table_width > 0))
    return fail(kInval, "null pointer argument");
  const int64_t aligned[] = {c.query_row_stride_bytes, c.query_head_stride_bytes,
                             c.out_row_stride_bytes, c.out_head_stride_bytes,
                             static_cast<int64_t>(reinterpret_cast<uintptr_t>(c.query)),
                             static_cast<int64_t>(reinterpret_cast<uintptr_t>(c.out))};
  for (int64_t v : aligned)
    if (v % 16)
      return fail(kInval, "query's and out's pointers and strides must be multiples of 16 bytes");
  return mx4_check_layer(c.mx_ptr, c.mx_kv_stride_bytes, c.mx_block_stride_bytes, c.num_mx_blocks,
                         2, mx4_chunk_bytes(c.tokens_per_block, c.num_heads, c.head_size));
}

template <class T>
void launch_attention(const Args& a, int dim, dim3 grid, hipStream_t s) {
  if (dim == 64) hipLaunchKernelGGL((mx4_attention_kernel<T, 64>), grid, dim3(64), 0, s, a);
  else if (dim == 128) hipLaunchKernelGGL((mx4_attention_kernel<T, 128>), grid, dim3(64), 0, s, a);
  else hipLaunchKernelGGL((mx4_attention_kernel<T, 256>), grid, dim3(64), 0, s, a);
}

}  // namespace

extern "C" {

int fkv_mx4_attention(const fkv_mx4_attention_args* args, fkv_stream_t stream) {
  try {
    last_error().clear();
    if (!args) return fail(kInval, "null pointer argument");
    const fkv_mx4_attention_args& c = *args;
    int rc = check_attention(c);
    if (rc || c.batch == 0 || c.num_queries == 0) return rc;
    Args a;
    a.q = static_cast<const char*>(c.query);
    a.out = static_cast<char*>(c.out);
    a.lse = c.lse;
    a.q_row = c.query_row_stride_bytes, a.q_head = c.query_head_stride_bytes;
    a.out_row = c.out_row_stride_bytes, a.out_head = c.out_head_stride_bytes;
    a.lse_row = c.lse_row_stride, a.lse_head = c.lse_head_stride;
    a.mx = static_cast<const char*>(c.mx_ptr);
    a.mks = c.mx_kv_stride_bytes, a.mbs = c.mx_block_stride_bytes;
    a.table = c.block_table, a.lens = c.seq_lens, a.starts = c.query_starts;
    a.table_row = c.table_row_stride;
    a.index64 = c.index_is_64bit;
    a.num_blocks = static_cast<int>(c.num_mx_blocks), a.width = c.table_width;
    a.batch = c.batch, a.heads = c.num_heads, a.group = c.group_size, a.queries = c.num_queries;
    a.tokens = c.tokens_per_block, a.causal = c.causal;
    a.scale_log2 = c.scale * kLog2e;
    a.tiles_per_block = FastDiv(c.tokens_per_block / kMx4TokenTile);
    a.group_div = FastDiv(c.group_size);
    const int64_t tiles = c.query_starts
        ? static_cast<int64_t>(c.num_queries) * c.group_size / kRows + c.batch
        : static_cast<int64_t>(c.batch) * ((c.group_size + kRows - 1) / kRows);
    if (tiles * c.num_heads >= int64_t(1) << 31)
      return fail(kInval, "%d queries of %d K/V heads are too many for one call", c.num_queries,
                  c.num_heads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int dev = 0;
    DeviceGuard guard;
    if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
    const dim3 grid(static_cast<uint32_t>(tiles * c.num_heads));
    (void)hipGetLastError();
    if (c.dtype == FKV_DTYPE_BF16) launch_attention<__bf16>(a, c.head_size, grid, s);
    else launch_attention<_Float16>(a, c.head_size, grid, s);
    FKV_HIP(hipGetLastError());
    return 0;
  } catch (const std::exception& e) {
    return fail(static_cast<int>(hipErrorUnknown), "exception: %s", e.what());
  } catch (...) {
    return fail(static_cast<int>(hipErrorUnknown), "unknown exception");
  }
}

}  // extern "C"

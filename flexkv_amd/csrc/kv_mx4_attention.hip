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
// scale a row (heads of 64 take two parts in one instruction); parts of elements 2^13
// below the row's largest lose bits under 2^-21 of it.  The instruction adds the products of
// eight neighbouring elements with the bits under 2^-13 of the largest cut off (so a probe:
// 1 + x comes out short by what x has below 2^-13, towards 0, for x in the same eight and
// no other).  S comes out with 4 tokens
// of one row in a lane.  Those lanes are the layout of the second product's
// operand if its 32 tokens are taken in the order (quad * 4 + i of one tile, then
// of the next), so P never leaves its lane.
// V's codes become bf16 in registers (exact: 2 significant bits), two tokens to a
// register by byte permutes.
//
// Softmax: one pass, running maximum and sum per row in 32 bits, in units of log2.
// The maximum is a reference that follows only when a score passes it by 2^8, so
// most steps neither compare across lanes nor scale the sums.
//
// A workgroup's wavefronts take the 32-token steps of its tile in turn, each loading
// its next step while it computes one, and add up in LDS.  Where there are many rows,
// a tile is two or three times 16, for which a step's V is converted once.  With few tiles
// the keys are cut among workgroups as well (find_work), whose sums a second
// kernel joins in a fixed order.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <type_traits>

#include "kv_mx4.h"

using namespace fkv_detail;

namespace {

typedef float v2f __attribute__((ext_vector_type(2)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t Vec2 __attribute__((ext_vector_type(2)));
typedef uint32_t Vec4 __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

constexpr int kRows = 16;          // rows of a tile: columns of a matrix instruction
constexpr int kStep = 32;          // tokens of a step: two tiles of 16, k of the second product
constexpr int kMinSteps = 32;      // of a workgroup, where the keys are cut
// Steps that cutting has to take off the longest sequence: the plan and the join cost
// 6 us, a wide workgroup's 12 steps 0.9.  16 sequences of 4096 keys, 8 heads: 26 us cut
// in two, 23 uncut (21 without a plan); one of 4096: 16 cut in four, 19 uncut.
constexpr int kCutSteps = 96;
// Weight up to which a score may pass the reference.  Sums of weights times values over n keys
// come to 2^8 n times the largest value before they are divided.
constexpr float kSlack = 256.f;
// The reference of a row that has seen nothing.  Any score passes it, and so does
// not -infinity, which a score that a row does not see becomes.
constexpr float kNothing = -3e38f;
// From this reference on, the products of scores and scale are rounded before the reference
// is taken off.  Below, a fused multiplication takes the exact product to it, which a
// rounded product, the reference, differs from by at most 1; at 2^31 by 64 and more,
// where weights overflow or vanish.
constexpr float kCoarse = 0x1p24f;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

__device__ inline float bits_f32(uint32_t u) { return __builtin_bit_cast(float, u); }
__device__ inline uint32_t f32_bits(float f) { return __builtin_bit_cast(uint32_t, f); }
__device__ inline uint32_t perm(uint32_t hi, uint32_t lo, uint32_t sel) {
  return __builtin_amdgcn_perm(hi, lo, sel);
}
__device__ inline int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
// A chunk of the cache as a buffer: its address is scalar, a lane adds 32 bits of
// offset, and nothing outside the chunk is read.
typedef __amdgpu_buffer_rsrc_t Chunk;
__device__ inline Chunk chunk_at(uint64_t address, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(address), 0, bytes, 0x00027000);
}
// quads: the 4 groups of 16 lanes
__device__ inline float max_over_quads(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
  v = fmaxf(bits_f32(r[0]), bits_f32(r[1]));
  r = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  return fmaxf(bits_f32(r[0]), bits_f32(r[1]));
}
__device__ inline float sum_over_quads(float v) {
  auto r = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
  v = bits_f32(r[0]) + bits_f32(r[1]);
  r = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
  return bits_f32(r[0]) + bits_f32(r[1]);
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
  int tokens, chunk;                 // of a block; bytes of a chunk
  int causal;
  int slots;                         // workgroups to cut the keys into; 0: uncut
  float scale_log2;
  float2* part_ml;                   // [cut][row]: maximum and sum
  float* part_o;                     // [cut][i][j][lane], see State
  int* any_cut;                      // whether some tile has more than one cut
  FastDiv tiles_per_block, group_div, heads_div;
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

// Inclusive sums over the lanes of a wavefront.
template <class V>
__device__ inline V scan_lanes(V v) {
  auto add = [&v](auto ctrl, auto rows) {
    v += __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v),
                                                           decltype(ctrl)::value,
                                                           decltype(rows)::value, 0xf, false));
  };
  using std::integral_constant;
  add(integral_constant<int, 0x111>(), integral_constant<int, 0xf>());   // 1, 2, 4, 8 lanes before
  add(integral_constant<int, 0x112>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x114>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x118>(), integral_constant<int, 0xf>());
  add(integral_constant<int, 0x142>(), integral_constant<int, 0xa>());   // lane 15 of the row before
  add(integral_constant<int, 0x143>(), integral_constant<int, 0xc>());   // lane 31
  return v;
}
__device__ inline int lane_value(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }

// How the workgroups are dealt out.  A sequence has ceil(queries * group / rows a tile)
// tiles; where the keys are cut, every tile of a sequence is cut alike, the
// longer the sequence the more often, so that all cuts together fill the
// `slots` the device has at a time and do not start a second round; with as many tiles
// as slots only sequences longer than the mean are cut.  The lengths are
// read here, on the device: every wavefront works the plan out for itself, sequence
// b = lane, then 64 further on.  The first 64 sequences go longest first, and a
// sequence's tiles last first, as causal rows see more the later they are.
struct Work {
  int seq;                    // < 0: none
  int tile, cut, cuts;
  bool any_cut;               // whether some tile is cut
  int steps;                  // of a cut
  int first;                  // the number of the tile's first cut
  Seq s;
};
__device__ inline int tiles_of(const Args& a, const Seq& s, int rows_a_tile) {
  return (s.count * a.group + rows_a_tile - 1) / rows_a_tile;
}
__device__ inline int steps_of(const Seq& s) { return (max(s.keys, 0) + kStep - 1) / kStep; }
// ceil(steps / per_cut), at least 1; in floats, so perhaps one more
__device__ inline int cuts_of(int steps, float inv_per_cut) {
  return max(1, static_cast<int>(steps * inv_per_cut + 0.9999f));
}

// Item `item` of the plan; by_tile: `item` counts tiles, the answer is its first cut.
__device__ inline Work find_work(const Args& a, int item, int rows_a_tile, bool by_tile) {
  const int lane = threadIdx.x & 63;
  Seq s{0, 0, 0};
  int tiles = 0, b = lane;
  if (lane < a.batch) {
    s = sequence(a, lane);
    tiles = tiles_of(a, s, rows_a_tile);
  }
  const bool few = a.batch <= 64;
  if (few && a.batch > 1) {
    int rank = 0;
    for (int j = 0; j < a.batch; ++j) {
      const int k = lane_value(s.keys, j);
      rank += k > s.keys || (k == s.keys && j < lane);
    }
    if (lane >= a.batch) rank = lane;
    auto move = [&](int v) { return __builtin_amdgcn_ds_permute(rank * 4, v); };
    s.first = move(s.first), s.count = move(s.count), s.keys = move(s.keys);
    tiles = move(tiles), b = move(b);
  }
  float inv_per_cut = 0.f;     // one cut
  int longest = 0;             // of a lane's sequences
  if (a.slots) {
    float total = 0.f;
    if (few) {
      total = static_cast<float>(tiles) * static_cast<float>(steps_of(s));
      longest = tiles ? steps_of(s) : 0;
    } else {
      for (int i = lane; i < a.batch; i += 64) {
        const Seq x = sequence(a, i);
        const int n = tiles_of(a, x, rows_a_tile);
        total += static_cast<float>(n) * static_cast<float>(steps_of(x));
        if (n) longest = max(longest, steps_of(x));
      }
    }
    total = bits_f32(lane_value(f32_bits(scan_lanes(total)), 63));
    // at least this many steps a cut; the sum's error and cuts_of's are less than 1 %
    const float even = fmaxf(total * a.heads / a.slots * 1.01f, kMinSteps);
    // cuts of even size overflow the slots by the last, short ones: longer cuts until
    // they do not, or to twice the size
    const bool pays = __any(longest >= even + kCutSteps);
    inv_per_cut = pays ? 0.5f / even : 0.f;
    for (int i = 0; few && pays && i < 8; ++i) {
      inv_per_cut = 1.f / (even * (1.f + i * 0.125f));
      const int n = lane_value(scan_lanes(tiles * cuts_of(steps_of(s), inv_per_cut)), 63);
      if (static_cast<int64_t>(n) * a.heads <= a.slots) break;
    }
  }
  Work w{-1, 0, 0, 0, static_cast<bool>(__any(cuts_of(longest, inv_per_cut) > 1)), 0, 0,
         Seq{0, 0, 0}};
  int before = 0, cuts_before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    if (b0) {
      b = b0 + lane;
      tiles = 0;
      if (b < a.batch) {
        s = sequence(a, b);
        tiles = tiles_of(a, s, rows_a_tile);
      }
    }
    const int steps = steps_of(s);
    const int cuts = cuts_of(steps, inv_per_cut);
    const int cut_ends = scan_lanes(tiles * cuts);
    const int ends = by_tile ? scan_lanes(tiles) : cut_ends;
    const uint64_t later = __ballot(before + ends > item);
    if (later) {
      const int at = __builtin_ctzll(later);
      const int n = lane_value(tiles, at), c = lane_value(cuts, at);
      const int local = item - (before + lane_value(ends, at) - (by_tile ? n : n * c));
      const int nth = by_tile || c == 1 ? local : uniform(local / c);
      w.seq = lane_value(b, at);
      w.cuts = c;
      w.tile = n - 1 - nth;
      w.cut = by_tile ? 0 : local - nth * c;
      w.steps = uniform((lane_value(steps, at) + c - 1) / c);
      w.first = cuts_before + lane_value(cut_ends, at) - n * c + nth * c;
      w.s = {lane_value(s.first, at), lane_value(s.count, at), lane_value(s.keys, at)};
      return w;
    }
    before += lane_value(ends, 63);
    cuts_before += lane_value(cut_ends, 63);
  }
  return w;
}

// The same where the keys are uncut and every sequence has one query: nothing
// but the sequence's own length is read.
__device__ inline Work find_single(const Args& a, int item, int rows_a_tile) {
  Work w{item, 0, 0, 1, false, 0, 0, Seq{0, 0, 0}};
  const int tiles = (a.group + rows_a_tile - 1) / rows_a_tile;
  if (tiles > 1) {
    w.seq = uniform(item / tiles);
    w.tile = item - w.seq * tiles;
  }
  if (w.seq >= a.batch) {      // of the last round of the XCDs
    w.seq = -1;
    return w;
  }
  w.s = sequence(a, w.seq);
  w.s.keys = uniform(w.s.keys);
  return w;
}

// The queries of 16 rows as e4m3 parts: operand registers for each part and
// 128-element step, and the scale bytes, operand p's in byte p.  D = 64: an operand's
// two halves hold two parts, which K's 64 elements meet twice over.
template <int D, int PARTS>
struct Query {
  static constexpr int kSteps = (D + 127) / 128;
  static constexpr int kOperands = D == 64 ? (PARTS + 1) / 2 : PARTS;
  static constexpr int kVectors = kOperands * kSteps * 2;   // of 16 bytes a lane
  v8i part[kOperands][kSteps];
  int scale;
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
  q.scale = 0;
#pragma unroll
  for (int p = 0; p < Query<D, PARTS>::kOperands; ++p) {
    // of the k that this lane's quad gives the scale for
    const int part = D == 64 ? min(2 * p + quad / 2, PARTS - 1) : p;
    q.scale |= (lost ? 255 : e - 4 * part) << (8 * p);
  }
#pragma unroll
  for (int s = 0; s < kSteps; ++s) {
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        float r[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float v = lost ? 0.f : x[s][h][4 * w + i] * up;
          r[i] = negate ? -v : v;
        }
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
          int c = __builtin_amdgcn_cvt_pk_fp8_f32(r[0], r[1], 0, false);
          c = __builtin_amdgcn_cvt_pk_fp8_f32(r[2], r[3], c, true);
          if constexpr (D == 64) q.part[p / 2][s][4 * (p & 1) + w] = c;
          else q.part[p][s][4 * h + w] = c;
          const v2f lo = __builtin_amdgcn_cvt_pk_f32_fp8(c, false);
          const v2f hi = __builtin_amdgcn_cvt_pk_f32_fp8(c, true);
          r[0] = (r[0] - lo[0]) * 16.f;
          r[1] = (r[1] - lo[1]) * 16.f;
          r[2] = (r[2] - hi[0]) * 16.f;
          r[3] = (r[3] - hi[1]) * 16.f;
        }
        if (D == 64 && PARTS % 2) q.part[PARTS / 2][s][4 + w] = 0;
      }
    }
  }
}

// What a lane loads of a step's two 16-token tiles.
template <int D>
struct Keys {
  static constexpr int kSteps = (D + 127) / 128;
  Vec4 code[2][kSteps];
  int scale[2][kSteps];
};
template <int D>
struct Values {
  static constexpr int kWords = D >= 128 ? D / 128 : 1;   // of a token: D / 16 codes
  uint32_t code[2][4][kWords];
  uint32_t scale[2];     // of 4 tokens
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
  // D = 64: quads 2 and 3 repeat what 0 and 1 load, for the queries' second parts
  const int block = D >= 128 ? quad : quad & 1;
  o.k_code = c * (D / 2) + 16 * block;
  o.k_scale = block * tokens + c;
  o.v_code = quad * 4 * (D / 2) + c * (D / 32);
  o.v_scale = (c * (D / 16) / 32) * tokens + quad * 4;
  return o;
}

// K's codes are read whole by one load and not again by this compute unit: past the
// L1 (96 sequences of 8192 keys 157 -> 148 us; V's, a cache line of which takes four
// loads, gain nothing).
constexpr int kOnce = 2;

// Where 16-token tiles lie, one a lane: the block's address and, in a chunk, the
// head's codes and scales of the tile.  Worked out once for 64 tiles, since in the
// steps' loop scalar arithmetic takes a wavefront's issue slots as well.
struct Tiles {
  uint32_t lo, hi;
  int codes, scales;
};
template <int D>
__device__ inline Tiles find_tiles(const Args& a, int tile, int64_t block, int head) {
  const uint64_t p = reinterpret_cast<uint64_t>(a.mx) + static_cast<uint64_t>(block * a.mbs);
  const int offset =
      (tile - a.tiles_per_block.div(tile) * static_cast<int>(a.tiles_per_block.d)) * kMx4TokenTile;
  return {static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32),
          (head * a.tokens + offset) * (D / 2),
          (a.heads * (D / 2) + head * (D / 32)) * a.tokens + offset};
}
__device__ inline uint64_t block_of(const Tiles& t, int lane) {
  return static_cast<uint64_t>(static_cast<uint32_t>(lane_value(t.hi, lane))) << 32 |
         static_cast<uint32_t>(lane_value(t.lo, lane));
}

// Tile h of a step, which `tile` of the tiles has.
template <int D>
__device__ inline void load_keys(const Args& a, const Lanes<D>& o, const Tiles& tiles, int tile,
                                 int h, Keys<D>& t) {
  const Chunk k = chunk_at(block_of(tiles, tile), a.chunk);
  const int codes = lane_value(tiles.codes, tile), scales = lane_value(tiles.scales, tile);
#pragma unroll
  for (int s = 0; s < Keys<D>::kSteps; ++s) {
    t.code[h][s] = __builtin_amdgcn_raw_buffer_load_b128(k, o.k_code + 64 * s, codes, kOnce);
    t.scale[h][s] =
        __builtin_amdgcn_raw_buffer_load_b8(k, o.k_scale, scales + 4 * s * a.tokens, 0);
  }
}
template <int D>
__device__ inline void load_values(const Args& a, const Lanes<D>& o, const Tiles& tiles, int tile,
                                   int h, Values<D>& t) {
  const Chunk v = chunk_at(block_of(tiles, tile) + static_cast<uint64_t>(a.mks), a.chunk);
  const int codes = lane_value(tiles.codes, tile), scales = lane_value(tiles.scales, tile);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (D == 64) {
      t.code[h][i][0] = __builtin_amdgcn_raw_buffer_load_b16(v, o.v_code + i * (D / 2), codes, 0);
    } else if constexpr (D == 128) {
      t.code[h][i][0] = __builtin_amdgcn_raw_buffer_load_b32(v, o.v_code + i * (D / 2), codes, 0);
    } else {
      const Vec2 w = __builtin_amdgcn_raw_buffer_load_b64(v, o.v_code + i * (D / 2), codes, 0);
      t.code[h][i][0] = w[0];
      t.code[h][i][1] = w[1];
    }
  }
  t.scale[h] = __builtin_amdgcn_raw_buffer_load_b32(v, o.v_scale, scales, 0);
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
  float m, l;      // the reference; the sum of this lane's tokens
  uint32_t lost;   // bit i: o[][i] is NaN
};

// Byte i of `scales` as the scale of a conversion, which reads its exponent
// field and nothing else (every sign and mantissa tried gave the same).
__device__ inline float byte_scale(uint32_t scales, int i) {
  return bits_f32(i == 0 ? scales << 23 : i == 1 ? scales << 15 : i == 2 ? scales << 7
                                                                        : scales >> 1);
}

__device__ inline v4f multiply_keys(v8i k, v8i q, v4f acc, int k_scale, int q_scale, int part) {
  switch (part) {
    case 0:
      return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q, acc, 4, 0, 0, k_scale, 0,
                                                              q_scale);
    case 1:
      return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q, acc, 4, 0, 0, k_scale, 1,
                                                              q_scale);
    default:
      return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(k, q, acc, 4, 0, 0, k_scale, 2,
                                                              q_scale);
  }
}

// The parts of a step of 32 tokens from token `at` on, for R row tiles.
// `visible`: the keys this lane's rows see; `keys`: those there are.

// s[r][h][i] = q . k of row tile r and token 16 h + 4 quad + i; query(r) gives r's.
template <int D, int PARTS, int R, class GetQuery>
__device__ inline void scores(GetQuery query, const Keys<D>& t, v4f (&s)[R][2]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const Query<D, PARTS> q = query(r);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      s[r][h] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < Keys<D>::kSteps; ++k) {
        const Vec4 c = t.code[h][k];
        const v8i kc = {static_cast<int>(c[0]), static_cast<int>(c[1]), static_cast<int>(c[2]),
                        static_cast<int>(c[3]), 0, 0, 0, 0};
#pragma unroll
        for (int p = Query<D, PARTS>::kOperands - 1; p >= 0; --p)
          s[r][h] = multiply_keys(kc, q.part[p][k], s[r][h], t.scale[h][k], q.scale, p);
      }
    }
  }
}

template <int R>
__device__ inline void hide(v4f (&s)[R][2], int at, const int (&visible)[R], int quad) {
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        if (at + 16 * h + quad * 4 + i >= visible[r]) s[r][h][i] = -INFINITY;
}

// The weights p of a step as the second product's operand.  P of bf16 has 8
// significant bits, its rounding averaging out over the keys; where the output has
// 11 (SPLIT) the rest of P is a second operand.
template <int R, bool SPLIT>
struct Weights {
  v8bf hi[R], lo[R];
  float l[R];     // what State::l becomes
};

// s * scale rounded, then less m
__device__ inline float rounded_less(float s, float scale, float m) {
#pragma clang fp contract(off)
  const float x = s * scale;
  return x - m;
}

// Row tile r's scores as weights; returns their sum, which is over kSlack where one
// of them passes the reference by more than that.
template <int D, int R, bool SPLIT>
__device__ inline float weigh(const v4f (&s)[R][2], const State<D>& st, int r, float scale_log2,
                              Weights<R, SPLIT>& w, bool coarse = false) {
  float p[8], sum = 0.f;
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const float score = s[r][x / 4][x % 4];
    p[x] = __builtin_amdgcn_exp2f(coarse ? rounded_less(score, scale_log2, st.m)
                                         : __builtin_fmaf(score, scale_log2, -st.m));
    sum = x ? sum + p[x] : p[x];
  }
  w.l[r] = st.l + sum;
  uint32_t hi[4], lo[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    hi[x] = pack_bf16(p[2 * x], p[2 * x + 1]);
    if constexpr (SPLIT)
      lo[x] = pack_bf16(p[2 * x] - bits_f32(hi[x] << 16),
                        p[2 * x + 1] - bits_f32(hi[x] & 0xffff0000u));
  }
  w.hi[r] = __builtin_bit_cast(v8bf, make_uint4(hi[0], hi[1], hi[2], hi[3]));
  if constexpr (SPLIT) w.lo[r] = __builtin_bit_cast(v8bf, make_uint4(lo[0], lo[1], lo[2], lo[3]));
  return sum;
}

// Some score passes its row's reference: the references follow, and the weights
// are made again.  Returns the sum of weights past which the next step is to come here:
// any, where a reference is kCoarse or more.
template <int D, int R, bool SPLIT>
__device__ inline float follow(const v4f (&s)[R][2], State<D> (&st)[R], float scale_log2,
                               Weights<R, SPLIT>& w) {
  bool any_coarse = false;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float top = st[r].m;
#pragma unroll
    for (int x = 0; x < 8; ++x) top = fmaxf(top, s[r][x / 4][x % 4] * scale_log2);
    const float m = max_over_quads(top);
    const float fade = __builtin_amdgcn_exp2f(st[r].m - m);
    st[r].m = m;
    st[r].l *= fade;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) st[r].o[j] *= fade;
    const bool coarse = fabsf(m) >= kCoarse && m != kNothing;
    any_coarse |= coarse;
    weigh(s, st[r], r, scale_log2, w, coarse);
  }
  return __any(any_coarse) ? -1.f : kSlack;
}

// Weights of 0 leave out what a row does not see only while V is finite, which it is in
// bf16 unless a scale byte is over 252: NaN, or bytes of a block that nothing was
// written to.  Those tokens are taken out here, and what the rows that do see
// them hold is marked as NaN.
// bit 8 i + 7 of each byte i that is
__device__ inline uint32_t over_252(uint32_t x) {
  return ((x & 0x7f7f7f7fu) + 0x03030303u) & x & 0x80808080u;
}
template <int D>
__device__ inline bool not_finite(const Values<D>& t) {
  return (over_252(t.scale[0]) | over_252(t.scale[1])) != 0;
}
template <int D, int R>
__device__ inline void take_out(Values<D>& t, int at, const int (&visible)[R], int keys, int quad,
                                State<D> (&st)[R]) {
  bool any_lost = false;
  uint32_t lost[2] = {0, 0};     // byte i: token i's group
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t over = over_252(t.scale[h]);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!(over >> (8 * i) & 0x80u)) continue;
      if (at + 16 * h + quad * 4 + i < keys) {
        lost[h] |= 255u << (8 * i);
        any_lost = true;
      }
      t.scale[h] &= ~(255u << (8 * i));
#pragma unroll
      for (int w = 0; w < Values<D>::kWords; ++w) t.code[h][i][w] = 0;
    }
  }
  if (!__any(any_lost)) return;
#pragma unroll 1
  for (int tok = 0; tok < 32; ++tok) {
    const uint32_t mine = tok < 16 ? lost[0] : lost[1];
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const uint32_t f = static_cast<uint32_t>(
          __shfl(static_cast<int>(mine), (tok / 4 % 4) * 16 + quad * 4 + i));
      const bool is = (f >> (8 * (tok % 4))) & 255u;
#pragma unroll
      for (int r = 0; r < R; ++r)
        if (is && at + tok < visible[r]) st[r].lost |= 1u << i;
    }
  }
}

// Elements j and j + 1 of a lane's 8 tokens of V as bf16 operands.
template <int D>
__device__ inline void widen(const Values<D>& t, int j, v8bf& even, v8bf& odd) {
  uint32_t w[2][4];     // of each token both
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w[h][i] = cvt_bf16(t.code[h][i][D >= 128 ? j / 8 : 0], byte_scale(t.scale[h], i),
                         (j / 2) % 4);
  uint32_t e[4], d[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const uint32_t lo = w[x / 2][2 * (x % 2)], hi = w[x / 2][2 * (x % 2) + 1];
    e[x] = perm(hi, lo, 0x05040100u);
    d[x] = perm(hi, lo, 0x07060302u);
  }
  even = __builtin_bit_cast(v8bf, make_uint4(e[0], e[1], e[2], e[3]));
  odd = __builtin_bit_cast(v8bf, make_uint4(d[0], d[1], d[2], d[3]));
}

// o[j] += p v of element j of V
template <int D, int R, bool SPLIT>
__device__ inline void accumulate(v8bf v, int j, const Weights<R, SPLIT>& p, State<D> (&st)[R]) {
#pragma unroll
  for (int r = 0; r < R; ++r) {
    st[r].o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p.hi[r], st[r].o[j], 0, 0, 0);
    if constexpr (SPLIT)
      st[r].o[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p.lo[r], st[r].o[j], 0, 0, 0);
  }
}

// Quantising rounds up to 65536, which reads back as fp16's largest: finite sums past that
// are that here too.
__device__ inline float within_fp16(float x) {
  return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f) : x;
}
template <class T>
__device__ inline uint32_t narrow2(float a, float b) {
  if constexpr (__is_same(T, __bf16)) return pack_bf16(a, b);
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  v2h r;
  r[0] = static_cast<_Float16>(within_fp16(a));
  r[1] = static_cast<_Float16>(within_fp16(b));
  return __builtin_bit_cast(uint32_t, r);
}

// Row r of a tile: the packed query row, its head and the keys it sees.
struct Row {
  int64_t at;
  int head, visible;
};
__device__ inline Row row_of(const Args& a, const Seq& s, int r, int kv_head) {
  const int pos = a.group_div.div(r);
  Row row;
  row.at = static_cast<int64_t>(s.first) + pos;
  row.head = kv_head * a.group + (r - pos * a.group);
  const int keys = max(s.keys, 0);
  row.visible = a.causal ? max(0, keys - s.count + pos + 1) : keys;
  return row;
}

__device__ inline void write_lse(const Args& a, const Row& row, int visible, float m, float l) {
  a.lse[row.at * a.lse_row + row.head * a.lse_head] =
      l == 0.f ? (visible ? bits_f32(0x7fc00000u) : -INFINITY)
               : (m + __builtin_amdgcn_logf(l)) * kLn2;
}

// NJ elements from (D / 16) * (4 quad + i) + j0 of a row on as the output's type, and
// its lse.  No weight at all: zeros for a row that sees no key, NaN for one whose scores
// are all below what 32 bits hold.
template <class T, int D, int NJ>
__device__ inline void write_row(const Args& a, const Row& row, int visible, int quad, int i,
                                 int j0, const float (&o)[NJ], float m, float l) {
  constexpr int NT = D / 16;
  const float inv = l == 0.f ? (visible ? bits_f32(0x7fc00000u) : 0.f) : 1.f / l;
  uint32_t w[NJ / 2];
#pragma unroll
  for (int j = 0; j < NJ; j += 2) w[j / 2] = narrow2<T>(o[j] * inv, o[j + 1] * inv);
  char* const out =
      a.out + row.at * a.out_row + row.head * a.out_head + ((quad * 4 + i) * NT + j0) * 2;
  if constexpr (NJ == 2) {
    *reinterpret_cast<uint32_t*>(out) = w[0];
  } else {
#pragma unroll
    for (int x = 0; x < NJ / 2; x += 2)
      *reinterpret_cast<uint2*>(out + x * 4) = make_uint2(w[x], w[x + 1]);
  }
  if (a.lse && quad == 0 && i == 0 && j0 == 0) write_lse(a, row, visible, m, l);
}

// Which item of the plan, and which K/V head, a workgroup has.  Workgroups go round the
// 8 XCDs.  Where K and V are read once, an item's heads are on one XCD, so that a
// block is read whole by one L2 at about one time.  Where many tiles read them, a
// head's tiles are on one XCD if there are 8 heads.
constexpr int kXcds = 8;
struct Place {
  int item, head;
};
__device__ inline Place heads_together(const Args& a, int block) {
  const int nth = block / kXcds, group = a.heads_div.div(nth);
  return {group * kXcds + block % kXcds, nth - group * a.heads};
}
__device__ inline Place heads_apart(const Args& a, int block) {
  const int item = a.heads_div.div(block);
  return {item, block - item * a.heads};
}
// The number that a cut's part of the workspace has.
__device__ inline int64_t part_of(const Args& a, int item, int head) {
  return static_cast<int64_t>(item) * a.heads + head;
}

// The tiles of the steps that a wavefront takes, every W-th from its first on, 32 steps
// at a time: `kChunk` of them and the first two of the next, which are asked for early.
// The next block ids are loaded a chunk ahead: in the steps' loop, a load of them
// would be waited for with the steps' own.
constexpr int kChunk = 30;     // a multiple of the steps' loops' 2 and 3
constexpr int kNoTile = 0x7fffffff;
template <int D, int W>
struct Walk {
  const Args& a;
  int seq, head, lane;
  int from;             // the chunk's first step
  int last_tile, end;   // tiles and steps there are keys in
  int64_t ids;          // of the chunk, then of the next
  Tiles tiles;
  int bad = kNoTile;    // a lane's first tile with keys whose block is outside the cache

  __device__ int tile() const { return (from + (lane >> 1) * W) * 2 + (lane & 1); }
  // before last_tile and end are known
  __device__ void ask(int step) {
    from = step;
    ids = load_ids();
  }
  __device__ void start(int last, int ends) {
    last_tile = last, end = ends;
    settle();
  }
  __device__ void next_chunk() {
    from += kChunk * W;
    settle();
  }
  // A step that a wavefront asks for past its last is the last of all, perhaps another
  // wavefront's, for which this gives some block's tile.
  __device__ int place(int step) const { return 2 * min((step - from) / W, 31); }

 private:
  __device__ int64_t load_ids() const {
    if (!a.width) return -1;
    const int page = a.tiles_per_block.div(tile());
    return index_at(a.table, seq * a.table_row + min(page, a.width - 1), a.index64);
  }
  __device__ void settle() {
    const bool outside = ids < 0 || ids >= a.num_blocks;
    if (outside && tile() <= last_tile && tile() < 2 * end) bad = min(bad, tile());
    tiles = find_tiles<D>(a, tile(), outside ? 0 : ids, head);
    from += kChunk * W;
    ids = load_ids();
    from -= kChunk * W;
  }
};

template <int D>
__device__ inline void clear(State<D>& st) {
  st.m = kNothing;
  st.l = 0.f;
  st.lost = 0;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) st.o[j] = {0.f, 0.f, 0.f, 0.f};
}

// The scale of the scores; not 0, so that -infinity stays that, but the smallest there is,
// with which no finite score comes to more than 2^-21.
__device__ inline float score_scale(const Args& a) {
  return fmaxf(fabsf(a.scale_log2), 0x1p-149f);
}

// Row tiles of a workgroup for many queries, as registers allow.
constexpr int most_row_tiles(int dim) { return dim <= 128 ? 3 : 2; }
// Wavefronts a SIMD is to hold: more than these cost spilled registers.
constexpr int waves_a_simd(int row_tiles, int dim) {
  return row_tiles == 1 ? (dim <= 128 ? 3 : 2) : dim <= 128 ? 2 : 1;
}
// Wavefronts of a wide workgroup, which takes a compute unit for itself.
constexpr int most_waves(int dim) { return 4 * waves_a_simd(1, dim); }

// One workgroup of W wavefronts for a cut of the keys of a tile of 16 R rows of one K/V
// head, whose wavefronts take the steps in turn.
//
// R = 1, single queries and few: memory bounds it, K and V being read once.  MI355X, 32
// sequences of 8192 keys, 8 heads: 286 MB in 60 us, 64 sequences 571 MB in 97; with the
// arithmetic left out 62 for 66 then, with K and V in the L2 41.  W = 12 where few
// sequences have to fill a compute unit each, which then need few cuts, else 4.
// R = 3 (2 of 256 elements, and where 3 make too few workgroups), many queries:
// arithmetic bounds it.  A step of 16 rows is 256 cycles of matrix instructions, 190 of
// vector ones (128 for exponentials), and a third of the 288 that V's conversion takes;
// counted over a prompt, matrix instructions are busy 43 % of the cycles, vector ones
// 54 %, which two wavefronts a SIMD hardly overlap.  2048 queries of 32 heads over 8192
// keys: 255 us (935 TFLOP/s); 2 row tiles 266; 4 with spilled registers 243, but more
// where workgroups are few; V converted once for four wavefronts of 32 rows each,
// through LDS, 257, and half as slow again for short prompts, whose workgroups are
// then few.  256 elements: 654 us with one wavefront a SIMD, 1054 with two and
// spilled registers.
template <class T, int D, int R, int W>
__global__ __launch_bounds__(64 * W, waves_a_simd(R, D)) void mx4_attention_kernel(
    const Args a) {
  constexpr int PARTS = __is_same(T, __bf16) ? 2 : 3;
  constexpr bool SPLIT_P = !__is_same(T, __bf16);
  constexpr int NT = D / 16;
  using Q = Query<D, PARTS>;
  // the queries, then a row tile's sums of every wavefront
  __shared__ uint4 shared[std::max(R * Q::kVectors, W * NT)][64];
  __shared__ int shared_scale[R][64];
  __shared__ float sum_m[W][R][16], sum_l[W][R][16];
  const Place at = R == 1 ? heads_together(a, blockIdx.x) : heads_apart(a, blockIdx.x);
  const Work w = a.slots || a.starts ? find_work(a, at.item, kRows * R, false)
                                     : find_single(a, at.item, kRows * R);
  if (a.slots && blockIdx.x == 0 && threadIdx.x == 0) *a.any_cut = w.any_cut;
  if (w.seq < 0) return;
  const int first = w.tile * kRows * R;
  const int rows = min(kRows * R, w.s.count * a.group - first);
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, quad = lane >> 4;
  auto row_at = [&](int n) { return row_of(a, w.s, first + min(n, rows - 1), at.head); };
  Walk<D, W> walk{a, w.seq, at.head, lane};
  int step = (w.cuts > 1 ? w.cut * w.steps : 0) + wave;
  walk.ask(step);
  const int keys = max(w.s.keys, 0);
  int visible[R];
#pragma unroll
  for (int r = 0; r < R; ++r) visible[r] = row_at(16 * r + (lane & 15)).visible;
  // of the rows, in order, the first sees the fewest, the last the most
  const int fewest = lane_value(visible[0], 0), most = lane_value(visible[R - 1], 15);
  const int all_steps = (most + kStep - 1) / kStep;
  const int end = w.cuts > 1 ? min(all_steps, (w.cut + 1) * w.steps) : all_steps;
  walk.start((most - 1) / kMx4TokenTile, end);
  const Lanes<D> o = lane_offsets<D>(lane, a.tokens);
  // Steps in flight beside the one that is computed (two measured as one).  Loads past
  // the last step are of that one again: were they conditional, no wait could be for
  // a number of them, and each would be for all.
  constexpr int kAhead = 1, N = kAhead + 1;
  static_assert(kChunk % N == 0, "");
  Keys<D> k[N];
  Values<D> v[N];
  auto load = [&](int s, int n) {
    s = min(s, end - 1);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      load_keys<D>(a, o, walk.tiles, walk.place(s) + h, h, k[n]);
      load_values<D>(a, o, walk.tiles, walk.place(s) + h, h, v[n]);
    }
  };
  if (step < end) {
#pragma unroll
    for (int n = 0; n < kAhead; ++n) load(step + n * W, n);
  }
  // a wavefront prepares a row tile's queries, for all of them
  for (int r = wave; r < R; r += W) {
    const int n = 16 * r + (lane & 15);
    const Row row = row_at(n);
    Q q;
    load_query<T, D, PARTS>(a.q + row.at * a.q_row + row.head * a.q_head, n < rows, quad,
                            a.scale_log2 < 0.f, q);
#pragma unroll
    for (int x = 0; x < Q::kVectors; ++x) {
      uint4 u;
      __builtin_memcpy(&u, reinterpret_cast<const char*>(&q.part[0][0]) + 16 * x, 16);
      shared[r * Q::kVectors + x][lane] = u;
    }
    shared_scale[r][lane] = q.scale;
  }
  __syncthreads();
  auto read_query = [&](int r) {
    Q q;
#pragma unroll
    for (int x = 0; x < Q::kVectors; ++x) {
      const uint4 u = shared[r * Q::kVectors + x][lane];
      __builtin_memcpy(reinterpret_cast<char*>(&q.part[0][0]) + 16 * x, &u, 16);
    }
    q.scale = shared_scale[r][lane];
    return q;
  };
  Q kept;
  if constexpr (R == 1) kept = read_query(0);
  auto query = [&](int r) {
    if constexpr (R == 1) return kept;
    // every step anew: held, they would be 16 registers a tile and part
    if (r == 0) asm volatile("" ::: "memory");
    return read_query(r);
  };
  const float scale_log2 = score_scale(a);
  float slack = kSlack;
  State<D> st[R];
#pragma unroll
  for (int r = 0; r < R; ++r) clear(st[r]);
  // N steps at a time: a step's registers are named by its place, so that no copy of
  // them waits for their loads.
  for (bool more = step < end; more;) {
    // a start 4 bytes off a cache line measured 671 us for 654, 2048 queries of heads of 256
    if constexpr (R > 1) asm volatile(".p2align 6");
    for (int c = 0; c < kChunk / N && more; ++c) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (!more) break;
        load(step + kAhead * W, (n + kAhead) % N);
        v4f s[R][2];
        scores<D, PARTS, R>(query, k[n], s);
        const int token = step * kStep;
        if (token + kStep > fewest) hide(s, token, visible, quad);
        Weights<R, SPLIT_P> p;
        bool passes = false;
#pragma unroll
        for (int r = 0; r < R; ++r) passes |= weigh(s, st[r], r, scale_log2, p) > slack;
        if (__any(passes)) slack = follow(s, st, scale_log2, p);
        // expected not to: 256 queries over 32768 keys 197 us, 202 with the path in the loop's line
        if (__builtin_expect(__any(not_finite(v[n])), 0))
          take_out(v[n], token, visible, keys, quad, st);
#pragma unroll
        for (int r = 0; r < R; ++r) st[r].l = p.l[r];
#pragma unroll
        for (int j = 0; j < NT; j += 2) {
          v8bf even, odd;
          widen(v[n], j, even, odd);
          accumulate(even, j, p, st);
          accumulate(odd, j + 1, p, st);
        }
        step += W;
        more = step < end;
      }
    }
    walk.next_chunk();
  }
  // The wavefronts' sums, each to the common reference; wavefront i (and i + 4, half
  // each) adds up the elements [][i] of all.
  int bad = kNoTile;
  if (__any(walk.bad != kNoTile)) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i) bad = min(bad, lane_value(walk.bad, i));
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const float l = sum_over_quads(st[r].l);
    if (quad == 0) {
      sum_m[wave][r][lane] = st[r].m;
      const bool lost =
          w.s.keys < 0 || (visible[r] > 0 && (visible[r] - 1) / kMx4TokenTile >= bad);
      sum_l[wave][r][lane] = lost ? bits_f32(0x7fc00000u) : l;
    }
  }
  __syncthreads();     // and the queries have been read
  constexpr int kParts = W >= 8 ? 2 : 1, NJ = NT / kParts;
  const int i = wave & 3, j0 = wave / 4 * NJ;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    float m = kNothing, l = 0.f;
#pragma unroll
    for (int x = 0; x < W; ++x) m = fmaxf(m, sum_m[x][r][lane & 15]);
#pragma unroll
    for (int x = 0; x < W; ++x)
      l += sum_l[x][r][lane & 15] * __builtin_amdgcn_exp2f(sum_m[x][r][lane & 15] - m);
    const float f = __builtin_amdgcn_exp2f(st[r].m - m);
    v4f factor;
#pragma unroll
    for (int y = 0; y < 4; ++y) factor[y] = st[r].lost >> y & 1 ? bits_f32(0x7fc00000u) : f;
    if (r) __syncthreads();
#pragma unroll
    for (int j = 0; j < NT; ++j)
      reinterpret_cast<v4f*>(shared[wave * NT + j])[lane] = st[r].o[j] * factor;
    __syncthreads();
    if (wave >= 4 * kParts) continue;
    float sums[NJ];
#pragma unroll
    for (int j = 0; j < NJ; ++j) {
      sums[j] = 0.f;
#pragma unroll
      for (int x = 0; x < W; ++x)
        sums[j] += reinterpret_cast<const float*>(shared[x * NT + j0 + j])[lane * 4 + i];
    }
    const int n = 16 * r + (lane & 15);
    if (n >= rows) continue;
    if (w.cuts == 1) {
      write_row<T, D, NJ>(a, row_at(n), visible[r], quad, i, j0, sums, m, l);
    } else {
      const int64_t part = part_of(a, at.item, at.head) * R + r;
      if (wave == 0 && quad == 0) a.part_ml[part * kRows + lane] = make_float2(m, l);
#pragma unroll
      for (int j = 0; j < NJ; ++j) a.part_o[((part * 4 + i) * NT + j0 + j) * 64 + lane] = sums[j];
    }
  }
}

// Joins the cuts of a tile: of the 4 G wavefronts, i + 4 g takes the elements [][i] of
// State of every G-th cut from g on, some at a time in flight; their sums are
// added in the order of g.
template <class T, int D, int R, int G>
__global__ __launch_bounds__(256 * G) void mx4_join_kernel(const Args a) {
  constexpr int NT = D / 16, kAhead = D == 256 ? 2 : 4;
  if (!*a.any_cut) return;
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, quad = lane >> 4;
  const int i = wave & 3, g = wave >> 2;
  const int block = blockIdx.x / R, r = blockIdx.x % R;
  const int tile = a.heads_div.div(block);
  const int kv_head = block - tile * a.heads;
  const Work w = find_work(a, tile, kRows * R, true);
  if (w.seq < 0 || w.cuts == 1) return;
  __shared__ float sum_o[G * 4][NT][64];
  __shared__ float sum_m[G][16], sum_l[G][16];
  const int first = (w.tile * R + r) * kRows;
  const bool valid = first + (lane & 15) < w.s.count * a.group;
  float o[NT], m = kNothing, l = 0.f;
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j] = 0.f;
  if (valid) {
    const int64_t part = part_of(a, w.first, kv_head) * R + r;
    const float2* const ml = a.part_ml + part * kRows + (lane & 15);
    const float* const po = a.part_o + (part * 4 + i) * NT * 64 + lane;
    const int64_t next = static_cast<int64_t>(a.heads) * R;
    for (int c0 = g; c0 < w.cuts; c0 += G * kAhead) {
      float2 x[kAhead];
      float y[kAhead][NT];
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const int c = c0 + n * G;
        x[n] = make_float2(kNothing, 0.f);
#pragma unroll
        for (int j = 0; j < NT; ++j) y[n][j] = 0.f;
        if (c < w.cuts) {
          x[n] = ml[c * next * kRows];
#pragma unroll
          for (int j = 0; j < NT; ++j) y[n][j] = po[(c * next * 4 * NT + j) * 64];
        }
      }
#pragma unroll
      for (int n = 0; n < kAhead; ++n) {
        const float top = fmaxf(m, x[n].x);
        const float f = __builtin_amdgcn_exp2f(m - top), h = __builtin_amdgcn_exp2f(x[n].x - top);
        m = top;
        l = l * f + x[n].y * h;
#pragma unroll
        for (int j = 0; j < NT; ++j) o[j] = o[j] * f + y[n][j] * h;
      }
    }
  }
  if (i == 0 && quad == 0) sum_m[g][lane] = m, sum_l[g][lane] = l;
#pragma unroll
  for (int j = 0; j < NT; ++j) sum_o[wave][j][lane] = o[j];
  __syncthreads();
  if (g || !valid) return;
  float top = kNothing;
#pragma unroll
  for (int x = 0; x < G; ++x) top = fmaxf(top, sum_m[x][lane & 15]);
  l = 0.f;
#pragma unroll
  for (int j = 0; j < NT; ++j) o[j] = 0.f;
#pragma unroll
  for (int x = 0; x < G; ++x) {
    const float f = __builtin_amdgcn_exp2f(sum_m[x][lane & 15] - top);
    l += sum_l[x][lane & 15] * f;
#pragma unroll
    for (int j = 0; j < NT; ++j) o[j] += sum_o[x * 4 + i][j][lane] * f;
  }
  const Row row = row_of(a, w.s, first + (lane & 15), kv_head);
  write_row<T, D, NT>(a, row, row.visible, quad, i, 0, o, top, l);
}

// ---------------------------------------------------------------------------
// Host side

int check_sizes(const fkv_mx4_attention_args& c) {
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
  if (!c.query_starts && c.num_queries < c.batch && c.num_queries > 0)
    return fail(kInval, "%d sequences of one query each, but %d queries", c.batch, c.num_queries);
  return 0;
}

int check_attention(const fkv_mx4_attention_args& c) {
  const int rc = check_sizes(c);
  if (rc || c.batch == 0 || c.num_queries == 0) return rc;
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

struct LaunchPlan {
  int row_tiles;          // R
  int64_t tiles;          // times heads: the most there can be
  bool wide;              // a workgroup has all wavefronts of a compute unit, else 4
  int slots;
  int64_t workgroups;
  size_t ml_bytes, o_bytes;
};

constexpr int kComputeUnits = 256;
constexpr int kLongSteps = 256;    // of a table row, from which tiles of many rows are cut

LaunchPlan launch_plan(const fkv_mx4_attention_args& c) {
  LaunchPlan p;
  const int64_t rows = static_cast<int64_t>(c.query_starts ? c.num_queries : c.batch) * c.group_size;
  auto tiles = [&](int row_tiles) {
    const int n = kRows * row_tiles;
    return (c.query_starts ? rows / n + c.batch
                           : static_cast<int64_t>(c.batch) * ((c.group_size + n - 1) / n)) *
           c.num_heads;
  };
  const int64_t most_steps =
      (static_cast<int64_t>(c.table_width) * c.tokens_per_block + kStep - 1) / kStep;
  // Many rows a tile share V's conversion, but have fewer workgroups, which have to fill
  // the compute units.  Not the most there can be counts, but what to expect: of a
  // sequence's last tile, half.  1 sequence of 400 queries of 32 heads over 8192 keys:
  // 78 us with 2 row tiles in 400 workgroups, 98 with 3 in 272; 600 queries: 117 with 2 in
  // 600, 98 with 3 in 400; 16 sequences of 16 queries over 4096: 34 with 2, 44 with 3.
  // Fewer are cut along the keys, which pays for long ones: 300 queries over 8192 keys 66
  // us for 78 with 2 row tiles uncut, 8 sequences of 40 rows 33 for 42 with 1, but 16
  // of 40 rows over 2000 keys 27 for 25.
  const int many = most_row_tiles(c.head_size);
  auto fills = [&](int row_tiles, int64_t workgroups) {
    const int n = kRows * row_tiles;
    return rows > static_cast<int64_t>(c.batch) * kRows * (row_tiles - 1) &&
           (rows / n + c.batch / 2) * c.num_heads >= workgroups;
  };
  const bool three = many > 2 && fills(many, kComputeUnits + kComputeUnits / 4);
  const bool cut = !three && most_steps >= kLongSteps && fills(many, 0) &&
                   !fills(many, kComputeUnits);
  p.row_tiles = three || cut ? many : fills(2, kComputeUnits) ? 2 : 1;
  p.tiles = tiles(p.row_tiles);
  p.wide = p.row_tiles == 1 && p.tiles <= kComputeUnits;
  // Tiles of 16 rows for every compute unit: smaller workgroups, three a compute unit, take
  // turns better (40 sequences of 8192 keys: 78 us; wide ones 91), and only sequences
  // longer than the mean are cut: 64 of 2048 keys 31 us, uncut 26, but one of 16384 among
  // 39 of 500 keys 27 us, uncut 82.  With many more tiles the plan costs more.
  p.slots = most_steps < kMinSteps + kCutSteps || p.tiles > 4 * kComputeUnits ? 0
            : p.row_tiles > 1 ? (cut ? 2 * kComputeUnits : 0)
            : p.wide ? kComputeUnits : static_cast<int>(p.tiles);
  // items (cuts of a tile, of all heads), in whole rounds of the XCDs
  const int64_t items = (p.tiles + p.slots + c.num_heads - 1) / c.num_heads;
  p.workgroups = (items + kXcds - 1) / kXcds * kXcds * c.num_heads;
  const int64_t part_rows = p.slots ? p.workgroups * kRows * p.row_tiles : 0;
  p.ml_bytes = part_rows * sizeof(float2) + (p.slots ? 16 : 0);    // and any_cut
  p.o_bytes = part_rows * c.head_size * sizeof(float);
  return p;
}

// A launch has less than 2^32 threads.  Wide workgroups and joins are of few tiles.
int check_plan(const fkv_mx4_attention_args& c, const LaunchPlan& p) {
  if (p.workgroups >= int64_t(1) << 24)
    return fail(kInval, "%d queries of %d K/V heads are too many for one call", c.num_queries,
                c.num_heads);
  return 0;
}

template <class T, int D, int R, int W>
void launch(const Args& a, const LaunchPlan& p, hipStream_t s) {
  hipLaunchKernelGGL((mx4_attention_kernel<T, D, R, W>), dim3(p.workgroups), dim3(64 * W), 0, s, a);
}
template <class T, int D>
void launch(const Args& a, const LaunchPlan& p, hipStream_t s) {
  if (p.row_tiles > 1) {
    constexpr int R = most_row_tiles(D);
    if (p.row_tiles == R) launch<T, D, R, 4>(a, p, s);
    else launch<T, D, 2, 4>(a, p, s);
    if (p.slots)
      hipLaunchKernelGGL((mx4_join_kernel<T, D, R, 1>), dim3(p.tiles * R), dim3(256), 0, s, a);
  } else if (p.wide) {
    launch<T, D, 1, most_waves(D)>(a, p, s);
    if (p.slots)
      hipLaunchKernelGGL((mx4_join_kernel<T, D, 1, 4>), dim3(p.tiles), dim3(1024), 0, s, a);
  } else {
    launch<T, D, 1, 4>(a, p, s);
    if (p.slots)
      hipLaunchKernelGGL((mx4_join_kernel<T, D, 1, 1>), dim3(p.tiles), dim3(256), 0, s, a);
  }
}
template <class T>
void launch_attention(const Args& a, const LaunchPlan& p, int dim, hipStream_t s) {
  if (dim == 64) launch<T, 64>(a, p, s);
  else if (dim == 128) launch<T, 128>(a, p, s);
  else launch<T, 256>(a, p, s);
}

}  // namespace

extern "C" {

int fkv_mx4_attention_workspace(const fkv_mx4_attention_args* args, size_t* bytes) {
  last_error().clear();
  if (!args || !bytes) return fail(kInval, "null pointer argument");
  *bytes = 0;
  int rc = check_sizes(*args);
  if (rc || args->batch == 0 || args->num_queries == 0) return rc;
  const LaunchPlan p = launch_plan(*args);
  if ((rc = check_plan(*args, p))) return rc;
  *bytes = p.ml_bytes + p.o_bytes;
  return 0;
}

int fkv_mx4_attention(const fkv_mx4_attention_args* args, fkv_stream_t stream) {
  try {
    last_error().clear();
    if (!args) return fail(kInval, "null pointer argument");
    const fkv_mx4_attention_args& c = *args;
    int rc = check_attention(c);
    if (rc || c.batch == 0 || c.num_queries == 0) return rc;
    const LaunchPlan p = launch_plan(c);
    if ((rc = check_plan(c, p))) return rc;
    if (p.slots && (!c.workspace || c.workspace_bytes < p.ml_bytes + p.o_bytes ||
                     reinterpret_cast<uintptr_t>(c.workspace) % 16))
      return fail(kInval, "the workspace must hold %zu bytes on a multiple of 16, got %zu",
                  p.ml_bytes + p.o_bytes, c.workspace ? c.workspace_bytes : 0);
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
    a.chunk = static_cast<int>(mx4_chunk_bytes(c.tokens_per_block, c.num_heads, c.head_size));
    a.slots = p.slots;
    a.scale_log2 = c.scale * kLog2e;
    a.part_o = static_cast<float*>(c.workspace);
    a.any_cut = reinterpret_cast<int*>(static_cast<char*>(c.workspace) + p.o_bytes);
    a.part_ml = reinterpret_cast<float2*>(static_cast<char*>(c.workspace) + p.o_bytes + 16);
    a.tiles_per_block = FastDiv(c.tokens_per_block / kMx4TokenTile);
    a.group_div = FastDiv(c.group_size);
    a.heads_div = FastDiv(c.num_heads);
    hipStream_t s = static_cast<hipStream_t>(stream);
    int dev = 0;
    DeviceGuard guard;
    if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
    (void)hipGetLastError();
    if (c.dtype == FKV_DTYPE_BF16) launch_attention<__bf16>(a, p, c.head_size, s);
    else launch_attention<_Float16>(a, p, c.head_size, s);
    FKV_HIP(hipGetLastError());
    return 0;
  } catch (const std::exception& e) {
    return fail(static_cast<int>(hipErrorUnknown), "exception: %s", e.what());
  } catch (...) {
    return fail(static_cast<int>(hipErrorUnknown), "unknown exception");
  }
}

}  // extern "C"

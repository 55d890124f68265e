// kv_attention.h - what the attention kernels share: the sequences of a call and how
// their rows and keys are dealt out to workgroups (kv_mx4_attention.hip,
// kv_paged_attention.hip).  Not installed; not part of the C ABI.
#pragma once

#include <cstdint>
#include <type_traits>

#include "kv_device.h"

namespace fkv_detail {
#pragma GCC visibility push(hidden)

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

// The sequences of a call and their place in the cache.
struct Sequences {
  const void* table;
  const void* lens;
  const void* starts;                // null: one query a sequence
  int64_t table_row;                 // elements
  int index64;                       // table, lens and starts are int64
  int num_blocks, width;             // of the cache; of a table row
  int batch, heads, group, queries;
  int tokens;                        // of a block
  int causal;
  int slots;                         // workgroups to cut the keys into; 0: uncut
  FastDiv group_div, heads_div;
};

__device__ inline int64_t index_at(const void* p, int64_t i, int is64) {
  return is64 ? static_cast<const int64_t*>(p)[i]
              : static_cast<int64_t>(static_cast<const int32_t*>(p)[i]);
}

struct Seq {
  int first, count;   // its queries
  int keys;           // -1: more than its table row can hold
};
__device__ inline Seq sequence(const Sequences& a, int b) {
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
__device__ inline int tiles_of(const Sequences& a, const Seq& s, int rows_a_tile) {
  return (s.count * a.group + rows_a_tile - 1) / rows_a_tile;
}
template <class P>
__device__ inline int steps_of(const Seq& s) {
  return (max(s.keys, 0) + P::kStep - 1) / P::kStep;
}
// ceil(steps / per_cut), at least 1; in floats, so perhaps one more
__device__ inline int cuts_of(int steps, float inv_per_cut) {
  return max(1, static_cast<int>(steps * inv_per_cut + 0.9999f));
}

// Item `item` of the plan; by_tile: `item` counts tiles, the answer is its first cut.
// P: tokens of a step (kStep), the fewest steps of a cut (kMinSteps) and how many cutting has
// to take off the longest sequence (kCutSteps).
template <class P>
__device__ inline Work find_work(const Sequences& a, int item, int rows_a_tile, bool by_tile) {
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
      total = static_cast<float>(tiles) * static_cast<float>(steps_of<P>(s));
      longest = tiles ? steps_of<P>(s) : 0;
    } else {
      for (int i = lane; i < a.batch; i += 64) {
        const Seq x = sequence(a, i);
        const int n = tiles_of(a, x, rows_a_tile);
        total += static_cast<float>(n) * static_cast<float>(steps_of<P>(x));
        if (n) longest = max(longest, steps_of<P>(x));
      }
    }
    total = bits_f32(lane_value(f32_bits(scan_lanes(total)), 63));
    // at least this many steps a cut; the sum's error and cuts_of's are less than 1 %
    const float even = fmaxf(total * a.heads / a.slots * 1.01f, P::kMinSteps);
    // cuts of even size overflow the slots by the last, short ones: longer cuts until
    // they do not, or to twice the size
    const bool pays = __any(longest >= even + P::kCutSteps);
    inv_per_cut = pays ? 0.5f / even : 0.f;
    for (int i = 0; few && pays && i < 8; ++i) {
      inv_per_cut = 1.f / (even * (1.f + i * 0.125f));
      const int n = lane_value(scan_lanes(tiles * cuts_of(steps_of<P>(s), inv_per_cut)), 63);
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
    const int steps = steps_of<P>(s);
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
__device__ inline Work find_single(const Sequences& a, int item, int rows_a_tile) {
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

// s * scale rounded, then less m
__device__ inline float rounded_less(float s, float scale, float m) {
#pragma clang fp contract(off)
  const float x = s * scale;
  return x - m;
}

// The scale of the scores; not 0, so that -infinity stays that, but the smallest there is,
// with which no finite score comes to more than 2^-21.
__device__ inline float score_scale(float scale_log2) {
  return fmaxf(fabsf(scale_log2), 0x1p-149f);
}

// Row r of a tile: the packed query row, its head and the keys it sees.
struct Row {
  int64_t at;
  int head, visible;
};
__device__ inline Row row_of(const Sequences& a, const Seq& s, int r, int kv_head) {
  const int pos = a.group_div.div(r);
  Row row;
  row.at = static_cast<int64_t>(s.first) + pos;
  row.head = kv_head * a.group + (r - pos * a.group);
  const int keys = max(s.keys, 0);
  row.visible = a.causal ? max(0, keys - s.count + pos + 1) : keys;
  return row;
}

// Which item of the plan, and which K/V head, a workgroup has.  Workgroups go round the
// 8 XCDs.  Where K and V are read once, an item's heads are on one XCD, so that a
// block is read whole by one L2 at about one time.  Where many tiles read them, a
// head's tiles are on one XCD if there are 8 heads.
constexpr int kXcds = 8;
struct Place {
  int item, head;
};
__device__ inline Place heads_together(const Sequences& a, int block) {
  const int nth = block / kXcds, group = a.heads_div.div(nth);
  return {group * kXcds + block % kXcds, nth - group * a.heads};
}
__device__ inline Place heads_apart(const Sequences& a, int block) {
  const int item = a.heads_div.div(block);
  return {item, block - item * a.heads};
}
// The number that a cut's part of the workspace has.
__device__ inline int64_t part_of(const Sequences& a, int item, int head) {
  return static_cast<int64_t>(item) * a.heads + head;
}

#pragma GCC visibility pop
}  // namespace fkv_detail

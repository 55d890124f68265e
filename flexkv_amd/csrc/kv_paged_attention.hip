// kv_paged_attention.hip - attention over a paged KV cache of bf16 or fp16, and what each
// cached token got of it: for query i of head hq in a sequence, with K/V head h = hq / group,
//
//   o = sum_t p_t v_t / sum_t p_t,   p_t = exp(scale q . k_t - max),   t <= its own position
//   weights[h][t] += sum over those queries and heads of p_t / sum p
//
// The queries of a group and of neighbouring positions are the rows of one tile (row =
// position * group + head in the group), so K and V are read once for all of them.
//
// Both products are matrix instructions with the tokens, then the elements, as rows of the
// result and the query rows as columns.  S = K Q^T comes out with some tokens of one row in a
// lane, which is the layout of the second product's operand if its tokens are taken in that
// order, so P never leaves its lane.  bf16 weights of 8 significant bits, fp16 ones of 11
// (of what is at least 2^-21 of the largest; below, a multiple of 2^-31 of it): a result is off by
// half a step of its type at most, less where the roundings average out over the keys.  The sum
// they are divided by is of the unrounded ones.
//
// Softmax: one pass, running maximum and sum per row in 32 bits, in units of log2.
// The maximum (in fp16 a 2^7th of it, see Mat) is a reference that follows only when a score passes it
// by 2^8, so most steps neither compare across lanes nor scale the sums.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <type_traits>
#include <utility>

#include "kv_attention.h"
#include "kv_paged.h"

using namespace fkv_detail;

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t Vec2 __attribute__((ext_vector_type(2)));
typedef uint32_t Vec4 __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

// The matrix instructions of a type, by how much (in units of log 2) a row's reference is below its
// largest score when it is set, and the weight up to which a score may pass it.  fp16 has 2^16 above 1
// and nothing below 2^-25, so weights start at 2^7 and may grow to 2^15: with 65536 keys of 1.4 * 2^-24
// of the largest, references at the largest lose 29 % of what these add, and 0.2 % so.
template <class T>
struct Mat;
template <>
struct Mat<__bf16> {
  typedef v8bf Op;
  static __device__ inline v4f mul16(Op a, Op b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ inline v16f mul32(Op a, Op b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) { return pack_bf16(a, b); }
  static __device__ inline float low(uint32_t u) { return bits_f32(u << 16); }
  static __device__ inline float high(uint32_t u) { return bits_f32(u & 0xffff0000u); }
  static constexpr uint32_t kExponents = 0x7f807f80u;
  static constexpr float kBelow = 0.f, kMost = kSlack;
};
template <>
struct Mat<_Float16> {
  typedef v8h Op;
  typedef _Float16 v2h __attribute__((ext_vector_type(2)));
  static __device__ inline v4f mul16(Op a, Op b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ inline v16f mul32(Op a, Op b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  static __device__ inline uint32_t pack(float a, float b) {
    v2h r;
    r[0] = static_cast<_Float16>(a);
    r[1] = static_cast<_Float16>(b);
    return __builtin_bit_cast(uint32_t, r);
  }
  static __device__ inline float low(uint32_t u) {
    return static_cast<float>(__builtin_bit_cast(v2h, u)[0]);
  }
  static __device__ inline float high(uint32_t u) {
    return static_cast<float>(__builtin_bit_cast(v2h, u)[1]);
  }
  static constexpr uint32_t kExponents = 0x7c007c00u;
  static constexpr float kBelow = 7.f, kMost = kSlack * 128.f;
};

// Whether one of the two elements of a register is an infinity or a NaN.
template <class T>
__device__ inline bool not_finite(uint32_t u) {
  constexpr uint32_t lo = Mat<T>::kExponents & 0xffffu, hi = Mat<T>::kExponents & 0xffff0000u;
  return (u & lo) == lo || (u & hi) == hi;
}

struct Args : Sequences {
  const char* q;
  char* out;
  float* lse;                        // null: not asked for
  int64_t q_row, q_head, out_row, out_head;   // bytes
  int64_t lse_row, lse_head;         // elements
  Half k, v;
  float scale_log2;
  int together;                      // how heads lie on the XCDs, see Place
  FastDiv tokens_div;
  float2* part_ml;                   // [part][row]: maximum and sum
  float* part_o;                     // [part][row][element]
  int* any_cut;                      // whether some tile has more than one cut
  // for the tokens' weights, all null where they are not asked for
  float* weights;
  int64_t w_seq, w_head;             // elements
  float2* stats;                     // [query][head]: reference and 1 / sum of a row
  // [query][head][token]: the scores before they are scaled, where the kernel for few rows leaves
  // them; null where they are made again
  float* scores;
  int64_t scores_row;
  // workgroups that share the rows where they are made again, and, of more than one, what each adds
  // up, [sequence][head][share][token]
  int shares;
  FastDiv shares_div;
  float* share_sums;
  int64_t share_row;
};

// Eight elements of a query: their negatives where the scale is negative, so that it is not looked
// at again.
template <class T>
__device__ inline typename Mat<T>::Op query_part(const char* p, bool negate) {
  const uint32_t flip = negate ? 0x80008000u : 0u;
  return __builtin_bit_cast(typename Mat<T>::Op, *reinterpret_cast<const Vec4*>(p) ^ flip);
}

// 16 bytes of device memory; not a flat access, which would wait for LDS as well.
template <class V>
__device__ inline V load(uint64_t address) {
  return *reinterpret_cast<const __attribute__((address_space(1))) V*>(address);
}

// The same of what is read once and by one instruction: past the caches (V so: 32 sequences of 8192
// keys, 8 heads: 188 us for 205, 5.7 TB/s for 5.3; K as well, in whole rows: 178).
template <class V>
__device__ inline V load_once(uint64_t address) {
  return __builtin_nontemporal_load(
      reinterpret_cast<const __attribute__((address_space(1))) V*>(address));
}

// ---------------------------------------------------------------------------
// Where the rows of tokens lie

// A block id as it lies in the table, two words of which the second is the first again in a table
// of 32 bits: made a number where it is used, since what is done with a load's result where it is
// asked for waits for all loads before it.
struct RawId {
  uint32_t lo, hi;
};
__device__ inline RawId ask_block(const Args& a, int seq, int token) {
  const uint64_t at = reinterpret_cast<uint64_t>(a.table) +
                      (static_cast<uint64_t>(seq * a.table_row + a.tokens_div.div(token))
                       << (a.index64 ? 3 : 2));
  return {load<uint32_t>(at), load<uint32_t>(at + (a.index64 ? 4 : 0))};
}
__device__ inline int64_t block_id(const Args& a, const RawId& r) {
  const uint32_t hi = a.index64 ? r.hi : static_cast<uint32_t>(static_cast<int32_t>(r.lo) >> 31);
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | r.lo);
}
__device__ inline int64_t block_id(const Args& a, int seq, int token) {
  return block_id(a, ask_block(a, seq, token));
}
// The row of a token in block `id`, of one half and head.  A block outside the cache is block 0
// here (and noted by whoever calls).
__device__ inline bool outside(const Args& a, int64_t id) { return id < 0 || id >= a.num_blocks; }
__device__ inline uint64_t row_address(const Args& a, const Half& x, int64_t id, int token,
                                       int head) {
  const int in_block = token - a.tokens_div.div(token) * static_cast<int>(a.tokens_div.d);
  return reinterpret_cast<uint64_t>(x.p) + (outside(a, id) ? 0 : id) * x.block +
         in_block * x.token + head * x.head;
}

constexpr int kNoToken = 0x7fffffff;
// The least value over the wavefront.
__device__ inline int least(int v) {
#pragma unroll
  for (int i = 1; i < 64; i *= 2) v = min(v, __shfl_xor(v, i));
  return v;
}

// ---------------------------------------------------------------------------
// What a row ends with

// The reference and the factor that its weights take.  No weight at all: 0 for a row that
// sees no key, NaN for one whose scores are all below what 32 bits hold.
__device__ inline float inverse(float l, int visible) {
  return l == 0.f ? (visible ? bits_f32(0x7fc00000u) : 0.f) : 1.f / l;
}
__device__ inline void write_stats(const Args& a, const Row& row, float m, float l) {
  if (a.lse)
    a.lse[row.at * a.lse_row + row.head * a.lse_head] =
        l == 0.f ? (row.visible ? bits_f32(0x7fc00000u) : -INFINITY)
                 : (m + __builtin_amdgcn_logf(l)) * kLn2;
  if (a.stats)
    a.stats[row.at * (a.heads * a.group) + row.head] = make_float2(m, inverse(l, row.visible));
}
// A result as the output's type holds it: the weights' roundings may carry one past the largest value
// of V, and fp16 has no more than 65504.
template <class T>
__device__ inline float held(float x) {
  if constexpr (std::is_same<T, _Float16>::value)
    return fabsf(x) < INFINITY ? __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f) : x;
  return x;
}
// N neighbouring elements from `first` on as the output's type.
template <class T, int N>
__device__ inline void write_elements(const Args& a, const Row& row, int first, const float (&o)[N],
                                      float inv) {
  static_assert(N % 2 == 0, "");
  uint32_t w[N / 2];
#pragma unroll
  for (int j = 0; j < N; j += 2) w[j / 2] = Mat<T>::pack(held<T>(o[j] * inv), held<T>(o[j + 1] * inv));
  char* const out = a.out + row.at * a.out_row + row.head * a.out_head + first * 2;
  if constexpr (N == 2) {
    *reinterpret_cast<uint32_t*>(out) = w[0];
  } else if constexpr (N % 8 == 0) {
#pragma unroll
    for (int x = 0; x < N / 2; x += 4)
      *reinterpret_cast<Vec4*>(out + x * 4) = Vec4{w[x], w[x + 1], w[x + 2], w[x + 3]};
  } else {
#pragma unroll
    for (int x = 0; x < N / 2; x += 2)
      *reinterpret_cast<Vec2*>(out + x * 4) = Vec2{w[x], w[x + 1]};
  }
}

// ---------------------------------------------------------------------------
// Few rows: K and V go to registers as they are read, and the wavefronts of a workgroup take
// the 32-token steps of its tile in turn.  Bound by memory where there are many keys: 32 sequences of up
// to 8192, 8 heads of 128 elements, 718 MB in 126 us (5.7 TB/s; reads alone reach 7.1), of 256 elements
// twice that at 6.2.  Short calls are bound by the start, lengths, block ids, keys and the sum over the
// wavefronts one after the other: 777 keys 10 us.

constexpr int kRows = 16;          // rows of a tile: columns of a matrix instruction
struct FewPlan {
  static constexpr int kStep = 32;       // tokens: two tiles of 16, k of the second product
  // Steps of a workgroup where the keys are dealt out: a sequence of 4906 keys 19 us, with 32 of them
  // 24, with 8 18; one of 65536 keys of one head, whose parts one tile's join adds up, 26, 25 and 36.
  static constexpr int kMinSteps = 16;
};
constexpr int kStep = FewPlan::kStep;

// How the keys are dealt out, where they are: the 32-token steps of all tiles, sequence by
// sequence, are one line for every head, and workgroup j of a head's `slots` has the steps from
// j * per on, `per` of them.  All workgroups end at about one time, whatever the lengths; a tile that
// several have a piece of is joined afterwards.  The lengths are read here, on the device, by
// every wavefront, sequence b = lane, then 64 further on.  A tile has a step at least, so that its
// rows are written.
struct Piece {
  int seq, tile;      // < 0: none
  int from, steps;    // its first step in the tile, and all steps of the tile
  int start;          // of the tile on the line
  Seq s;
};
struct Line {
  Seq s;
  int tiles, steps;
  __device__ Line(const Sequences& a, int b, int rows_a_tile) : s{0, 0, 0}, tiles(0), steps(1) {
    if (b >= a.batch) return;
    s = sequence(a, b);
    tiles = tiles_of(a, s, rows_a_tile);
    steps = max(1, steps_of<FewPlan>(s));
  }
};
// Steps of all tiles, and those that a workgroup has: an even share, but no less than
// kMinSteps, or the longest tile if that is shorter.  `line`: the first 64 sequences'.
__device__ inline int deal(const Sequences& a, int rows_a_tile, const Line& line, int* total) {
  const int lane = threadIdx.x & 63;
  int sum = 0, longest = 0;
  for (int b = lane; b < a.batch; b += 64) {
    const Line x = b == lane ? line : Line(a, b, rows_a_tile);
    sum += x.tiles * x.steps;
    if (x.tiles) longest = max(longest, x.steps);
  }
  *total = lane_value(scan_lanes(sum), 63);
  longest = uniform(-least(-longest));
  return max(uniform((*total + a.slots - 1) / a.slots), min(longest, FewPlan::kMinSteps));
}
// Where step `at` of the line is; by_tile: where tile `at` starts.
__device__ inline Piece find_piece(const Sequences& a, int rows_a_tile, const Line& line, int at,
                                   bool by_tile) {
  const int lane = threadIdx.x & 63;
  int before = 0, tiles_before = 0;
  for (int b0 = 0; b0 < a.batch; b0 += 64) {
    const Line x = b0 ? Line(a, b0 + lane, rows_a_tile) : line;
    const int ends = scan_lanes(x.tiles * x.steps), tile_ends = scan_lanes(x.tiles);
    const uint64_t later =
        __ballot(by_tile ? tiles_before + tile_ends > at : before + ends > at);
    if (later) {
      const int l = __builtin_ctzll(later);
      const int n = lane_value(x.tiles, l), steps = lane_value(x.steps, l);
      const int first = before + lane_value(ends, l) - n * steps;
      const int tile = by_tile ? at - (tiles_before + lane_value(tile_ends, l) - n)
                               : uniform((at - first) / steps);
      const int start = first + tile * steps;
      return {b0 + l, tile, by_tile ? 0 : at - start, steps, start,
              {lane_value(x.s.first, l), lane_value(x.s.count, l), lane_value(x.s.keys, l)}};
    }
    before += lane_value(ends, 63);
    tiles_before += lane_value(tile_ends, 63);
  }
  return {-1, 0, 0, 0, 0, {0, 0, 0}};
}
// A tile for each workgroup, uncut, one query a sequence: nothing but that length is read.
__device__ inline Piece find_alone(const Sequences& a, int item, int rows_a_tile) {
  const Work w = find_single(a, item, rows_a_tile);
  return {w.seq, w.tile, 0, max(1, steps_of<FewPlan>(w.s)), 0, w.s};
}
// A workgroup has parts of two tiles at most: of one that starts before it, and of one that
// starts in it and goes on after it.
__device__ inline int64_t part_of_piece(const Sequences& a, int slot, int head, bool starts) {
  return (static_cast<int64_t>(slot) * a.heads + head) * 2 + (starts ? 1 : 0);
}

// A row of K or V in LDS is D / 8 pieces of 16 bytes, piece c at c ^ f(row).  K is read with 8 and
// more neighbouring rows of one piece at a time, V (transposed) with 4 neighbouring rows of 4
// pieces: so that either takes all banks.
template <int D>
__device__ constexpr int k_swizzle(int row) {
  return D == 64 ? row & 7 : row & 15;
}
template <int D>
__device__ constexpr int v_swizzle(int row) {
  return D == 64 ? (row >> 1 & 1) << 2 | (row >> 2 & 3) : (row & 3) << 2 | (row >> 2 & 3);
}

// The queries of 16 rows: lane (row, quad) holds elements 32 s + 8 quad .. + 7.
template <class T, int D>
struct Query {
  typename Mat<T>::Op part[D / 32];
};
// What a lane loads of a step: of K whole rows, D / 8 lanes a row, which are put into the order
// of the queries through LDS; of V the elements (D / 16) * (lane & 15) on of tokens 16 h + 4 quad + i.
template <int D>
struct Keys {
  Vec4 part[D / 16];
};
template <int D>
struct Values {
  static constexpr int kWords = D / 32;
  uint32_t part[2][4][kWords];
};
// A row tile's state: lane (row, quad) holds row `lane & 15`.
template <int D>
struct State {
  v4f o[D / 16];   // o[j][i]: element (D / 16) * (4 quad + i) + j
  float m, l;      // the reference; the sum of this lane's tokens
};

// Calls f with the numbers from 0 to N - 1, as types.
template <int N, class F, int... I>
__device__ __attribute__((always_inline)) inline void each_index(F f,
                                                                 std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, class F>
__device__ __attribute__((always_inline)) inline void each_index(F f) {
  each_index<N>(f, std::make_integer_sequence<int, N>());
}

// The address of a row, which a lane finds and tells the 16 lanes of its quad: lane LANE's, or, of a
// pair, to the first 8 lanes lane LANE's and to the others the next one's.
struct Rows {
  uint32_t lo, hi;
};
template <int LANE, bool PAIR>
__device__ inline uint32_t told(uint32_t x) {
  constexpr int kBroadcast = 0x150;      // of a lane to its 16
  const int y = __builtin_amdgcn_mov_dpp(x, kBroadcast + LANE, 0xf, 0xf, true);
  if constexpr (!PAIR) return y;
  else return __builtin_amdgcn_update_dpp(y, x, kBroadcast + LANE + 1, 0xf, 0xc, false);
}
template <int LANE, bool PAIR>
__device__ inline uint64_t told(const Rows& r) {
  return __builtin_bit_cast(uint64_t, Vec2{told<LANE, PAIR>(r.lo), told<LANE, PAIR>(r.hi)});
}

// Which rows of a step's K and V the lanes of a quad find for it: lane e, below 8, one of K's loads and
// the others V's.  Of 256 elements K's loads are 16, so K's rows and V's are found one after the other.
template <int D>
struct StepPlaces {
  static constexpr int kFinds = D == 256 ? 2 : 1;
  // the N-th finding
  template <int N>
  static __device__ inline bool value(int lane) {
    return D == 256 ? N == 1 : (lane & 8) != 0;
  }
  template <int N>
  static __device__ inline int token(int lane) {
    const int e = lane & 15, quad = lane >> 4;
    const int of_v = 16 * (e >> 2 & 1) + 4 * quad + (e & 3);
    if constexpr (D == 256) return N ? of_v : 2 * e + (quad >> 1);
    const int of_k = D == 64 ? 8 * (e >> 1 & 3) + 2 * quad + (e & 1) : 4 * (e & 7) + quad;
    return e < 8 ? of_k : of_v;
  }
};
template <int D>
struct StepRows {
  Rows of[StepPlaces<D>::kFinds];
};
template <int D>
struct StepIds {
  RawId of[StepPlaces<D>::kFinds];
};

template <int D>
__device__ inline void load_keys(const StepRows<D>& r, int lane, Keys<D>& k) {
  const int piece = lane % (D / 8) * 16;
  each_index<D / 16>([&](auto j) __attribute__((always_inline)) {
    k.part[j] = load_once<Vec4>(told<D == 64 ? 2 * j : j, D == 64>(r.of[0]) + piece);
  });
}
// A wavefront's 32 rows of K in LDS.
template <int D>
__device__ inline void put_keys(const Keys<D>& k, int lane, char* lds) {
  constexpr int kPieces = D / 8, kRowsAtOnce = 64 / kPieces;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    const int row = j * kRowsAtOnce + lane / kPieces;
    *reinterpret_cast<Vec4*>(lds + row * D * 2 + ((lane % kPieces ^ k_swizzle<D>(row)) << 4)) =
        k.part[j];
  }
}
// D / 16 elements of a row
template <int D>
__device__ inline void load_part(uint64_t p, uint32_t (&x)[D / 32]) {
  if constexpr (D == 64) {
    const Vec2 u = load_once<Vec2>(p);
    x[0] = u[0], x[1] = u[1];
  } else {
#pragma unroll
    for (int w = 0; w < D / 32; w += 4) {
      const Vec4 u = load_once<Vec4>(p + 4 * w);
#pragma unroll
      for (int y = 0; y < 4; ++y) x[w + y] = u[y];
    }
  }
}
template <int D>
__device__ inline void load_values(const StepRows<D>& r, int lane, Values<D>& v) {
  each_index<8>([&](auto x) __attribute__((always_inline)) {
    load_part<D>(told<D == 256 ? x : 8 + x, false>(r.of[D == 256 ? 1 : 0]) +
                     (lane & 15) * (D / 8),
                 v.part[x / 4][x % 4]);
  });
}

// s[r][h][i] = q[r] . k of token 16 h + 4 quad + i
template <class T, int D, int R>
__device__ inline void scores(const Query<T, D> (&q)[R], const char* lds, int lane,
                              v4f (&s)[R][2]) {
  using Op = typename Mat<T>::Op;
  const int at = (lane & 15) * D * 2 + (((lane >> 4) ^ k_swizzle<D>(lane & 15)) << 4);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
#pragma unroll
    for (int r = 0; r < R; ++r) s[r][h] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int x = 0; x < D / 32; ++x) {
      const Op k = __builtin_bit_cast(
          Op, *reinterpret_cast<const Vec4*>(lds + (at ^ (x % 4 * 64)) + x / 4 * 256 +
                                             16 * h * D * 2));
#pragma unroll
      for (int r = 0; r < R; ++r) s[r][h] = Mat<T>::mul16(k, q[r].part[x], s[r][h]);
    }
  }
}

__device__ inline void hide(v4f (&s)[2], int at, int visible, int quad) {
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (at + 16 * h + quad * 4 + i >= visible) s[h][i] = -INFINITY;
}

// The scores as weights p; returns their sum, which is over kMost where one of them passes
// the reference by more than that.
__device__ inline float weigh(const v4f (&s)[2], float m, float scale_log2, bool coarse,
                              float (&p)[8]) {
  float sum = 0.f;
#pragma unroll
  for (int x = 0; x < 8; ++x) {
    const float score = s[x / 4][x % 4];
    p[x] = __builtin_amdgcn_exp2f(coarse ? rounded_less(score, scale_log2, m)
                                         : __builtin_fmaf(score, scale_log2, -m));
    sum = x ? sum + p[x] : p[x];
  }
  return sum;
}

// Elements j and j + 1 of a lane's 8 tokens of V as operands.
template <class T, int D>
__device__ inline void columns(const Values<D>& v, int j, typename Mat<T>::Op& even,
                               typename Mat<T>::Op& odd) {
  uint32_t e[4], d[4];
#pragma unroll
  for (int x = 0; x < 4; ++x) {
    const uint32_t lo = v.part[x / 2][2 * (x % 2)][j / 2], hi = v.part[x / 2][2 * (x % 2) + 1][j / 2];
    e[x] = __builtin_amdgcn_perm(hi, lo, 0x05040100u);
    d[x] = __builtin_amdgcn_perm(hi, lo, 0x07060302u);
  }
  even = __builtin_bit_cast(typename Mat<T>::Op, make_uint4(e[0], e[1], e[2], e[3]));
  odd = __builtin_bit_cast(typename Mat<T>::Op, make_uint4(d[0], d[1], d[2], d[3]));
}

template <class T, int D>
__device__ inline bool any_not_finite(const Values<D>& v) {
  bool any = false;
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int w = 0; w < Values<D>::kWords; ++w) any |= not_finite<T>(v.part[h][i][w]);
  return __any(any);
}

// A step whose values hold an infinity or a NaN that some row may not see: a weight of 0 does not
// leave it out of a matrix product, so the products are made one by one.
template <class T, int D>
__device__ inline void add_one_by_one(const Args& a, int seq, int head, int at, int keys,
                                      int visible, int lane, const float (&p)[8], State<D>& st) {
  const int quad = lane >> 4;
#pragma unroll 1
  for (int x = 0; x < 32; ++x) {
    const int token = at + x;
    if (token >= keys) break;
    const int at_x = x / 16 * 4 + x % 4;
    float w = p[0];
#pragma unroll
    for (int y = 1; y < 8; ++y) w = y == at_x ? p[y] : w;
    w = __shfl(w, (lane & 15) + 16 * (x / 4 % 4));
    const uint64_t row = row_address(a, a.v, block_id(a, seq, token), token, head);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u[D / 32];
      load_part<D>(row + (4 * quad + i) * (D / 8), u);
      if (token >= visible) continue;
#pragma unroll
      for (int j = 0; j < D / 16; j += 2) {
        st.o[j][i] += w * Mat<T>::low(u[j / 2]);
        st.o[j + 1][i] += w * Mat<T>::high(u[j / 2]);
      }
    }
  }
}

template <int D>
__device__ inline void clear(State<D>& st) {
  st.m = kNothing;
  st.l = 0.f;
#pragma unroll
  for (int j = 0; j < D / 16; ++j) st.o[j] = {0.f, 0.f, 0.f, 0.f};
}

constexpr int few_waves_a_simd(int dim) { return dim == 256 ? 1 : 2; }

template <class T, int D, int R, int W>
__global__ __launch_bounds__(64 * W, few_waves_a_simd(D)) void attend_few_kernel(const Args a) {
  using Op = typename Mat<T>::Op;
  constexpr int NT = D / 16, kRowsATile = kRows * R;
  // K of a wavefront's step, then a row tile's sums of every wavefront
  __shared__ v4f shared[W * NT][64];
  __shared__ float sum_m[W][R][16], sum_l[W][R][16];
  const Place at = a.together ? heads_together(a, blockIdx.x) : heads_apart(a, blockIdx.x);
  const int wave = uniform(threadIdx.x >> 6);
  char* const k_lds = reinterpret_cast<char*>(shared[wave * NT]);
  const float scale_log2 = score_scale(a.scale_log2);
  // nothing but its own sequence's length is read where each has a tile for one workgroup
  const bool alone = !a.slots && !a.starts;
  const Line line(a, alone ? a.batch : threadIdx.x & 63, kRowsATile);
  int pos = 0, pos_end = 0;
  if (a.slots) {
    int total;
    const int per = deal(a, kRowsATile, line, &total);
    // up to 2^31 steps of 2^10 workgroups: both in 64 bits
    pos = static_cast<int>(min(static_cast<int64_t>(at.item) * per, static_cast<int64_t>(total)));
    pos_end = static_cast<int>(min(static_cast<int64_t>(pos) + per, static_cast<int64_t>(total)));
    if (pos == pos_end) return;
  }
  for (bool again = false;; again = true) {
    if (again) __syncthreads();      // the sums of the tile before have been read
    int lane = threadIdx.x & 63;
    asm volatile("" : "+v"(lane));   // what follows from it is worked out for each tile, not kept
    int quad = lane >> 4;
    const Piece w = alone ? find_alone(a, at.item, kRowsATile)
                          : find_piece(a, kRowsATile, line, a.slots ? pos : at.item, !a.slots);
    if (w.seq < 0) return;
    const int to = a.slots ? min(w.steps, w.from + pos_end - pos) : w.steps;
    const bool whole = w.from == 0 && to == w.steps;
    const int first = w.tile * kRowsATile;
    const int rows = min(kRowsATile, w.s.count * a.group - first);
    auto row_at = [&](int n) { return row_of(a, w.s, first + min(n, rows - 1), at.head); };
    const int keys = max(w.s.keys, 0);
    int visible[R];
#pragma unroll
    for (int r = 0; r < R; ++r) visible[r] = row_at(16 * r + (lane & 15)).visible;
    // of the rows, in order, the first sees the fewest, the last the most
    const int fewest = lane_value(visible[0], 0), most = lane_value(visible[R - 1], 15);
    const int end = min((most + kStep - 1) / kStep, to);
    int step = w.from + wave;
    const bool any = step < end;
    // the block ids are asked for a step ahead of the rows, the rows a step ahead of their use; past
    // the last key everything is of that one again
    int bad = kNoToken;
    using P = StepPlaces<D>;
    auto ask = [&](int s) __attribute__((always_inline)) {
      StepIds<D> ids;
      each_index<P::kFinds>([&](auto n) __attribute__((always_inline)) {
        ids.of[n] = ask_block(a, w.seq, min(s * kStep + P::template token<n>(lane), keys - 1));
      });
      return ids;
    };
    auto find = [&](int s, const StepIds<D>& ids) __attribute__((always_inline)) {
      StepRows<D> rows;
      each_index<P::kFinds>([&](auto n) __attribute__((always_inline)) {
        const int t = min(s * kStep + P::template token<n>(lane), keys - 1);
        const int64_t id = block_id(a, ids.of[n]);
        if (outside(a, id)) bad = min(bad, t);
        const uint64_t p =
            row_address(a, P::template value<n>(lane) ? a.v : a.k, id, t, at.head);
        rows.of[n] = {static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32)};
      });
      return rows;
    };
    Keys<D> k;
    Values<D> v;
    StepIds<D> ids{};
    if (any) ids = ask(step);
    Query<T, D> q[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const Row row = row_at(16 * r + (lane & 15));
      const char* const p = a.q + row.at * a.q_row + row.head * a.q_head + quad * 16;
#pragma unroll
      for (int x = 0; x < D / 32; ++x)
        q[r].part[x] = query_part<T>(p + 64 * x, a.scale_log2 < 0.f);
    }
    if (any) {
      const StepRows<D> next = find(step, ids);
      ids = ask(step + W);
      load_keys<D>(next, lane, k);
      load_values<D>(next, lane, v);
    }
    // waited for here: in the loop the wait would be one for all loads, at every step
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int x = 0; x < D / 32; ++x) asm volatile("" : "+v"(q[r].part[x]));
    float slack = Mat<T>::kMost;
    State<D> st[R];
#pragma unroll
    for (int r = 0; r < R; ++r) clear(st[r]);
    // where this lane's scores go; they are not kept of more than one tile of 16 rows
    const bool scores_kept = R == 1 && a.scores && (lane & 15) < rows;
    const Row scores_of = row_at(lane & 15);
    const uint64_t scores_at = reinterpret_cast<uint64_t>(
        a.scores + (scores_of.at * (a.heads * a.group) + scores_of.head) * a.scores_row + quad * 4);
    float p[R][8];
    // A step's scores, with K in LDS, its weights, and what these change of the rows' states.
    auto weights = [&]() __attribute__((always_inline)) {
      const int token = step * kStep;
      v4f s[R][2];
      scores<T, D, R>(q, k_lds, lane, s);
      float l[R];
      bool passes = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        if (token + kStep > fewest) hide(s[r], token, visible[r], quad);
        if (scores_kept) {
          const uint64_t to = scores_at + static_cast<uint64_t>(token) * 4;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            *reinterpret_cast<__attribute__((address_space(1))) v4f*>(to + 64 * h) = s[r][h];
        }
        l[r] = weigh(s[r], st[r].m, scale_log2, false, p[r]);
        passes |= l[r] > slack;
      }
      if (__any(passes)) {
        // Some score passes its row's reference: the references follow, and the weights are made
        // again; at every step from then on, where a reference is kCoarse or more.
        bool any_coarse = false;
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float top = -INFINITY;
#pragma unroll
          for (int x = 0; x < 8; ++x) top = fmaxf(top, s[r][x / 4][x % 4] * scale_log2);
          const float m = fmaxf(st[r].m, max_over_quads(top) - Mat<T>::kBelow);
          const float fade = __builtin_amdgcn_exp2f(st[r].m - m);
          st[r].m = m;
          st[r].l *= fade;
#pragma unroll
          for (int j = 0; j < NT; ++j) st[r].o[j] *= fade;
          const bool coarse = fabsf(m) >= kCoarse && m != kNothing;
          any_coarse |= coarse;
          l[r] = weigh(s[r], m, scale_log2, coarse, p[r]);
        }
        slack = __any(any_coarse) ? -1.f : Mat<T>::kMost;
      }
#pragma unroll
      for (int r = 0; r < R; ++r) st[r].l += l[r];
    };
    auto add_values = [&]() __attribute__((always_inline)) {
      Op weight[R];
#pragma unroll
      for (int r = 0; r < R; ++r)
        weight[r] = __builtin_bit_cast(
            Op, make_uint4(Mat<T>::pack(p[r][0], p[r][1]), Mat<T>::pack(p[r][2], p[r][3]),
                           Mat<T>::pack(p[r][4], p[r][5]), Mat<T>::pack(p[r][6], p[r][7])));
#pragma unroll
      for (int j = 0; j < NT; j += 2) {
        Op even, odd;
        columns<T, D>(v, j, even, odd);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          st[r].o[j] = Mat<T>::mul16(even, weight[r], st[r].o[j]);
          st[r].o[j + 1] = Mat<T>::mul16(odd, weight[r], st[r].o[j + 1]);
        }
      }
    };
    // a step that some row does not see all of, and whose values hold an infinity or a NaN
    auto odd_values = [&]() __attribute__((always_inline)) {
      return step * kStep + kStep > fewest && any_not_finite<T, D>(v);
    };
    bool one_by_one = false;
    for (; step < end; step += W) {
      if (odd_values()) {
        one_by_one = true;
        break;
      }
      const StepRows<D> next = find(step + W, ids);
      ids = ask(step + 2 * W);
      put_keys<D>(k, lane, k_lds);
      load_keys<D>(next, lane, k);
      weights();
      add_values();
      load_values<D>(next, lane, v);
    }
    if (one_by_one) {
      // All over again, and without loads ahead: a loop that goes on with the sums costs the other its
      // registers.
      asm volatile("" : "+v"(lane));
      quad = lane >> 4;
#pragma unroll
      for (int r = 0; r < R; ++r) clear(st[r]);
      slack = Mat<T>::kMost;
#pragma unroll 1
      for (step = w.from + wave; step < end; step += W) {
        const StepRows<D> here = find(step, ask(step));
        load_keys<D>(here, lane, k);
        load_values<D>(here, lane, v);
        put_keys<D>(k, lane, k_lds);
        weights();
        if (!odd_values()) {
          add_values();
          continue;
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
          add_one_by_one<T, D>(a, w.seq, at.head, step * kStep, keys, visible[r], lane, p[r], st[r]);
      }
    }
    bad = least(bad);
    // The wavefronts' sums, each to the common reference; wavefront i (and i + 4, half
    // each) adds up the elements [][i] of all.
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const float l = sum_over_quads(st[r].l);
      if (quad == 0) {
        sum_m[wave][r][lane] = st[r].m;
        const bool lost = w.s.keys < 0 || visible[r] > bad;
        sum_l[wave][r][lane] = lost ? bits_f32(0x7fc00000u) : l;
      }
    }
    __syncthreads();
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
      if (r) __syncthreads();
#pragma unroll
      for (int j = 0; j < NT; ++j) shared[wave * NT + j][lane] = st[r].o[j] * f;
      __syncthreads();
      float sums[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        sums[j] = 0.f;
#pragma unroll
        for (int x = 0; x < W; ++x)
          sums[j] += reinterpret_cast<const float*>(shared[x * NT + j0 + j])[lane * 4 + i];
      }
      const int n = 16 * r + (lane & 15), element = NT * (4 * quad + i) + j0;
      if (n >= rows) continue;
      if (whole) {
        const Row row = row_at(n);
        write_elements<T, NJ>(a, row, element, sums, inverse(l, visible[r]));
        if (wave == 0 && quad == 0) write_stats(a, row, m, l);
      } else {
        const int64_t part =
            (part_of_piece(a, at.item, at.head, w.from == 0) * R + r) * kRows + (lane & 15);
        if (wave == 0 && quad == 0) a.part_ml[part] = make_float2(m, l);
#pragma unroll
        for (int j = 0; j < NJ; ++j) a.part_o[part * D + element + j] = sums[j];
      }
    }
    pos += to - w.from;
    if (pos >= pos_end) return;
  }
}

// ---------------------------------------------------------------------------
// Many rows: each wavefront has 32 rows, and all of a workgroup share 64 tokens of K and V at a
// time in LDS.  There are two places for them, and the next tile goes straight from memory into the
// one while the other is used.  32 rows a wavefront, since each reads all of K and V from LDS; two
// workgroups a compute unit (one of 256 elements), so that the exponentials of one pass beside the
// products of the other.  Bound by both: 2048 queries of 32 heads over 8192 keys 250 us, 960 TFLOP/s,
// the matrix units at work for 54 % of the cycles (heads of 256: 517 us, 930; of 64: 160, 750).

struct ManyPlan {
  static constexpr int kStep = 64;       // tokens of a tile
  // Steps of a workgroup where the keys are cut, and that cutting has to take off the longest
  // sequence.  64 queries over 2000 keys 25 us, with 16 for both 32, with 4 23; 128 queries of two heads
  // over 8000 keys 27, 34 and 32.
  static constexpr int kMinSteps = 8, kCutSteps = 8;
};
constexpr int kTile = ManyPlan::kStep;

typedef short v4s __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) v4s* LdsTransposed;

// 16 bytes a lane from memory to LDS, lane after lane from `to` on.
__device__ inline void load_to_lds(uint64_t from, char* to) {
  __builtin_amdgcn_global_load_lds(reinterpret_cast<const __attribute__((address_space(1))) void*>(from),
                                   (__attribute__((address_space(3))) void*)to, 16, 0, 0);
}
__device__ inline void wait_for_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
// The order of the instructions from the last barrier on: AHEAD reads of LDS, then, N times, M
// matrix instructions and R reads, so that a read's latency passes behind the products before it.
template <int AHEAD, int N, int M, int R>
__device__ inline void reads_ahead() {
  __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x008, M, 0);
    __builtin_amdgcn_sched_group_barrier(0x100, R, 0);
  }
}

// The 16 rows of a tile that a wavefront brings (of K and of V), D / 8 lanes each, in the quads of 16
// lanes: lane e of a quad finds row e of what its quad loads, [tile][K|V][pass][row in the quad], and
// tells it to all by a broadcast within the quad.  Rows of 256 elements take two quads, which both
// find them.
template <int D, int W>
struct Places {
  static constexpr int kPieces = D / 8, kPasses = kPieces / W;
  static constexpr int kInQuad = kPieces < 16 ? 16 / kPieces : 1;
  static constexpr int kOfTile = 2 * kPasses * kInQuad, kTiles = 16 / kOfTile;
  static_assert(kTiles * kOfTile == 16 && kTiles <= 2, "");
  int nth, value, pass, in_pass;
  __device__ Places(int lane) {
    const int e = lane & 15;
    nth = e / kOfTile;
    value = e / (kPasses * kInQuad) % 2;
    pass = e / kInQuad % kPasses;
    in_pass = kInQuad > 1 ? (lane >> 4) * kInQuad + e % kInQuad : (lane >> 4) * 16 / kPieces;
  }
  // of the tile
  __device__ int row(int wave) const { return (pass * W + wave) * (64 / kPieces) + in_pass; }
  template <int NTH, int PASS, int VALUE>
  static __device__ inline uint64_t row_of_quad(const Rows& r) {
    return told<NTH * kOfTile + (VALUE * kPasses + PASS) * kInQuad, kInQuad == 2>(r);
  }
};

template <class T, int D, int W>
__global__ __launch_bounds__(64 * W, D == 256 ? 1 : 2) void attend_many_kernel(const Args a) {
  using Op = typename Mat<T>::Op;
  constexpr int kPieces = D / 8;              // of a row
  constexpr int kPasses = kPieces / W;        // of the workgroup over a tile's pieces
  constexpr int kPassRows = 64 / kPieces;     // of a wavefront in a pass
  constexpr int kHalf = kTile * D * 2;        // bytes of a tile of K or V
  constexpr int KS = D / 16, NT = D / 32;
  // The two places are objects of their own: were they one, every read of the one would wait for the
  // loads into the other.
  __shared__ __attribute__((aligned(1024))) char place0[2][kHalf];
  __shared__ __attribute__((aligned(1024))) char place1[2][kHalf];
  __shared__ int odd[W];                      // whether a wavefront saw V that is not finite
  const Place at = heads_apart(a, blockIdx.x);
  const Work w = find_work<ManyPlan>(a, at.item, 32 * W, false);
  if (a.slots && blockIdx.x == 0 && threadIdx.x == 0) *a.any_cut = w.any_cut;
  if (w.seq < 0) return;
  const int first = w.tile * 32 * W;
  const int rows = min(32 * W, w.s.count * a.group - first);
  const int wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int column = lane & 31, half = lane >> 5;
  const int keys = max(w.s.keys, 0);
  const int mine = 32 * wave + column;        // this lane's row of the tile
  auto row_here = [&] { return row_of(a, w.s, first + min(mine, rows - 1), at.head); };
  const int visible = row_here().visible;
  // of the rows, in order, the first sees the fewest, the last the most
  const int fewest = row_of(a, w.s, first, at.head).visible;
  const int most = row_of(a, w.s, first + rows - 1, at.head).visible;
  const int all_tiles = (most + kTile - 1) / kTile;
  const int begin = w.cuts > 1 ? w.cut * w.steps : 0;
  const int end = w.cuts > 1 ? min(all_tiles, (w.cut + 1) * w.steps) : all_tiles;

  Op q[KS];
  {
    const Row row = row_here();
    const char* const p = a.q + row.at * a.q_row + row.head * a.q_head + half * 16;
#pragma unroll
    for (int x = 0; x < KS; ++x)
      q[x] = query_part<T>(p + 32 * x, a.scale_log2 < 0.f);
  }

  // Which rows of a tile a wavefront brings: the 16 lanes of a quad find the rows that the quad
  // loads, in `Places`, of as many tiles as there are lanes for.  Block ids are asked for that much ahead
  // of the rows, these as much ahead of their use; past the last key everything is of that one again.
  using P = Places<D, W>;
  int bad = kNoToken;
  const P mine_of(lane);
  Half of = mine_of.value ? a.v : a.k;
  of.p += at.head * of.head;
  const int found_row = mine_of.row(wave), nth = mine_of.nth;
  auto token_of = [&](int tile) { return min(tile * kTile + found_row, keys - 1); };
  auto find = [&](int t, const RawId& raw) {
    const int64_t id = block_id(a, raw);
    if (outside(a, id)) bad = min(bad, t);
    const uint64_t p = row_address(a, of, id, t, 0);
    return Rows{static_cast<uint32_t>(p), static_cast<uint32_t>(p >> 32)};
  };
  // where in its row lies the piece that a lane brings; pieces are exchanged alike in every 16 rows
  constexpr int kPeriod = W * kPassRows < 16 ? 16 / (W * kPassRows) : 1;
  uint32_t k_piece[kPeriod], v_piece[kPeriod];
#pragma unroll
  for (int i = 0; i < kPeriod; ++i) {
    const int row = (i * W + wave) * kPassRows + lane / kPieces, piece = lane % kPieces;
    k_piece[i] = (piece ^ k_swizzle<D>(row)) << 4, v_piece[i] = (piece ^ v_swizzle<D>(row)) << 4;
  }
  // the rows found for the n-th of kTiles tiles
  auto bring = [&](const Rows& r, auto n, char (*place)[kHalf])__attribute__((always_inline)) {
    each_index<kPasses>([&](auto i) __attribute__((always_inline)) {
      load_to_lds(P::template row_of_quad<n, i, 0>(r) + k_piece[i % kPeriod],
                  place[0] + (i * W + wave) * 1024);
      load_to_lds(P::template row_of_quad<n, i, 1>(r) + v_piece[i % kPeriod],
                  place[1] + (i * W + wave) * 1024);
    });
  };
  // a tile that some row of the workgroup does not see all of
  auto partly = [&](int tile) { return (tile + 1) * kTile > fewest; };
  // whether its V holds an infinity or a NaN; the same to all
  auto any_odd = [&](char (*place)[kHalf]) __attribute__((always_inline)) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const Vec4 x = *reinterpret_cast<const Vec4*>(place[1] + (i * W + wave) * 1024 + lane * 16);
#pragma unroll
      for (int y = 0; y < 4; ++y) any |= not_finite<T>(x[y]);
    }
    any = __any(any);
    if (lane == 0) odd[wave] = any;
    __syncthreads();
    int all = 0;
#pragma unroll
    for (int x = 0; x < W; ++x) all |= odd[x];
    return uniform(all) != 0;
  };

  const float scale_log2 = score_scale(a.scale_log2);
  float m, l, slack;
  v16f o[NT];
  auto clear = [&]() __attribute__((always_inline)) {
    m = kNothing, l = 0.f, slack = Mat<T>::kMost;
#pragma unroll
    for (int d = 0; d < NT; ++d)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
  };
  clear();

  RawId ids{0, 0};
  Rows ahead{0, 0};           // of the kTiles tiles that come next
  constexpr std::integral_constant<int, 0> k0{};
  constexpr std::integral_constant<int, P::kTiles - 1> k1{};
  if (begin < end) {
    ids = ask_block(a, w.seq, token_of(begin));
    const RawId next_ids = ask_block(a, w.seq, token_of(begin + 1 + nth));
    bring(find(token_of(begin), ids), k0, place0);
    ahead = find(token_of(begin + 1 + nth), next_ids);
    ids = ask_block(a, w.seq, token_of(begin + 1 + P::kTiles + nth));
  }
  // waited for here: in the loop the wait would be one for all loads, at every tile
#pragma unroll
  for (int x = 0; x < KS; ++x) asm volatile("" : "+v"(q[x]));
  // where a lane reads: K's row `column`, piece `half`; V's rows 4 half + ((lane & 15) >> 2)
  const int k_at = column * D * 2 + ((half ^ k_swizzle<D>(column)) << 4);
  int v_at[2];
#pragma unroll
  for (int j = 0; j < 2; ++j) {
    const int r = 8 * j + 4 * half + ((lane & 15) >> 2);
    const int piece = ((lane >> 4 & 1) << 1) | (lane >> 1 & 1);
    v_at[j] = r * D * 2 + ((piece ^ v_swizzle<D>(r)) << 4) + (lane & 1) * 8;
  }
  int tile = begin;
  // A tile's scores, in their place its weights, and what these change of the row's state.
  v16f s[2];
  auto scores = [&](const char* kt) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[h][i] = 0.f;
#pragma unroll
    for (int x = 0; x < KS; ++x)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Op k = __builtin_bit_cast(
            Op, *reinterpret_cast<const Vec4*>(kt + (k_at ^ (x % 8 * 32)) + x / 8 * 256 +
                                               32 * h * D * 2));
        s[h] = Mat<T>::mul32(k, q[x], s[h]);
      }
    reads_ahead<6, KS, 2, 2>();
    __builtin_amdgcn_sched_barrier(0);
    if (partly(tile)) {
      int seen = visible - tile * kTile - 4 * half;
      asm volatile("" : "+v"(seen));       // not 32 differences, one for each token, kept
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * h + 8 * (i / 4) + i % 4 >= seen) s[h][i] = -INFINITY;
    }
  };
  auto weigh_all = [&](bool coarse) __attribute__((always_inline)) {
    float sum[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[h][i] = __builtin_amdgcn_exp2f(coarse ? rounded_less(s[h][i], scale_log2, m)
                                                : __builtin_fmaf(s[h][i], scale_log2, -m));
        sum[h] = i ? sum[h] + s[h][i] : s[h][i];
      }
    return sum[0] + sum[1];
  };
  // Of 256 elements the sums and the query are 192 registers: kept where matrix instructions alone
  // reach them, which the compiler does not do by itself.  With them among the others it put a part
  // of the query into scratch memory and waited there for every read (256 queries of 32 heads over
  // up to 4906 keys of 4 sequences 141 us, 333 without; 2048 over 8192 of one 517 us).
  auto keep_aside = [&]() __attribute__((always_inline)) {
    if constexpr (D == 256) {
#pragma unroll
      for (int d = 0; d < NT; ++d) asm volatile("" : "+a"(o[d]));
#pragma unroll
      for (int x = 0; x < KS; ++x) asm volatile("" : "+a"(q[x]));
    }
  };
  auto weights = [&](const char* kt) __attribute__((always_inline)) {
    float sum = weigh_all(false);
    keep_aside();
    if (__any(sum > slack)) {
      // Some score passes its row's reference: the references follow, and the weights are made
      // again, from scores made again, which would be 32 registers more if they were kept.
      scores(kt);
      float top = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[h][i] * scale_log2);
      const auto other = __builtin_amdgcn_permlane32_swap(f32_bits(top), f32_bits(top), false, false);
      top = fmaxf(m, fmaxf(bits_f32(other[0]), bits_f32(other[1])) - Mat<T>::kBelow);
      const float fade = __builtin_amdgcn_exp2f(m - top);
      m = top;
      l *= fade;
#pragma unroll
      for (int d = 0; d < NT; ++d) o[d] *= fade;
      keep_aside();
      const bool coarse = fabsf(m) >= kCoarse && m != kNothing;
      sum = weigh_all(coarse);
      slack = __any(coarse) ? -1.f : Mat<T>::kMost;
      keep_aside();
    }
    l += sum;
  };
  auto add_values = [&](const char* vt) __attribute__((always_inline)) {
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      uint32_t u[4];
#pragma unroll
      for (int x = 0; x < 4; ++x)
        u[x] = Mat<T>::pack(s[b / 2][8 * (b % 2) + 2 * x], s[b / 2][8 * (b % 2) + 2 * x + 1]);
      const Op weight = __builtin_bit_cast(Op, make_uint4(u[0], u[1], u[2], u[3]));
#pragma unroll
      for (int d = 0; d < NT; ++d) {
        v4s x[2];
#pragma unroll
        for (int j = 0; j < 2; ++j)
          x[j] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsTransposed)(
              vt + (v_at[j] ^ (d % 4 * 64)) + d / 4 * 256 + 16 * b * D * 2));
        const Op v =
            __builtin_bit_cast(Op, __builtin_shufflevector(x[0], x[1], 0, 1, 2, 3, 4, 5, 6, 7));
        o[d] = Mat<T>::mul32(v, weight, o[d]);
      }
    }
    reads_ahead<8, 4 * NT, 1, 2>();
    __builtin_amdgcn_sched_barrier(0);
  };
  // The next tile's way to `there`: of two tiles whose rows were found together the first, or the second
  // (or only one), after which those of the next are found.
  auto bring_next = [&](auto second_of_two, char (*there)[kHalf]) __attribute__((always_inline)) {
    if constexpr (P::kTiles == 1 || second_of_two) {
      bring(ahead, k1, there);
      ahead = find(token_of(tile + 2 + nth), ids);
      ids = ask_block(a, w.seq, token_of(tile + 2 + P::kTiles + nth));
    } else {
      bring(ahead, k0, there);
    }
  };
  // One tile from `here`, the next one's way to `there`; false where its products may have to be made
  // one by one.
  auto take = [&](char (*here)[kHalf], char (*there)[kHalf],
                  auto second_of_two) __attribute__((always_inline)) {
    wait_for_loads();
    asm volatile("" : "+v"(ids.lo), "+v"(ids.hi));   // so that these are not waited for again
    __syncthreads();
    if (partly(tile) && any_odd(here)) return false;
    keep_aside();
    __builtin_amdgcn_sched_barrier(0);
    // the wavefront of the other workgroup on this SIMD has the vector instructions meanwhile (1 %)
    __builtin_amdgcn_s_setprio(1);
    scores(here[0]);
    __builtin_amdgcn_s_setprio(0);
    bring_next(second_of_two, there);
    weights(here[0]);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    add_values(here[1]);
    __builtin_amdgcn_s_setprio(0);
    keep_aside();
    return true;
  };
  bool one_by_one = false;
  keep_aside();
  while (tile < end) {
    keep_aside();
    if (!take(place0, place1, std::false_type())) {
      one_by_one = true;
      break;
    }
    if (++tile == end) break;
    if (!take(place1, place0, std::true_type())) {
      one_by_one = true;
      break;
    }
    ++tile;
  }
  if (one_by_one) {
    // V holds an infinity or a NaN that some row may not see, and a weight of 0 does not leave it out
    // of a matrix product: those tiles' products are made one by one.  All over again, and without
    // loads ahead, since a loop that goes on with the sums costs the other its registers.
    clear();
#pragma unroll 1
    for (tile = begin; tile < end; ++tile) {
      wait_for_loads();
      __syncthreads();                    // the tile before has been read by all
      ids = ask_block(a, w.seq, token_of(tile));
      bring(find(token_of(tile), ids), k0, place0);
      wait_for_loads();
      __syncthreads();
      const bool odd_values = partly(tile) && any_odd(place0);
      scores(place0[0]);
      weights(place0[0]);
      if (!odd_values) {
        add_values(place0[1]);
        continue;
      }
#pragma unroll 1
      for (int t = 0; t < kTile; ++t) {
        float x = s[0][0];
#pragma unroll
        for (int i = 1; i < 32; ++i)
          x = (t / 32 * 16 + t % 32 / 8 * 4 + t % 4) == i ? s[i / 16][i % 16] : x;
        x = __shfl(x, column + 32 * (t / 4 % 2));
        const bool seen = tile * kTile + t < visible;
#pragma unroll
        for (int d = 0; d < NT; ++d) {
          asm volatile("" ::: "memory");
#pragma unroll
          for (int i = 0; i < 16; i += 2) {
            const uint32_t u = *reinterpret_cast<const uint32_t*>(
                place0[1] + t * D * 2 + (((4 * d + i / 4) ^ v_swizzle<D>(t)) << 4) + half * 8 +
                i % 4 * 2);
            if (!seen) continue;
            o[d][i] += x * Mat<T>::low(u);
            o[d][i + 1] += x * Mat<T>::high(u);
          }
        }
      }
    }
  }
  // nothing may still be on its way to LDS when the workgroup ends and others get it
  wait_for_loads();
  // the least bad token that any wavefront came across
  bad = least(bad);
  __shared__ int bads[W];
  if (lane == 0) bads[wave] = bad;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < W; ++x) bad = min(bad, bads[x]);
  const auto both = __builtin_amdgcn_permlane32_swap(f32_bits(l), f32_bits(l), false, false);
  l = bits_f32(both[0]) + bits_f32(both[1]);
  if (w.s.keys < 0 || visible > bad) l = bits_f32(0x7fc00000u);
  if (mine >= rows) return;
  const Row row = row_here();
  const float inv = inverse(l, visible);
  const int64_t part = part_of(a, at.item, at.head) * (32 * W) + mine;
#pragma unroll
  for (int d = 0; d < NT; ++d)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      const int element = 32 * d + 8 * (i / 4) + 4 * half;
      const float x[4] = {o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
      if (w.cuts == 1)
        write_elements<T, 4>(a, row, element, x, inv);
      else
        *reinterpret_cast<v4f*>(a.part_o + part * D + element) = v4f{x[0], x[1], x[2], x[3]};
    }
  if (half) return;
  if (w.cuts == 1) write_stats(a, row, m, l);
  else a.part_ml[part] = make_float2(m, l);
}

// The parts of a tile as the join reads them: part(c) of `count`, of ROWS rows each.
// Of a line: a tile's first part is in the place for those that start there.
template <int ROWS>
struct PiecesOfTile {
  Piece w;
  int first, count;        // workgroups
  __device__ PiecesOfTile(const Args& a, int tile) {
    int total;
    const Line line(a, threadIdx.x & 63, ROWS);
    const int per = deal(a, ROWS, line, &total);
    w = find_piece(a, ROWS, line, tile, true);
    first = uniform(w.start / per);
    count = uniform((w.start + w.steps - 1) / per) - first + 1;
  }
  __device__ bool none() const { return w.seq < 0 || count == 1; }
  __device__ int64_t part(const Args& a, int c, int head) const {
    return part_of_piece(a, first + c, head, c == 0);
  }
};
// Of a plan that cuts every tile alike.
template <int ROWS>
struct CutsOfTile {
  Work w;
  int count;
  __device__ CutsOfTile(const Args& a, int tile) {
    w.seq = -1;
    if (!*a.any_cut) return;
    w = find_work<ManyPlan>(a, tile, ROWS, true);
    count = w.cuts;
  }
  __device__ bool none() const { return w.seq < 0 || count == 1; }
  __device__ int64_t part(const Args& a, int c, int head) const {
    return part_of(a, w.first + c, head);
  }
};

// Joins the parts of 16 rows of a tile of ROWS: 256 threads, each D / 16 neighbouring elements of a
// row, take every G-th part, and their sums are added in the order of g.  Bound by the latency of a
// launch and of the parts of the longest tile: 4 to 6 us, 10 where 256 to 512 tiles of 128 rows are cut.
template <class T, int D, int ROWS, class Parts, int G>
__global__ __launch_bounds__(256 * G) void join_kernel(const Args a) {
  constexpr int N = D / 16, kAhead = D == 256 ? 2 : 4;
  const int t = threadIdx.x & 255, g = threadIdx.x >> 8, n = t >> 4;
  const int block = blockIdx.x / (ROWS / 16), r = blockIdx.x % (ROWS / 16);
  const int tile = a.heads_div.div(block);
  const int head = block - tile * a.heads;
  const Parts parts(a, tile);
  if (parts.none()) return;
  const Seq s = parts.w.s;
  __shared__ float sum_o[G][N][256], sum_m[G][16], sum_l[G][16];
  const int first = parts.w.tile * ROWS + 16 * r;
  const bool valid = first + n < s.count * a.group;
  float o[N], m = kNothing, l = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) o[j] = 0.f;
  if (valid) {
    for (int c0 = g; c0 < parts.count; c0 += G * kAhead) {
      float2 x[kAhead];
      v4f y[kAhead][N / 4];
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int c = c0 + i * G;
        x[i] = make_float2(kNothing, 0.f);
#pragma unroll
        for (int j = 0; j < N / 4; ++j) y[i][j] = {0.f, 0.f, 0.f, 0.f};
        if (c < parts.count) {
          const int64_t part = parts.part(a, c, head) * ROWS + 16 * r + n;
          x[i] = a.part_ml[part];
#pragma unroll
          for (int j = 0; j < N / 4; ++j)
            y[i][j] = reinterpret_cast<const v4f*>(a.part_o + part * D + (t & 15) * N)[j];
        }
      }
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const float top = fmaxf(m, x[i].x);
        const float f = __builtin_amdgcn_exp2f(m - top), h = __builtin_amdgcn_exp2f(x[i].x - top);
        m = top;
        l = l * f + x[i].y * h;
#pragma unroll
        for (int j = 0; j < N; ++j) o[j] = o[j] * f + y[i][j / 4][j % 4] * h;
      }
    }
  }
  if ((t & 15) == 0) sum_m[g][n] = m, sum_l[g][n] = l;
#pragma unroll
  for (int j = 0; j < N; ++j) sum_o[g][j][t] = o[j];
  __syncthreads();
  if (g || !valid) return;
  float top = kNothing;
#pragma unroll
  for (int x = 0; x < G; ++x) top = fmaxf(top, sum_m[x][n]);
  l = 0.f;
#pragma unroll
  for (int j = 0; j < N; ++j) o[j] = 0.f;
#pragma unroll
  for (int x = 0; x < G; ++x) {
    const float f = __builtin_amdgcn_exp2f(sum_m[x][n] - top);
    l += sum_l[x][n] * f;
#pragma unroll
    for (int j = 0; j < N; ++j) o[j] += sum_o[x][j][t] * f;
  }
  const Row row = row_of(a, s, first + n, head);
  write_elements<T, N>(a, row, (t & 15) * N, o, inverse(l, row.visible));
  if ((t & 15) == 0) write_stats(a, row, top, l);
}

// ---------------------------------------------------------------------------
// What each token got, from scores that lie there: a thread adds up 4 tokens' over the rows, in
// their order.  They are scaled as where the row's sum was made of them: rounded before the reference
// is taken off they would be off by up to 0.5 where it is near 2^24.  Bound by memory: 4 bytes a row
// and token (and as many to write them), where making the scores again takes K's 2 D bytes a token.
// 32 sequences of up to 8192 keys, groups of 4: 9.6 us.

constexpr int kAddTokens = 1024;     // of a workgroup

__global__ __launch_bounds__(256) void add_weights_kernel(const Args a) {
  const int head = blockIdx.y, seq = blockIdx.z;
  const int at = blockIdx.x * kAddTokens + static_cast<int>(threadIdx.x) * 4;
  const Seq s = sequence(a, seq);
  const int keys = max(s.keys, 0), rows = s.count * a.group;
  if (at >= keys) return;
  const float scale_log2 = score_scale(a.scale_log2);
  float sums[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int n = 0; n < rows; ++n) {
    const Row row = row_of(a, s, n, head);
    const int64_t place = row.at * (a.heads * a.group) + row.head;
    const float2 st = a.stats[place];
    const v4f x = *reinterpret_cast<const v4f*>(a.scores + place * a.scores_row + at);
    // of steps that no row of a tile sees nothing has been written
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float e = __builtin_amdgcn_exp2f(fabsf(st.x) >= kCoarse
                                                 ? rounded_less(x[i], scale_log2, st.x)
                                                 : __builtin_fmaf(x[i], scale_log2, -st.x)) *
                      st.y;
      sums[i] += at + i < row.visible ? e : 0.f;
    }
  }
  float* const w = a.weights + seq * a.w_seq + head * a.w_head + at;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (at + i < keys) w[i] += sums[i];
}

// ---------------------------------------------------------------------------
// What each token got, from K: a wavefront keeps 64 tokens of K in registers and goes over the
// queries, 32 rows at a time, which the workgroup's wavefronts share in LDS.  Here the tokens are the
// columns of the products, so that a lane adds up its own token's weights, in the rows' order.  The
// scores are the attention's bit for bit, also those of attend_few_kernel: two instructions of k = 16
// add the products in the order of one of k = 32, and either operand may come first.  Where
// there are few tokens the rows are shared out to several workgroups, whose sums are then added up.
// Bound by the exponentials and products, of which each takes about as long (64 queries of 32 heads
// over up to 16384 keys, 4 sequences: 58 us).

constexpr int kWeighTokens = 256;    // of a workgroup

template <class T, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void weigh_kernel(const Args a) {
  using Op = typename Mat<T>::Op;
  constexpr int KS = D / 16, W = 4, kPieces = D / 8, kPasses = kPieces / 8;
  // two places for 32 rows, objects of their own as the tiles of attend_many_kernel
  __shared__ __attribute__((aligned(1024))) char place0[32 * D * 2];
  __shared__ __attribute__((aligned(1024))) char place1[32 * D * 2];
  __shared__ __attribute__((aligned(16))) float2 row_stats[W][32];   // of a wavefront's own reading
  __shared__ __attribute__((aligned(16))) int row_visible[W][32];
  const int head = blockIdx.y, seq = blockIdx.z;
  const int wave = uniform(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, column = lane & 31, half = lane >> 5;
  const int tile = a.shares_div.div(blockIdx.x), share = blockIdx.x - tile * a.shares;
  const int first = tile * kWeighTokens, at = first + wave * 64;
  const Seq s = sequence(a, seq);
  // too long for its table row: NaN in all rows, and in the tokens of no block
  const int keys = max(s.keys, 0), rows = s.count * a.group;
  if (first >= keys || rows <= 0) return;
  Op k[2][KS];
  float2 stats;
  int visible;
  auto bring = [&](int r0, char* place) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const int n = (i * W + wave) * (64 / kPieces) + lane / kPieces, piece = lane % kPieces;
      const Row row = row_of(a, s, min(r0 + n, rows - 1), head);
      load_to_lds(reinterpret_cast<uint64_t>(a.q) + row.at * a.q_row + row.head * a.q_head +
                      ((piece ^ k_swizzle<D>(n)) << 4),
                  place + (i * W + wave) * 1024);
    }
    const Row row = row_of(a, s, min(r0 + column, rows - 1), head);
    visible = r0 + column < rows ? row.visible : 0;
    stats = a.stats[row.at * (a.heads * a.group) + row.head];
  };
  // the first row that sees the first of the tokens
  const int hidden = a.causal ? max(0, first + s.count - keys) * a.group : 0;
  const int shown = hidden & ~31;
  const int per_share = a.shares_div.div((rows - shown + 31) / 32 + a.shares - 1) * 32;
  int r0 = shown + share * per_share;
  const int stop = min(rows, r0 + per_share);
  const RawId id[2] = {ask_block(a, seq, min(at + column, keys - 1)),
                       ask_block(a, seq, min(at + 32 + column, keys - 1))};
  bring(r0, place0);
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int t = min(at + 32 * h + column, keys - 1);
    const uint64_t p = row_address(a, a.k, block_id(a, id[h]), t, head) + half * 16;
    const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
#pragma unroll
    for (int x = 0; x < KS; ++x)
      k[h][x] = __builtin_bit_cast(Op, load<Vec4>(p + 32 * x) ^ flip);
  }
  const float scale_log2 = score_scale(a.scale_log2);
  const int q_at = column * D * 2 + ((half ^ k_swizzle<D>(column)) << 4);
  float sums[2] = {0.f, 0.f};
  auto take = [&](const char* here, char* there) __attribute__((always_inline)) {
    wait_for_loads();
    // a wavefront's own: its LDS accesses are in order
    if (half == 0) row_stats[wave][column] = stats, row_visible[wave][column] = visible;
    __syncthreads();
    // of the rows there are, in order, the first sees the fewest; past the last nothing is seen
    const bool all_see = r0 + 32 <= rows && lane_value(visible, 0) >= at + 64;
    const bool any_coarse = __any(fabsf(stats.x) >= kCoarse);
    __builtin_amdgcn_sched_barrier(0);
    v16f acc[2];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 16; ++i) acc[h][i] = 0.f;
#pragma unroll
    for (int x = 0; x < KS; ++x) {
      const Op q = __builtin_bit_cast(
          Op, *reinterpret_cast<const Vec4*>(here + (q_at ^ (x % 8 * 32)) + x / 8 * 256));
      acc[0] = Mat<T>::mul32(q, k[0][x], acc[0]);
      acc[1] = Mat<T>::mul32(q, k[1][x], acc[1]);
    }
    reads_ahead<3, KS, 2, 1>();
    __builtin_amdgcn_sched_barrier(0);
    bring(r0 + 32, there);
    auto weigh_all = [&](bool coarse, bool masked) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int n = 8 * (i / 4) + 4 * half + i % 4;
        const float2 st = row_stats[wave][n];
        const int seen = masked ? row_visible[wave][n] : 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float e = __builtin_amdgcn_exp2f(
              coarse && fabsf(st.x) >= kCoarse ? rounded_less(acc[h][i], scale_log2, st.x)
                                               : __builtin_fmaf(acc[h][i], scale_log2, -st.x));
          if (!masked || at + 32 * h + column < seen) sums[h] = __builtin_fmaf(e, st.y, sums[h]);
        }
      }
    };
    if (all_see && !any_coarse) weigh_all(false, false);
    else weigh_all(true, true);
    r0 += 32;
  };
  while (r0 < stop) {
    take(place0, place1);
    if (r0 >= stop) break;
    take(place1, place0);
  }
  // nothing may still be on its way to LDS when the workgroup ends and others get it
  wait_for_loads();
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto both =
        __builtin_amdgcn_permlane32_swap(f32_bits(sums[h]), f32_bits(sums[h]), false, false);
    sums[h] = bits_f32(both[0]) + bits_f32(both[1]);
  }
  // lanes below 32 have the first 32 tokens' sums to store, the others the second's
  const int t = at + lane;
  const float sum = half ? sums[1] : sums[0];
  if (a.shares > 1)
    a.share_sums[((static_cast<int64_t>(seq) * a.heads + head) * a.shares + share) * a.share_row + t] =
        sum;
  else if (t < keys)
    a.weights[seq * a.w_seq + head * a.w_head + t] += sum;
}

// The shares' sums added up, in their order: a token a thread.
__global__ __launch_bounds__(256) void add_shares_kernel(const Args a) {
  const int head = blockIdx.y, seq = blockIdx.z;
  const int t = blockIdx.x * 256 + static_cast<int>(threadIdx.x);
  const Seq s = sequence(a, seq);
  if (t >= s.keys || s.count <= 0) return;
  const float* const from =
      a.share_sums + (static_cast<int64_t>(seq) * a.heads + head) * a.shares * a.share_row + t;
  float sum = 0.f;
#pragma unroll 8
  for (int i = 0; i < a.shares; ++i) sum += from[i * a.share_row];
  a.weights[seq * a.w_seq + head * a.w_head + t] += sum;
}

// ---------------------------------------------------------------------------
// Host side

int check_sizes(const fkv_paged_attention_args& c) {
  int rc;
  const fkv_paged_layer& layer = c.layer;
  if (c.batch < 0 || c.num_queries < 0)
    return fail(kInval, "negative count: batch=%d num_queries=%d", c.batch, c.num_queries);
  if ((rc = paged_check_sizes(layer))) return rc;
  if (layer.head_size != 64 && layer.head_size != 128 && layer.head_size != 256)
    return fail(kInval, "attention takes a head_size of 64, 128 or 256, got %d", layer.head_size);
  if (layer.dtype != FKV_DTYPE_BF16 && layer.dtype != FKV_DTYPE_FP16)
    return fail(kInval, "attention takes a bf16 or fp16 cache, got dtype %d", layer.dtype);
  if (c.group_size < 1 || c.group_size > 1024)
    return fail(kInval, "group_size must be in [1, 1024], got %d", c.group_size);
  // an infinite one would make NaN of scores of 0
  if (!std::isfinite(c.scale * kLog2e))
    return fail(kInval, "scale must be finite, and in units of log 2 as well (up to 2^127)");
  const int64_t most = static_cast<int64_t>(c.table_width) * layer.tokens_per_block;
  if (c.table_width < 0 || most > int64_t(1) << 28)
    return fail(kInval, "table_width must be non-negative and hold at most 2^28 tokens, got %d "
                "blocks of %d", c.table_width, layer.tokens_per_block);
  if (static_cast<int64_t>(c.num_queries) * c.group_size >= int64_t(1) << 30)
    return fail(kInval, "%d queries of %d heads a K/V head are too many for one call",
                c.num_queries, c.group_size);
  if (!c.query_starts && c.num_queries < c.batch && c.num_queries > 0)
    return fail(kInval, "%d sequences of one query each, but %d queries", c.batch, c.num_queries);
  if (c.weights && c.weights_width < most)
    return fail(kInval, "weights' rows of %d do not hold the %lld tokens of a row of block_table",
                c.weights_width, (long long)most);
  if (c.weights && c.batch > 65535)
    return fail(kInval, "%d sequences with weights are too many for one call", c.batch);
  return 0;
}

int check_attention(const fkv_paged_attention_args& c) {
  if (!c.query || !c.out || !c.seq_lens || (!c.block_table && c.table_width > 0))
    return fail(kInval, "null pointer argument");
  if (!c.layer.value) return fail(kInval, "null cache pointer");
  const int64_t aligned[] = {c.query_row_stride_bytes, c.query_head_stride_bytes,
                             c.out_row_stride_bytes, c.out_head_stride_bytes,
                             static_cast<int64_t>(reinterpret_cast<uintptr_t>(c.query)),
                             static_cast<int64_t>(reinterpret_cast<uintptr_t>(c.out))};
  for (int64_t v : aligned)
    if (v % 16)
      return fail(kInval, "query's and out's pointers and strides must be multiples of 16 bytes");
  return paged_check_layer(c.layer);
}

struct LaunchPlan {
  int rows;               // of a tile
  bool many;              // rows are shared out to the wavefronts, else keys are
  int64_t tiles;          // times heads: the most there can be
  int waves;              // of a workgroup
  int slots;              // see Sequences and Piece
  bool together;
  int64_t workgroups;
  size_t ml_bytes, o_bytes, stats_bytes, scores_bytes, shares_bytes;
  int64_t scores_row;     // 0: the scores are not kept
  int shares;             // of the rows, where the scores are made again
  int64_t share_row;
  size_t bytes() const { return o_bytes + ml_bytes + stats_bytes + scores_bytes + shares_bytes; }
};

constexpr int kComputeUnits = 256;
// Scores are kept up to this size of the workspace: a table far wider than the sequences are long
// makes it large.
constexpr int64_t kMostScores = int64_t(1) << 30;
// Steps of a table row from which keys are dealt out, which costs 6 to 8 us: 32 sequences of 2048 keys 43
// us uncut and 51 dealt out; 32 of 2048 to 8192 keys 161 uncut and 133 dealt out.  Half of them where
// uncut tiles leave half of the compute units without work (one sequence of 3114 keys 34 uncut and 24
// dealt out, 32 of them 55 and 58), or have four wavefronts, as those of 256 elements (71 and 39, 108 and
// 100).
constexpr int kDealSteps = 128;

LaunchPlan launch_plan(const fkv_paged_attention_args& c) {
  LaunchPlan p;
  const int heads = c.layer.num_heads, dim = c.layer.head_size;
  const int64_t rows = static_cast<int64_t>(c.query_starts ? c.num_queries : c.batch) * c.group_size;
  // Few rows are up to 32 a sequence: a wavefront's registers hold the sums of two tiles of 16, of one
  // where an element has 256.  16 sequences of 40 rows of 64 elements: 22 us with the kernel for many,
  // 24 with three tiles.
  auto over = [&](int n) { return rows > static_cast<int64_t>(c.batch) * n; };
  p.many = over(2 * kRows);
  p.rows = p.many ? 128 : !over(kRows) || dim == 256 ? kRows : 2 * kRows;
  const int64_t tiles = c.query_starts
                            ? rows / p.rows + c.batch
                            : static_cast<int64_t>(c.batch) * ((c.group_size + p.rows - 1) / p.rows);
  p.tiles = tiles * heads;
  const int step = p.many ? ManyPlan::kStep : FewPlan::kStep;
  const int64_t most_steps =
      (static_cast<int64_t>(c.table_width) * c.layer.tokens_per_block + step - 1) / step;
  int64_t parts;
  p.waves = 4;
  if (p.many) {
    p.slots = most_steps < ManyPlan::kMinSteps + ManyPlan::kCutSteps || p.tiles > 4 * kComputeUnits
                  ? 0 : 2 * kComputeUnits;
    // items (cuts of a tile, of all heads), in whole rounds of the XCDs
    const int64_t items = (p.tiles + p.slots + heads - 1) / heads;
    p.workgroups = (items + kXcds - 1) / kXcds * kXcds * heads;
    p.together = false;
    parts = p.slots ? p.workgroups : 0;
  } else {
    // A workgroup of 8 wavefronts a compute unit, each with an even share of the steps; a tile for each
    // workgroup where there are so many sequences that working the shares out takes long, or few keys.
    const int deal_steps =
        dim == 256 || p.tiles <= kComputeUnits / 2 ? kDealSteps / 2 : kDealSteps;
    // the kernel adds the number of slots, a compute unit's each at most, to all steps in 32 bits
    const bool dealt = c.batch <= 4 * 64 && most_steps >= deal_steps &&
                       tiles * most_steps <= INT32_MAX - kComputeUnits;
    p.waves = (dealt || p.tiles <= kComputeUnits) && dim <= 128 ? 8 : 4;
    const int64_t places = kComputeUnits * 8 / p.waves / (dim == 256 ? 2 : 1);
    int64_t items = dealt ? std::max<int64_t>(1, places / heads) : tiles;
    p.together = p.rows == kRows && items >= kXcds;
    if (p.together)                          // whole rounds of the XCDs
      items = dealt ? items / kXcds * kXcds : (items + kXcds - 1) / kXcds * kXcds;
    p.slots = dealt ? static_cast<int>(items) : 0;
    p.workgroups = items * heads;
    parts = p.slots ? 2 * p.workgroups : 0;
  }
  p.ml_bytes = parts * p.rows * sizeof(float2) + (parts ? 16 : 0);    // and any_cut
  p.o_bytes = parts * p.rows * dim * sizeof(float);
  const int64_t all_rows = static_cast<int64_t>(c.num_queries) * heads * c.group_size;
  p.stats_bytes = c.weights ? (all_rows * sizeof(float2) + 15) / 16 * 16 : 0;
  // Kept of up to 16 rows a sequence: 32 sequences of 4 rows take 173 us with them, 322 where they are
  // made again; 16 of 40 rows 55 us with them, 43 where they are made again.
  p.scores_row = c.weights && !over(kRows) ? most_steps * step : 0;
  if (static_cast<__int128>(all_rows) * p.scores_row * 4 > kMostScores) p.scores_row = 0;
  p.scores_bytes = all_rows * p.scores_row * sizeof(float);
  // As many as give each compute unit six workgroups (three are there at a time), of at least 64 rows,
  // a step for each of the two places: 8 sequences of up to 390 queries of 10 heads of 64 elements over
  // up to 620 keys take 33 us with the attention, 103 without shares, and 38 with shares of 128 rows; 2000
  // queries of 32 heads over themselves 114 us, 324 without, and 122 with three workgroups.
  const int64_t weigh_tiles =
      (static_cast<int64_t>(c.table_width) * c.layer.tokens_per_block + kWeighTokens - 1) /
      kWeighTokens;
  const int64_t weigh_items = std::max<int64_t>(1, weigh_tiles * heads * c.batch);
  p.share_row = weigh_tiles * kWeighTokens;
  p.shares = p.scores_row ? 1 : static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>({32, 6 * kComputeUnits / weigh_items, rows / c.batch / 64})));
  p.shares_bytes = c.weights && p.shares > 1
                       ? static_cast<int64_t>(c.batch) * heads * p.shares * p.share_row * sizeof(float)
                       : 0;
  return p;
}

// A launch has less than 2^32 threads.
int check_plan(const fkv_paged_attention_args& c, const LaunchPlan& p) {
  const int64_t weigh = p.share_row / kWeighTokens * c.layer.num_heads * c.batch;
  if (p.workgroups >= int64_t(1) << 22 || (c.weights && weigh >= int64_t(1) << 23))
    return fail(kInval, "%d queries of %d K/V heads are too many for one call", c.num_queries,
                c.layer.num_heads);
  return 0;
}

template <class T, int D, int ROWS, class Parts, int G>
void join(const Args& a, const LaunchPlan& p, hipStream_t s) {
  if (p.slots)
    hipLaunchKernelGGL((join_kernel<T, D, ROWS, Parts, G>), dim3(p.tiles * (ROWS / 16)),
                       dim3(256 * G), 0, s, a);
}
template <class T, int D, int R, int W>
void launch_few(const Args& a, const LaunchPlan& p, hipStream_t s) {
  hipLaunchKernelGGL((attend_few_kernel<T, D, R, W>), dim3(p.workgroups), dim3(64 * W), 0, s, a);
  join<T, D, kRows * R, PiecesOfTile<kRows * R>, 4>(a, p, s);
}
template <class T, int D, int R>
void launch_few(const Args& a, const LaunchPlan& p, hipStream_t s) {
  if (p.waves == 8) launch_few<T, D, R, D == 256 ? 4 : 8>(a, p, s);
  else launch_few<T, D, R, 4>(a, p, s);
}
template <class T, int D, int W>
void launch_many(const Args& a, const LaunchPlan& p, hipStream_t s) {
  hipLaunchKernelGGL((attend_many_kernel<T, D, W>), dim3(p.workgroups), dim3(64 * W), 0, s, a);
  join<T, D, 32 * W, CutsOfTile<32 * W>, 1>(a, p, s);
}
template <class T, int D>
void launch(const Args& a, const LaunchPlan& p, const fkv_paged_attention_args& c, hipStream_t s) {
  if (p.many) launch_many<T, D, 4>(a, p, s);
  else if (p.rows == kRows) launch_few<T, D, 1>(a, p, s);
  else launch_few<T, D, D == 256 ? 1 : 2>(a, p, s);
  const int64_t most = static_cast<int64_t>(a.width) * a.tokens;
  if (a.scores) {
    hipLaunchKernelGGL(add_weights_kernel,
                       dim3((most + kAddTokens - 1) / kAddTokens, a.heads, a.batch), dim3(256), 0,
                       s, a);
  } else if (a.weights && a.width) {
    const int64_t tiles = (most + kWeighTokens - 1) / kWeighTokens;
    hipLaunchKernelGGL((weigh_kernel<T, D>), dim3(tiles * a.shares, a.heads, a.batch), dim3(256), 0,
                       s, a);
    if (a.shares > 1)
      hipLaunchKernelGGL(add_shares_kernel, dim3((most + 255) / 256, a.heads, a.batch), dim3(256), 0,
                         s, a);
  }
}
template <class T>
void launch_attention(const Args& a, const LaunchPlan& p, const fkv_paged_attention_args& c,
                      hipStream_t s) {
  if (c.layer.head_size == 64) launch<T, 64>(a, p, c, s);
  else if (c.layer.head_size == 128) launch<T, 128>(a, p, c, s);
  else launch<T, 256>(a, p, c, s);
}

int attention(const fkv_paged_attention_args& c, fkv_stream_t stream) {
  int rc = check_sizes(c);
  if (rc || c.batch == 0 || c.num_queries == 0) return rc;
  if ((rc = check_attention(c))) return rc;
  const LaunchPlan p = launch_plan(c);
  if ((rc = check_plan(c, p))) return rc;
  const size_t need = p.bytes();
  if (need && (!c.workspace || c.workspace_bytes < need ||
               reinterpret_cast<uintptr_t>(c.workspace) % 16))
    return fail(kInval, "the workspace must hold %zu bytes on a multiple of 16, got %zu", need,
                c.workspace ? c.workspace_bytes : 0);
  Args a{};
  a.q = static_cast<const char*>(c.query);
  a.out = static_cast<char*>(c.out);
  a.lse = c.lse;
  a.q_row = c.query_row_stride_bytes, a.q_head = c.query_head_stride_bytes;
  a.out_row = c.out_row_stride_bytes, a.out_head = c.out_head_stride_bytes;
  a.lse_row = c.lse_row_stride, a.lse_head = c.lse_head_stride;
  a.k = key_half(c.layer), a.v = value_half(c.layer);
  a.table = c.block_table, a.lens = c.seq_lens, a.starts = c.query_starts;
  a.table_row = c.table_row_stride;
  a.index64 = c.index_is_64bit;
  a.num_blocks = static_cast<int>(c.layer.num_blocks), a.width = c.table_width;
  a.batch = c.batch, a.heads = c.layer.num_heads, a.group = c.group_size;
  a.queries = c.num_queries;
  a.tokens = c.layer.tokens_per_block, a.causal = c.causal;
  a.slots = p.slots;
  a.together = p.together;
  a.scale_log2 = c.scale * kLog2e;
  char* const space = static_cast<char*>(c.workspace);
  a.part_o = reinterpret_cast<float*>(space);
  a.any_cut = reinterpret_cast<int*>(space + p.o_bytes);
  a.part_ml = reinterpret_cast<float2*>(space + p.o_bytes + 16);
  a.weights = c.weights, a.w_seq = c.weights_seq_stride, a.w_head = c.weights_head_stride;
  a.stats = c.weights ? reinterpret_cast<float2*>(space + p.o_bytes + p.ml_bytes) : nullptr;
  a.scores_row = p.scores_row;
  if (p.scores_row)
    a.scores = reinterpret_cast<float*>(space + p.o_bytes + p.ml_bytes + p.stats_bytes);
  a.shares = p.shares, a.shares_div = FastDiv(p.shares), a.share_row = p.share_row;
  a.share_sums = reinterpret_cast<float*>(space + p.o_bytes + p.ml_bytes + p.stats_bytes);
  a.tokens_div = FastDiv(a.tokens), a.group_div = FastDiv(a.group), a.heads_div = FastDiv(a.heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int dev = 0;
  DeviceGuard guard;
  if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
  (void)hipGetLastError();
  if (c.layer.dtype == FKV_DTYPE_BF16) launch_attention<__bf16>(a, p, c, s);
  else launch_attention<_Float16>(a, p, c, s);
  FKV_HIP(hipGetLastError());
  return 0;
}

// No C++ exception leaves a C entry.
template <class F>
int guarded(F call) {
  try {
    last_error().clear();
    return call();
  } catch (const std::exception& e) {
    return fail(static_cast<int>(hipErrorUnknown), "exception: %s", e.what());
  } catch (...) {
    return fail(static_cast<int>(hipErrorUnknown), "unknown exception");
  }
}

}  // namespace

extern "C" {

int fkv_paged_attention_workspace(const fkv_paged_attention_args* args, size_t* bytes) {
  return guarded([&] {
    if (!args || !bytes) return fail(kInval, "null pointer argument");
    *bytes = 0;
    int rc = check_sizes(*args);
    if (rc || args->batch == 0 || args->num_queries == 0) return rc;
    const LaunchPlan p = launch_plan(*args);
    if ((rc = check_plan(*args, p))) return rc;
    *bytes = p.bytes();
    return 0;
  });
}

int fkv_paged_attention(const fkv_paged_attention_args* args, fkv_stream_t stream) {
  return guarded([&] {
    if (!args) return fail(kInval, "null pointer argument");
    return attention(*args, stream);
  });
}

}  // extern "C"

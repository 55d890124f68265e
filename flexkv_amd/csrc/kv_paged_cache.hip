// kv_paged_cache.hip - a paged KV cache in its own type: new tokens into their slots, and
// eviction of what got little attention.
//
// Eviction: of a sequence's n tokens each K/V head keeps the `recent` last and, of the others,
// those with the largest weights (equal ones: the earlier), `budget` in all.  The choice is made by
// a workgroup for each (sequence, head), or by several where there are few and they are long; then
// the kept rows are copied to the blocks of a new table, whole rows by 16-byte accesses.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <exception>

#include "kv_attention.h"
#include "kv_paged.h"

using namespace fkv_detail;

namespace {

typedef uint32_t Vec4 __attribute__((ext_vector_type(4)));

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// New tokens

struct WriteArgs {
  const char* rows[2];
  int64_t row_stride[2], head_stride[2];
  Half to[2];
  const void* slots;
  int slots64;
  int64_t num_slots;
  int tokens;
  uint32_t units;                    // 16-byte pieces of one half
  FastDiv vecs, per_token;           // pieces of a row, of a token
};

// A thread takes one 16-byte piece of K and the same of V, so that a wavefront reads and writes whole
// rows.  Bound by memory: 8191 tokens of 8 heads of 128 elements, 67 MB in 12 us.
__global__ __launch_bounds__(kThreads) void write_tokens_kernel(const WriteArgs a) {
  const uint32_t unit = blockIdx.x * kThreads + threadIdx.x;
  if (unit >= a.units) return;
  const uint32_t n = a.per_token.div(unit), in_token = unit - n * a.per_token.d;
  const uint32_t head = a.vecs.div(in_token), vec = in_token - head * a.vecs.d;
  const int64_t slot = index_at(a.slots, n, a.slots64);
  Vec4 x[2];
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (a.rows[k])
      x[k] = *reinterpret_cast<const Vec4*>(a.rows[k] + n * a.row_stride[k] +
                                            head * a.head_stride[k] + vec * 16);
  if (slot < 0 || slot >= a.num_slots) return;
  const int64_t block = slot / a.tokens, t = slot - block * a.tokens;
#pragma unroll
  for (int k = 0; k < 2; ++k)
    if (a.rows[k])
      *reinterpret_cast<Vec4*>(a.to[k].p + block * a.to[k].block + t * a.to[k].token +
                               head * a.to[k].head + vec * 16) = x[k];
}

// ---------------------------------------------------------------------------
// Eviction

struct EvictArgs {
  Half half[2];
  int halves;
  const float* weights;
  float* new_weights;                // null: not asked for
  int64_t w_seq, w_head, nw_seq, nw_head;     // elements
  int nw_width;
  const void* table;
  const void* new_table;
  const void* lens;
  int64_t table_row, new_table_row;  // elements
  int index64;
  int64_t num_blocks;
  int width, tokens, heads;
  int budget, recent;
  int* kept;                         // [sequence][head][budget]
  int chunk_rows, chunks;            // of a copying workgroup; of a (sequence, head)
  int parts;                         // workgroups that choose for a (sequence, head)
  // of more than one: how often they count each digit, [sequence][head][pass][part][digit], what
  // is found of the threshold, [sequence][head][pass][part], and the kept tokens' weights,
  // [sequence][head][stash_row], null where new_weights is
  int* counted;
  int4* states;
  float* stash;
  int stash_row;
  FastDiv tokens_div, heads_div, chunks_div, parts_div, vecs;
};

// Keys of sequence b; -1: more than its table row can hold, and the sequence is left alone.
__device__ inline int keys_of(const EvictArgs& a, int b) {
  const int64_t n = index_at(a.lens, b, a.index64);
  return n < 0 ? 0 : n > static_cast<int64_t>(a.width) * a.tokens ? -1 : static_cast<int>(n);
}

// Orders floats as unsigned numbers: -0 as 0, NaN above all.
__device__ inline uint32_t order_of(float f) {
  if (f != f) return 0xffffffffu;
  const uint32_t u = f32_bits(f + 0.f);
  return u >> 31 ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr int kRadixBits = 11;       // of a pass: three of them
// Inclusive sums over the workgroup's threads.  `totals` holds kSelectWaves values and may not be
// in use.
__device__ inline int scan_threads(int v, int* totals) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  v = scan_lanes(v);
  if (lane == 63) totals[wave] = v;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int i = 0; i < kSelectWaves; ++i) before += i < wave ? totals[i] : 0;
  return v + before;
}
// A thread's values of kAtOnce * kSelectThreads tokens from t0 on: loads in flight together.
constexpr int kAtOnce = 8;
struct Batch {
  static constexpr int kTokens = kAtOnce * kSelectThreads;
  float x[kAtOnce];
  __device__ void load(const float* w, int t0, int n) {
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      x[j] = w[min(t0 + j * kSelectThreads + static_cast<int>(threadIdx.x), n - 1)];
  }
  // f(order, whether there is such a token)
  template <class F>
  __device__ void each(int t0, int n, F f) const {
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j)
      if (t0 + j * kSelectThreads < n)
        f(order_of(x[j]), t0 + j * kSelectThreads + static_cast<int>(threadIdx.x) < n);
  }
};
// All of n tokens, the next two batches on their way while one is looked at, the first two from
// the start on.
struct Orders {
  const float* const w;
  const int n;
  Batch x[3];
  __device__ Orders(const float* w, int n) : w(w), n(n) {
    if (n <= 0) return;
    x[0].load(w, 0, n);
    x[1].load(w, Batch::kTokens, n);
  }
  template <class F>
  __device__ void each(F f) {
    for (int t0 = 0; t0 < n; t0 += 3 * Batch::kTokens) {
#pragma unroll
      for (int i = 0; i < 3; ++i) {
        const int t = t0 + i * Batch::kTokens;
        if (t >= n) break;
        x[(i + 2) % 3].load(w, t + 2 * Batch::kTokens, n);
        x[i].each(t, n, f);
      }
    }
  }
};
template <class F>
__device__ inline void each_order(const float* w, int n, F f) {
  Orders(w, n).each(f);
}

// The digit (of the 2 to the kRadixBits that `histogram` counts) where the need-th largest is, and
// how many of those with that digit are still needed; `found` is for two threads to tell all.
struct Digit {
  int value, need, count;
};
__device__ inline Digit digit_of(const int* histogram, int need, int* totals, int* found) {
  // a thread has two digits, the first thread the largest
  const int top = (1 << kRadixBits) - 1 - 2 * static_cast<int>(threadIdx.x);
  const int c0 = histogram[top], c1 = histogram[top - 1];
  const int upto = scan_threads(c0 + c1, totals), before = upto - c0 - c1;
  if (before < need && need <= upto) {
    const bool first = need <= before + c0;
    found[0] = first ? top : top - 1;
    found[1] = need - before - (first ? 0 : c0);
    found[2] = first ? c0 : c1;
  }
  __syncthreads();
  return {found[0], found[1], found[2]};
}

// One more of `digit`, for the lanes that are `in`.
__device__ inline void count(int* histogram, uint32_t digit, bool in) {
  // weights that are alike (none has got any yet) would queue for one counter
  const uint64_t all = __ballot(in);
  if (!all) return;
  const int at = __builtin_ctzll(all);
  const uint32_t lead = lane_value(digit, at);
  if (__ballot(in && digit == lead) == all) {
    if (static_cast<int>(threadIdx.x & 63) == at) atomicAdd(&histogram[lead], __popcll(all));
  } else if (in) {
    atomicAdd(&histogram[digit], 1);
  }
}

// The need-th largest weight's order among w[0 .. n), 0 < need < n: the digits of the order from
// the highest on (11, 11 and 10 bits), each from a histogram of the values that share the digits
// before.  Those that share the first are mostly few, and then the rest is found among them alone.
// `ties`: how many of that order are among the need largest.
constexpr int kMostCandidates = 8192;
struct Chooser {
  int histogram[1 << kRadixBits];
  int totals[kSelectWaves], found[3], fill;
  uint32_t candidates[kMostCandidates];
};
__device__ inline uint32_t threshold_of(const float* w, int n, int need, Chooser& c, int* ties) {
  auto clear = [&] {
    for (int i = threadIdx.x; i < 1 << kRadixBits; i += kSelectThreads) c.histogram[i] = 0;
    if (threadIdx.x == 0) c.fill = 0;
    __syncthreads();
  };
  clear();
  each_order(w, n, [&](uint32_t k, bool in) { count(c.histogram, k >> 21, in); });
  __syncthreads();
  const Digit high = digit_of(c.histogram, need, c.totals, c.found);
  const uint32_t first = high.value;
  clear();
  const bool listed = high.count <= kMostCandidates;
  if (listed) {
    each_order(w, n, [&](uint32_t k, bool in) {
      if (in && k >> 21 == first) c.candidates[atomicAdd(&c.fill, 1)] = k;
    });
    __syncthreads();
    for (int i = threadIdx.x; i < high.count; i += kSelectThreads)
      atomicAdd(&c.histogram[c.candidates[i] >> 10 & 2047], 1);
  } else {
    each_order(w, n, [&](uint32_t k, bool in) {
      count(c.histogram, k >> 10 & 2047, in && k >> 21 == first);
    });
  }
  __syncthreads();
  const Digit middle = digit_of(c.histogram, high.need, c.totals, c.found);
  const uint32_t second = first << 11 | static_cast<uint32_t>(middle.value);
  clear();
  if (listed) {
    for (int i = threadIdx.x; i < high.count; i += kSelectThreads)
      if (c.candidates[i] >> 10 == second) atomicAdd(&c.histogram[c.candidates[i] & 1023], 1);
  } else {
    each_order(w, n, [&](uint32_t k, bool in) {
      count(c.histogram, k & 1023, in && k >> 10 == second);
    });
  }
  __syncthreads();
  const Digit low = digit_of(c.histogram, middle.need, c.totals, c.found);
  *ties = low.need;
  return second << 10 | static_cast<uint32_t>(low.value);
}

// What a sequence of n tokens keeps.
struct Choice {
  int count, others, need;           // in all; that are not recent, and how many of these
  __device__ Choice(const EvictArgs& a, int n) {
    count = min(max(n, 0), a.budget);
    const int recent = min(a.recent, count);
    others = max(n, 0) - recent, need = count - recent;
  }
  __device__ bool weighed() const { return need && need < others; }
};

// The tokens [from, to) that are kept, in their order: those past `others`, those above the
// threshold, and of its equals the first `ties`.  `above` and `equal` of the tokens before are
// kept for the former and are the latter.  put(rank, token, weight) may store over weights that lie
// no further on than the token's.
template <class Put>
__device__ inline void keep(const float* w, int from, int to, int others, uint32_t threshold,
                            int ties, int above, int equal, Put put) {
  __shared__ int counts[kAtOnce * kSelectWaves];
  static_assert(kAtOnce * kSelectWaves == 2 * 64, "two a lane below");
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  Batch x, next;
  if (from < to) next.load(w, from, to);
  for (int t0 = from; t0 < to; t0 += Batch::kTokens) {
    x = next;
    next.load(w, t0 + Batch::kTokens, to);
    uint64_t over[kAtOnce], same[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      over[j] = same[j] = 0;
      if (t0 + j * kSelectThreads < to) {
        const int t = t0 + j * kSelectThreads + static_cast<int>(threadIdx.x);
        const uint32_t k = order_of(x.x[j]);
        over[j] = __ballot(t < to && (t >= others || k > threshold));
        same[j] = __ballot(t < to && t < others && k == threshold);
      }
      if (lane == 0)
        counts[j * kSelectWaves + wave] = __popcll(over[j]) | __popcll(same[j]) << 16;
    }
    __syncthreads();                 // all have this batch, which the stores below may be to
    // sums over (round, wave) in the tokens' order: two of the 128 a lane, in every wave
    const int c0 = counts[2 * lane], c1 = counts[2 * lane + 1];
    const int pair = scan_lanes(c0 + c1);
    const int all = lane_value(pair, 63);
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      if (!(over[j] | same[j])) continue;
      const int at = j * kSelectWaves + wave;
      int before = lane_value(pair - c0 - c1, uniform(at >> 1));
      if (at & 1) before += lane_value(c0, uniform(at >> 1));
      const uint64_t mine = uint64_t(1) << lane, below = mine - 1;
      const int n_over = above + (before & 0xffff) + __popcll(over[j] & below);
      const int n_same = equal + (before >> 16) + __popcll(same[j] & below);
      if ((over[j] & mine) || ((same[j] & mine) && n_same < ties))
        put(n_over + min(n_same, ties), t0 + j * kSelectThreads + static_cast<int>(threadIdx.x),
            x.x[j]);
    }
    above += all & 0xffff;
    equal += all >> 16;
    __syncthreads();
  }
}

// One workgroup for a (sequence, head).  Bound by its compute unit's instructions and two dozen
// barriers: 8192 tokens 13 us, 777 9 (without the copy).
__global__ __launch_bounds__(kSelectThreads) void evict_choose_kernel(const EvictArgs a) {
  __shared__ Chooser chooser;
  const int b = a.heads_div.div(blockIdx.x), h = blockIdx.x - b * a.heads;
  const int n = keys_of(a, b);
  int* const kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  const float* const w = a.weights + b * a.w_seq + h * a.w_head;
  float* const nw = a.new_weights ? a.new_weights + b * a.nw_seq + h * a.nw_head : nullptr;
  const Choice c(a, n);
  uint32_t threshold = c.need ? 0 : 0xffffffffu;
  int ties = c.need;                 // all, where all stay
  if (c.weighed()) threshold = threshold_of(w, c.others, c.need, chooser, &ties);
  keep(w, 0, n, c.others, threshold, ties, 0, 0, [&](int rank, int t, float weight) {
    kept[rank] = t;
    if (nw) nw[rank] = weight;
  });
  // up to 2^31 of a row: both in 64 bits
  for (int64_t i = c.count + static_cast<int64_t>(threadIdx.x); i < a.budget; i += kSelectThreads)
    kept[i] = -1;
  if (nw && n >= 0)
    for (int64_t i = c.count + static_cast<int64_t>(threadIdx.x); i < a.nw_width;
         i += kSelectThreads)
      nw[i] = 0.f;
}

// The choice of long sequences, where there are few: a.parts workgroups for a (sequence, head), each
// with a share of the tokens.  A launch for each digit, in which a workgroup first finds the digits
// before from what all counted of them, then counts its own tokens', and one that keeps.  The
// order that the counts are added up in does not change them.  Bound by the launches, 5 to 9 us each:
// two sequences of 65536 tokens 26 us, 58 with a workgroup each (without the copy).
constexpr int kDigits = 1 << kRadixBits, kPasses = 3;
struct Part {
  int b, h, part, n, from, to;
  int* counted;                      // of this (sequence, head), [pass][part][digit]
  int4* states;                      // [pass][part]
  const float* w;
};
__device__ inline Part part_of(const EvictArgs& a) {
  Part p;
  const int row = a.parts_div.div(blockIdx.x);
  p.part = blockIdx.x - row * a.parts;
  p.b = a.heads_div.div(row), p.h = row - p.b * a.heads;
  p.n = keys_of(a, p.b);
  const int n = max(p.n, 0), each = a.parts_div.div(n + a.parts - 1);
  const int per = (each + kSelectThreads - 1) / kSelectThreads * kSelectThreads;
  p.from = min(per * p.part, n), p.to = min(p.from + per, n);
  p.counted = a.counted + static_cast<int64_t>(row) * kPasses * a.parts * kDigits;
  p.states = a.states + static_cast<int64_t>(row) * kPasses * a.parts;
  p.w = a.weights + p.b * a.w_seq + p.h * a.w_head;
  return p;
}

// The threshold's digits so far, how many of those that have them are needed, and how many of the
// parts before this are above them, or have them.
struct Found {
  int digits, need, above, equal;
};
struct Finder {
  int totals[2][kSelectWaves], found[4];
  // What `pass` adds to what was found before it, from what all parts counted in it.
  __device__ Found find(const EvictArgs& a, const Part& p, int pass, int need) {
    Found was{0, need, 0, 0};
    if (pass) was = __builtin_bit_cast(Found, p.states[(pass - 1) * a.parts + p.part]);
    const int thread = threadIdx.x, top = kDigits - 1 - 2 * thread;
    // a thread has two digits, the first thread the largest
    const int2* const counts =
        reinterpret_cast<const int2*>(p.counted + static_cast<int64_t>(pass) * a.parts * kDigits) +
        (kDigits / 2 - 1 - thread);
    int c0 = 0, c1 = 0, b0 = 0, b1 = 0;
#pragma unroll 8
    for (int i = 0; i < a.parts; ++i) {
      const int2 c = counts[i * (kDigits / 2)];
      c0 += c.y, c1 += c.x;
      if (i < p.part) b0 += c.y, b1 += c.x;
    }
    const int upto = scan_threads(c0 + c1, totals[0]), before = upto - c0 - c1;
    const int part_before = scan_threads(b0 + b1, totals[1]) - b0 - b1;
    if (before < was.need && was.need <= upto) {
      const bool first = was.need <= before + c0;
      found[0] = first ? top : top - 1;
      found[1] = was.need - before - (first ? 0 : c0);
      found[2] = part_before + (first ? 0 : b0);
      found[3] = first ? b0 : b1;
    }
    __syncthreads();
    const int bits = pass == kPasses - 1 ? 32 - 2 * kRadixBits : kRadixBits;
    return {was.digits << bits | found[0], found[1], was.above + found[2], found[3]};
  }
};

template <int PASS>
__global__ __launch_bounds__(kSelectThreads) void evict_count_kernel(const EvictArgs a) {
  __shared__ Finder finder;
  __shared__ __attribute__((aligned(8))) int histogram[kDigits];
  const Part p = part_of(a);
  const Choice c(a, p.n);
  if (!c.weighed()) return;
  const int tokens = max(min(p.to, c.others) - p.from, 0);
  Orders orders(p.w + p.from, tokens);
  uint32_t digits = 0;
  if (PASS) {
    const Found now = finder.find(a, p, PASS - 1, c.need);
    digits = now.digits;
    if (threadIdx.x == 0)
      p.states[(PASS - 1) * a.parts + p.part] = __builtin_bit_cast(int4, now);
  }
  int2* const mine = reinterpret_cast<int2*>(histogram) + threadIdx.x;
  *mine = make_int2(0, 0);
  __syncthreads();
  orders.each([&](uint32_t k, bool in) {
    if (PASS == 0) count(histogram, k >> 21, in);
    else if (PASS == 1) count(histogram, k >> 10 & 2047, in && k >> 21 == digits);
    else count(histogram, k & 1023, in && k >> 10 == digits);
  });
  __syncthreads();
  int* const to = p.counted + (static_cast<int64_t>(PASS) * a.parts + p.part) * kDigits;
  reinterpret_cast<int2*>(to)[threadIdx.x] = *mine;
}

__global__ __launch_bounds__(kSelectThreads) void evict_keep_kernel(const EvictArgs a) {
  __shared__ Finder finder;
  const Part p = part_of(a);
  const Choice c(a, p.n);
  uint32_t threshold = c.need ? 0 : 0xffffffffu;
  int ties = c.need, above = max(0, p.from - c.others), equal = 0;
  if (c.weighed()) {
    const Found all = finder.find(a, p, kPasses - 1, c.need);
    threshold = all.digits, ties = all.need, above += all.above, equal = all.equal;
  } else if (c.need) {
    above = p.from;                  // all before stay
  }
  const int64_t row = static_cast<int64_t>(p.b) * a.heads + p.h;
  int* const kept = a.kept + row * a.budget;
  float* const stash = a.stash ? a.stash + row * a.stash_row : nullptr;
  keep(p.w, p.from, p.to, c.others, threshold, ties, above, equal,
       [&](int rank, int t, float weight) {
         kept[rank] = t;
         if (stash) stash[rank] = weight;
       });
  for (int64_t i = c.count + p.part * int64_t(kSelectThreads) + threadIdx.x; i < a.budget;
       i += a.parts * kSelectThreads)
    kept[i] = -1;
}

// A workgroup copies chunk_rows kept rows of one (sequence, head), K and V.  Where each lies and
// goes is worked out once, a row a thread, and shared.  Bound by memory: 32 sequences and 8 heads that
// keep up to 2048 rows of 256 bytes, 530 MB in 113 us, past the caches and with K beside V (4.7 TB/s
// in scattered rows; a plain copy reaches 6.3).
constexpr int kMostRows = 64;
__global__ __launch_bounds__(kThreads) void evict_copy_kernel(const EvictArgs a) {
  __shared__ const char* from[2][kMostRows];
  __shared__ char* to[2][kMostRows];
  const int rest = a.heads_div.div(blockIdx.x), h = blockIdx.x - rest * a.heads;
  const int b = a.chunks_div.div(rest), chunk = rest - b * a.chunks;
  const int first = chunk * a.chunk_rows;
  const int keys = keys_of(a, b), count = min(max(keys, 0), a.budget);
  const int rows = min(a.chunk_rows, count - first);
  if (a.stash && keys >= 0) {
    // the weights, which may go to where the others of the choice were still reading
    const int64_t row = static_cast<int64_t>(b) * a.heads + h;
    float* const nw = a.new_weights + b * a.nw_seq + h * a.nw_head;
    if (static_cast<int>(threadIdx.x) < rows)
      nw[first + threadIdx.x] = a.stash[row * a.stash_row + first + threadIdx.x];
    const int64_t step = static_cast<int64_t>(a.chunks) * kThreads;
    for (int64_t i = count + chunk * int64_t(kThreads) + threadIdx.x; i < a.nw_width; i += step)
      nw[i] = 0.f;
  }
  if (rows <= 0) return;
  if (static_cast<int>(threadIdx.x) < rows) {
    const int i = first + static_cast<int>(threadIdx.x);
    const int t = a.kept[(static_cast<int64_t>(b) * a.heads + h) * a.budget + i];
    const int page = a.tokens_div.div(t), new_page = a.tokens_div.div(i);
    const int64_t old_block = index_at(a.table, b * a.table_row + page, a.index64);
    const int64_t new_block = index_at(a.new_table, b * a.new_table_row + new_page, a.index64);
    const bool there = old_block >= 0 && old_block < a.num_blocks && new_block >= 0 &&
                       new_block < a.num_blocks;
    for (int k = 0; k < a.halves; ++k) {
      const Half& x = a.half[k];
      from[k][threadIdx.x] = there ? x.p + old_block * x.block + (t - page * a.tokens) * x.token +
                                         h * x.head
                                   : nullptr;
      to[k][threadIdx.x] = there ? x.p + new_block * x.block +
                                       (i - new_page * a.tokens) * x.token + h * x.head
                                 : nullptr;
    }
  }
  __syncthreads();
  const int units = rows * static_cast<int>(a.vecs.d);
  constexpr int kAhead = 4;
  for (int u0 = threadIdx.x; u0 < units; u0 += kAhead * kThreads) {
    Vec4 x[2][kAhead];
    int row[kAhead], piece[kAhead];
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int u = u0 + j * kThreads;
      row[j] = a.vecs.div(u);
      piece[j] = (u - row[j] * static_cast<int>(a.vecs.d)) * 16;
      if (u >= units || !from[0][row[j]]) row[j] = -1;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        if (row[j] >= 0 && k < a.halves)
          x[k][j] = __builtin_nontemporal_load(
              reinterpret_cast<const Vec4*>(from[k][row[j]] + piece[j]));
    }
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
        if (row[j] >= 0 && k < a.halves)
          __builtin_nontemporal_store(x[k][j], reinterpret_cast<Vec4*>(to[k][row[j]] + piece[j]));
  }
}

int check_evict(const fkv_evict_args& c) {
  int rc;
  if (c.batch < 0) return fail(kInval, "negative count: batch=%d", c.batch);
  if ((rc = paged_check_sizes(c.layer))) return rc;
  if (c.budget < 1 || c.budget > 1 << 28)
    return fail(kInval, "budget must be in [1, 2^28], got %d", c.budget);
  if (c.recent < 0 || c.recent > c.budget)
    return fail(kInval, "recent must be in [0, budget], got %d of %d", c.recent, c.budget);
  const int64_t most = static_cast<int64_t>(c.table_width) * c.layer.tokens_per_block;
  if (c.table_width < 0 || most > int64_t(1) << 28)
    return fail(kInval, "table_width must be non-negative and hold at most 2^28 tokens, got %d "
                "blocks of %d", c.table_width, c.layer.tokens_per_block);
  if (c.new_table_width < 0 || static_cast<int64_t>(c.new_table_width) *
                                       c.layer.tokens_per_block < std::min<int64_t>(c.budget, most))
    return fail(kInval, "new_table's rows of %d blocks of %d tokens do not hold %lld",
                c.new_table_width, c.layer.tokens_per_block,
                (long long)std::min<int64_t>(c.budget, most));
  if (c.weights_width < most)
    return fail(kInval, "weights' rows of %d do not hold the %lld tokens of a row of block_table",
                c.weights_width, (long long)most);
  if (c.new_weights && c.new_weights_width < std::min<int64_t>(c.budget, most))
    return fail(kInval, "new_weights' rows of %d do not hold %lld", c.new_weights_width,
                (long long)std::min<int64_t>(c.budget, most));
  // less than 2^32 threads in a launch
  if (static_cast<int64_t>(c.batch) * c.layer.num_heads > int64_t(1) << 21)
    return fail(kInval, "%d sequences of %d heads are too many for one call", c.batch,
                c.layer.num_heads);
  return 0;
}

// Rows of a copying workgroup: as many as it has places for, fewer where that would leave the
// device with less than two workgroups a compute unit (500 rows of 8 heads 4 us).
int copy_rows(int64_t rows) {
  int n = kMostRows;
  while (n > 16 && rows / n < 512) n /= 2;
  return n;
}

// Workgroups that choose for one (sequence, head): one for each 2^13 tokens, of all no more than two a
// compute unit; and one alone where it would not be four, since several take three launches more
// (a call with its copy, two sequences: 8192 tokens 17 us with one, 26 with two; 65536 62 with one, 30
// with eight).
int choice_parts(int64_t heads, int64_t tokens) {
  const int64_t parts = std::min<int64_t>({32, 512 / heads, tokens / Batch::kTokens});
  return parts < 4 ? 1 : static_cast<int>(parts);
}
struct EvictPlan {
  int64_t heads, most, tokens;       // (sequence, head)s; that one keeps; that one has
  int parts;
  size_t counted_bytes, state_bytes, stash_bytes;
  explicit EvictPlan(const fkv_evict_args& c) {
    heads = static_cast<int64_t>(c.batch) * c.layer.num_heads;
    tokens = static_cast<int64_t>(c.table_width) * c.layer.tokens_per_block;
    most = std::min<int64_t>(c.budget, tokens);
    parts = choice_parts(heads, tokens);
    counted_bytes = parts > 1 ? heads * kPasses * parts * kDigits * sizeof(int) : 0;
    state_bytes = parts > 1 ? heads * kPasses * parts * sizeof(int4) : 0;
    stash_bytes = parts > 1 && c.new_weights ? heads * most * sizeof(float) : 0;
  }
  size_t bytes() const { return counted_bytes + state_bytes + stash_bytes; }
};

int evict(const fkv_evict_args& c, fkv_stream_t stream) {
  int rc;
  if ((rc = check_evict(c)) || c.batch == 0) return rc;
  // a table of no blocks has neither entries nor weights
  if (!c.kept || !c.seq_lens ||
      ((!c.weights || !c.block_table || !c.new_table) && c.table_width > 0))
    return fail(kInval, "null pointer argument");
  if ((rc = paged_check_layer(c.layer)) || (rc = paged_check_written(c.layer))) return rc;
  const EvictPlan p(c);
  const int64_t heads = p.heads, most = p.most;
  const size_t need = p.bytes();
  if (need && (!c.workspace || c.workspace_bytes < need ||
               reinterpret_cast<uintptr_t>(c.workspace) % 16))
    return fail(kInval, "the workspace must hold %zu bytes on a multiple of 16, got %zu", need,
                c.workspace ? c.workspace_bytes : 0);
  EvictArgs a{};
  a.half[0] = key_half(c.layer), a.half[1] = value_half(c.layer);
  a.halves = c.layer.value ? 2 : 1;
  a.weights = c.weights, a.new_weights = c.new_weights;
  a.w_seq = c.weights_seq_stride, a.w_head = c.weights_head_stride;
  a.nw_seq = c.new_weights_seq_stride, a.nw_head = c.new_weights_head_stride;
  a.nw_width = c.new_weights_width;
  a.table = c.block_table, a.new_table = c.new_table, a.lens = c.seq_lens;
  a.table_row = c.table_row_stride, a.new_table_row = c.new_table_row_stride;
  a.index64 = c.index_is_64bit;
  a.num_blocks = c.layer.num_blocks;
  a.width = c.table_width, a.tokens = c.layer.tokens_per_block, a.heads = c.layer.num_heads;
  a.budget = c.budget, a.recent = c.recent;
  a.kept = c.kept;
  a.chunk_rows = copy_rows(heads * most);
  a.chunks = static_cast<int>(std::max<int64_t>(1, (most + a.chunk_rows - 1) / a.chunk_rows));
  const int64_t workgroups = heads * a.chunks;
  if (workgroups >= int64_t(1) << 24)
    return fail(kInval, "%d sequences of %d heads that keep %lld tokens are too many for one call",
                c.batch, c.layer.num_heads, (long long)most);
  a.parts = p.parts;
  char* const space = static_cast<char*>(c.workspace);
  a.counted = reinterpret_cast<int*>(space);
  a.states = reinterpret_cast<int4*>(space + p.counted_bytes);
  if (p.stash_bytes)
    a.stash = reinterpret_cast<float*>(space + p.counted_bytes + p.state_bytes);
  a.stash_row = static_cast<int>(most);
  a.tokens_div = FastDiv(a.tokens), a.heads_div = FastDiv(a.heads), a.parts_div = FastDiv(a.parts);
  a.chunks_div = FastDiv(a.chunks);
  a.vecs = FastDiv(c.layer.head_size * paged_element_bytes(c.layer.dtype) / 16);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int dev = 0;
  DeviceGuard guard;
  if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
  (void)hipGetLastError();
  const dim3 grid(heads * p.parts), block(kSelectThreads);
  if (p.parts == 1) {
    hipLaunchKernelGGL(evict_choose_kernel, grid, block, 0, s, a);
  } else {
    hipLaunchKernelGGL(evict_count_kernel<0>, grid, block, 0, s, a);
    hipLaunchKernelGGL(evict_count_kernel<1>, grid, block, 0, s, a);
    hipLaunchKernelGGL(evict_count_kernel<2>, grid, block, 0, s, a);
    hipLaunchKernelGGL(evict_keep_kernel, grid, block, 0, s, a);
  }
  FKV_HIP(hipGetLastError());
  hipLaunchKernelGGL(evict_copy_kernel, dim3(workgroups), dim3(kThreads), 0, s, a);
  FKV_HIP(hipGetLastError());
  return 0;
}

int write_tokens(const fkv_paged_layer& layer, int num_tokens, const void* key, int64_t kts,
                 int64_t khs, const void* value, int64_t vts, int64_t vhs, const void* slots,
                 int slots64, fkv_stream_t stream) {
  int rc;
  if (num_tokens < 0) return fail(kInval, "negative count: num_tokens=%d", num_tokens);
  if ((rc = paged_check_sizes(layer))) return rc;
  const int64_t vecs = layer.head_size * paged_element_bytes(layer.dtype) / 16;
  const int64_t units = vecs * layer.num_heads * num_tokens;
  if (units > (int64_t(1) << 31) - kThreads)
    return fail(kInval, "%d tokens of %d heads of %d are too many for one call", num_tokens,
                layer.num_heads, layer.head_size);
  if ((rc = paged_check_layer(layer)) || num_tokens == 0) return rc;
  if (!key || !slots) return fail(kInval, "null pointer argument");
  if (!value != !layer.value)
    return fail(kInval, "value and the value cache must both be given, or neither");
  WriteArgs a{};
  a.rows[0] = static_cast<const char*>(key), a.rows[1] = static_cast<const char*>(value);
  a.row_stride[0] = kts, a.head_stride[0] = khs, a.row_stride[1] = vts, a.head_stride[1] = vhs;
  for (int k = 0; k < 2; ++k)
    if (a.rows[k] && (reinterpret_cast<uintptr_t>(a.rows[k]) % 16 || a.row_stride[k] % 16 ||
                      a.head_stride[k] % 16))
      return fail(kInval, "%s's pointer and strides must be multiples of 16 bytes (token %lld, "
                  "head %lld)", k ? "value" : "key", (long long)a.row_stride[k],
                  (long long)a.head_stride[k]);
  if ((rc = paged_check_written(layer))) return rc;
  a.to[0] = key_half(layer), a.to[1] = value_half(layer);
  a.slots = slots, a.slots64 = slots64;
  a.num_slots = layer.num_blocks * layer.tokens_per_block;
  a.tokens = layer.tokens_per_block;
  a.units = static_cast<uint32_t>(units);
  a.vecs = FastDiv(vecs), a.per_token = FastDiv(vecs * layer.num_heads);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int dev = 0;
  DeviceGuard guard;
  if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
  (void)hipGetLastError();
  hipLaunchKernelGGL(write_tokens_kernel, dim3((units + kThreads - 1) / kThreads), dim3(kThreads),
                     0, s, a);
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

int fkv_write_kv_tokens(const fkv_paged_layer* layer, int num_tokens, const void* key,
                        int64_t key_token_stride_bytes, int64_t key_head_stride_bytes,
                        const void* value, int64_t value_token_stride_bytes,
                        int64_t value_head_stride_bytes, const void* slots, int slots_are_64bit,
                        fkv_stream_t stream) {
  return guarded([&] {
    if (!layer) return fail(kInval, "null pointer argument");
    return write_tokens(*layer, num_tokens, key, key_token_stride_bytes, key_head_stride_bytes,
                        value, value_token_stride_bytes, value_head_stride_bytes, slots,
                        slots_are_64bit, stream);
  });
}

int fkv_evict_kv_tokens_workspace(const fkv_evict_args* args, size_t* bytes) {
  return guarded([&] {
    if (!args || !bytes) return fail(kInval, "null pointer argument");
    *bytes = 0;
    const int rc = check_evict(*args);
    if (!rc && args->batch) *bytes = EvictPlan(*args).bytes();
    return rc;
  });
}

int fkv_evict_kv_tokens(const fkv_evict_args* args, fkv_stream_t stream) {
  return guarded([&] {
    if (!args) return fail(kInval, "null pointer argument");
    return evict(*args, stream);
  });
}

}  // extern "C"

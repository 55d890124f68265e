// kv_paged_cache.hip - a paged KV cache in its own type: new tokens into their slots, and
// eviction of what got little attention.
//
// Eviction: of a sequence's n tokens each K/V head keeps the `recent` last and, of the others,
// those with the largest weights (equal ones: the earlier), `budget` in all.  Two launches:
// the choice, a workgroup for each (sequence, head), and the copy of the kept rows to the blocks of
// a new table, whole rows by 16-byte accesses.
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

// A thread takes one 16-byte piece of K and the same of V.
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
  FastDiv tokens_div, heads_div, chunks_div, vecs;
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
// All tokens, the next two batches on their way while one is looked at.
template <class F>
__device__ inline void each_order(const float* w, int n, F f) {
  Batch x[3];
  x[0].load(w, 0, n);
  x[1].load(w, Batch::kTokens, n);
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
  auto count = [&](uint32_t digit, bool in) {
    // weights that are alike (none has got any yet) would queue for one counter
    const uint64_t all = __ballot(in);
    if (!all) return;
    const int at = __builtin_ctzll(all);
    const uint32_t lead = lane_value(digit, at);
    if (__ballot(in && digit == lead) == all) {
      if ((threadIdx.x & 63) == at) atomicAdd(&c.histogram[lead], __popcll(all));
    } else if (in) {
      atomicAdd(&c.histogram[digit], 1);
    }
  };
  clear();
  each_order(w, n, [&](uint32_t k, bool in) { count(k >> 21, in); });
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
    each_order(w, n, [&](uint32_t k, bool in) { count(k >> 10 & 2047, in && k >> 21 == first); });
  }
  __syncthreads();
  const Digit middle = digit_of(c.histogram, high.need, c.totals, c.found);
  const uint32_t second = first << 11 | static_cast<uint32_t>(middle.value);
  clear();
  if (listed) {
    for (int i = threadIdx.x; i < high.count; i += kSelectThreads)
      if (c.candidates[i] >> 10 == second) atomicAdd(&c.histogram[c.candidates[i] & 1023], 1);
  } else {
    each_order(w, n, [&](uint32_t k, bool in) { count(k & 1023, in && k >> 10 == second); });
  }
  __syncthreads();
  const Digit low = digit_of(c.histogram, middle.need, c.totals, c.found);
  *ties = low.need;
  return second << 10 | static_cast<uint32_t>(low.value);
}

// Bound by one compute unit's instructions and two dozen barriers: 65536 tokens TODO us, 777 TODO.
__global__ __launch_bounds__(kSelectThreads) void evict_choose_kernel(const EvictArgs a) {
  __shared__ Chooser chooser;
  __shared__ int counts[kAtOnce * kSelectWaves];
  static_assert(kAtOnce * kSelectWaves == 2 * 64, "two a lane below");
  const int b = a.heads_div.div(blockIdx.x), h = blockIdx.x - b * a.heads;
  const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
  const int n = keys_of(a, b);
  int* const kept = a.kept + static_cast<int64_t>(blockIdx.x) * a.budget;
  const float* const w = a.weights + b * a.w_seq + h * a.w_head;
  float* const nw = a.new_weights ? a.new_weights + b * a.nw_seq + h * a.nw_head : nullptr;
  const int count = min(max(n, 0), a.budget), recent = min(a.recent, count);
  const int others = max(n, 0) - recent, need = count - recent;
  uint32_t threshold = need ? 0 : 0xffffffffu;
  int ties = need;                   // all, where all stay
  if (need && need < others) threshold = threshold_of(w, others, need, chooser, &ties);
  int above = 0, equal = 0;          // kept for their weight, and of the threshold's, so far
  Batch x, next;
  if (n > 0) next.load(w, 0, n);
  for (int t0 = 0; t0 < n; t0 += Batch::kTokens) {
    x = next;
    next.load(w, t0 + Batch::kTokens, n);
    uint64_t over[kAtOnce], same[kAtOnce];
#pragma unroll
    for (int j = 0; j < kAtOnce; ++j) {
      over[j] = same[j] = 0;
      if (t0 + j * kSelectThreads < n) {
        const int t = t0 + j * kSelectThreads + static_cast<int>(threadIdx.x);
        const uint32_t k = order_of(x.x[j]);
        over[j] = __ballot(t < n && (t >= others || k > threshold));
        same[j] = __ballot(t < others && k == threshold);
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
      if ((over[j] & mine) || ((same[j] & mine) && n_same < ties)) {
        const int rank = n_over + min(n_same, ties);
        kept[rank] = t0 + j * kSelectThreads + static_cast<int>(threadIdx.x);
        if (nw) nw[rank] = x.x[j];
      }
    }
    above += all & 0xffff;
    equal += all >> 16;
    __syncthreads();
  }
  for (int i = count + static_cast<int>(threadIdx.x); i < a.budget; i += kSelectThreads)
    kept[i] = -1;
  if (nw && n >= 0)
    for (int i = count + static_cast<int>(threadIdx.x); i < a.nw_width; i += kSelectThreads)
      nw[i] = 0.f;
}

// A workgroup copies chunk_rows kept rows of one (sequence, head), K and V.  Where each lies and
// goes is worked out once, a row a thread, and shared.
constexpr int kMostRows = 64;
__global__ __launch_bounds__(kThreads) void evict_copy_kernel(const EvictArgs a) {
  __shared__ const char* from[2][kMostRows];
  __shared__ char* to[2][kMostRows];
  const int rest = a.heads_div.div(blockIdx.x), h = blockIdx.x - rest * a.heads;
  const int b = a.chunks_div.div(rest), first = (rest - b * a.chunks) * a.chunk_rows;
  const int count = min(max(keys_of(a, b), 0), a.budget);
  const int rows = min(a.chunk_rows, count - first);
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
// device with less than two workgroups a compute unit.
int copy_rows(int64_t rows) {
  int n = kMostRows;
  while (n > 16 && rows / n < 512) n /= 2;
  return n;
}

int evict(const fkv_evict_args& c, fkv_stream_t stream) {
  int rc;
  if ((rc = check_evict(c)) || c.batch == 0) return rc;
  if (!c.kept || !c.weights || !c.seq_lens || ((!c.block_table || !c.new_table) && c.table_width > 0))
    return fail(kInval, "null pointer argument");
  if ((rc = paged_check_layer(c.layer))) return rc;
  const int64_t heads = static_cast<int64_t>(c.batch) * c.layer.num_heads;
  const int64_t most = std::min<int64_t>(
      c.budget, static_cast<int64_t>(c.table_width) * c.layer.tokens_per_block);
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
  a.tokens_div = FastDiv(a.tokens), a.heads_div = FastDiv(a.heads);
  a.chunks_div = FastDiv(a.chunks);
  a.vecs = FastDiv(c.layer.head_size * paged_element_bytes(c.layer.dtype) / 16);
  hipStream_t s = static_cast<hipStream_t>(stream);
  int dev = 0;
  DeviceGuard guard;
  if ((rc = stream_device(s, &dev)) || (rc = guard.set(dev))) return rc;
  (void)hipGetLastError();
  hipLaunchKernelGGL(evict_choose_kernel, dim3(heads), dim3(kSelectThreads), 0, s, a);
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
  a.to[0] = key_half(layer), a.to[1] = value_half(layer);
  a.slots = slots, a.slots64 = slots64;
  a.num_slots = layer.num_blocks * layer.tokens_per_block;
  a.tokens = layer.tokens_per_block;
  const int64_t vecs = layer.head_size * paged_element_bytes(layer.dtype) / 16;
  const int64_t units = vecs * layer.num_heads * num_tokens;
  if (units > (int64_t(1) << 31) - kThreads)
    return fail(kInval, "%d tokens of %d heads of %d are too many for one call", num_tokens,
                layer.num_heads, layer.head_size);
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

int fkv_evict_kv_tokens(const fkv_evict_args* args, fkv_stream_t stream) {
  return guarded([&] {
    if (!args) return fail(kInval, "null pointer argument");
    return evict(*args, stream);
  });
}

}  // extern "C"

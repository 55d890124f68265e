// kv_overlap.h - whether the rows of a cache that is written to share memory (no HIP, so that it
// can be checked without a device).  Not installed; not part of the C ABI.
#pragma once

#include <cstdint>

namespace fkv_detail {

// Rows of `bytes` bytes from p on, `count` of them `step` bytes apart in each of up to three
// dimensions, the closest first.
struct RowSet {
  uint64_t p;
  int64_t bytes;
  int dims = 0;
  int64_t step[3], count[3];
  RowSet(const void* at, int64_t row_bytes, const int64_t (&steps)[3], const int64_t (&counts)[3])
      : p(reinterpret_cast<uint64_t>(at)), bytes(row_bytes) {
    for (int d = 0; d < 3; ++d) {
      if (counts[d] <= 1) continue;
      int i = dims++;
      for (; i > 0 && step[i - 1] > steps[d]; --i) step[i] = step[i - 1], count[i] = count[i - 1];
      step[i] = steps[d], count[i] = counts[d];
    }
  }
  // From the first byte to the last, of the closest `n` dimensions.
  int64_t extent(int n) const {
    int64_t e = bytes;
    for (int i = 0; i < n; ++i) e += step[i] * (count[i] - 1);
    return e;
  }
};

// Whether no two rows share a byte; rows that lie between others' are taken to.
inline bool rows_apart(const RowSet& a) {
  for (int i = 0; i < a.dims; ++i)
    if (a.step[i] < a.extent(i)) return false;
  return true;
}

// Whether a row of a's closest n dimensions and one of b's, which starts `shift` bytes behind a,
// share a byte.  Both are apart in themselves, and have the same counts, though perhaps in another
// order.  Where the farthest dimension has one step for both, what lies in it is compared
// at the few distances at which it can meet; else what meets as a whole is taken to share one.
inline bool rows_meet(const RowSet& a, const RowSet& b, int n, int64_t shift) {
  const int64_t ea = a.extent(n), eb = b.extent(n);
  if (shift >= ea || shift <= -eb) return false;
  if (n == 0 || a.step[n - 1] != b.step[n - 1]) return true;
  const int64_t step = a.step[n - 1];
  // the rows of a at i * step and those of b at shift + j * step: of j - i the distances
  // around -shift / step, where what is in them, at most a step wide, can meet
  const int64_t middle = -shift / step;
  for (int64_t q = middle - 2; q <= middle + 2; ++q)
    if (q > -a.count[n - 1] && q < b.count[n - 1] && rows_meet(a, b, n - 1, shift + q * step))
      return true;
  return false;
}
inline bool rows_meet(const RowSet& a, const RowSet& b) {
  return rows_meet(a, b, a.dims, static_cast<int64_t>(b.p - a.p));
}

}  // namespace fkv_detail

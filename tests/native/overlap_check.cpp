// CPU-only check of how overlapping caches are told from others
// (flexkv_amd/csrc/kv_overlap.h): against a map of every byte, no HIP, no
// device.  Prints one line per case and exits non-zero when one fails.
#include "kv_overlap.h"

#include <cstdint>
#include <cstdio>
#include <random>
#include <set>
#include <vector>

using namespace fkv_detail;

namespace {

int failures = 0;

void check(bool ok, const char* what) {
  std::printf("%s: %s\n", ok ? "ok" : "FAIL", what);
  if (!ok) ++failures;
}

struct Half {
  int64_t at, step[3], count[3], bytes;
  RowSet rows() const { return RowSet(reinterpret_cast<const void*>(at), bytes, step, count); }
};

// Every row's first byte in units of 16, once a row.
std::vector<int64_t> units(const Half& h) {
  std::vector<int64_t> all;
  for (int64_t i = 0; i < h.count[0]; ++i)
    for (int64_t j = 0; j < h.count[1]; ++j)
      for (int64_t k = 0; k < h.count[2]; ++k)
        for (int64_t u = 0; u < h.bytes; u += 16)
          all.push_back(h.at + i * h.step[0] + j * h.step[1] + k * h.step[2] + u);
  return all;
}
bool apart(const Half& h) {
  std::set<int64_t> seen;
  for (int64_t u : units(h))
    if (!seen.insert(u).second) return false;
  return true;
}
bool meet(const Half& a, const Half& b) {
  const auto all = units(a);
  const std::set<int64_t> seen(all.begin(), all.end());
  for (int64_t u : units(b))
    if (seen.count(u)) return true;
  return false;
}

// Views of dense memory with dimensions in any order, padding and parts left out.
struct Dense {
  std::mt19937 g{7};
  int pick(int lo, int hi) { return std::uniform_int_distribution<int>(lo, hi)(g); }
};

void views_of_dense_memory() {
  bool self = true, pairs = true;
  int halves[2] = {0, 0};
  Dense r;
  for (int n = 0; n < 20000; ++n) {
    // blocks, tokens, heads and the halves, in an order of their own, the row innermost
    int64_t count[4] = {r.pick(1, 4), r.pick(1, 4), r.pick(1, 3), 2}, step[4];
    int order[4] = {0, 1, 2, 3};
    for (int i = 3; i > 0; --i) std::swap(order[i], order[r.pick(0, i)]);
    const int64_t bytes = 16 * r.pick(1, 3);
    int64_t size = bytes + 16 * r.pick(0, 1);
    for (int i : order) step[i] = size, size = size * count[i] + 16 * r.pick(0, 2);
    Half k{1 << 20, {step[0], step[1], step[2]}, {count[0], count[1], count[2]}, bytes}, v = k;
    v.at += step[3];
    self = self && rows_apart(k.rows()) && apart(k);
    pairs = pairs && !rows_meet(k.rows(), v.rows()) && !rows_meet(v.rows(), k.rows()) &&
            !meet(k, v);
    // moved against one another
    v.at = k.at + 16 * r.pick(-40, 40);
    const bool real = meet(k, v);
    pairs = pairs && rows_meet(k.rows(), v.rows()) == real && rows_meet(v.rows(), k.rows()) == real;
    ++halves[real];
  }
  check(self, "views of dense memory are apart in themselves");
  check(pairs, "two of the same steps are told apart exactly");
  check(halves[0] > 1000 && halves[1] > 1000, "of which many meet and many do not");
}

void steps_of_any_kind() {
  bool self = true, pairs = true;
  int refused = 0, kept = 0;
  Dense r;
  for (int n = 0; n < 40000; ++n) {
    Half h[2];
    const int64_t count[3] = {r.pick(1, 4), r.pick(1, 4), r.pick(1, 4)}, bytes = 16 * r.pick(1, 3);
    for (Half& x : h) {
      x = {(1 << 20) + 16 * r.pick(0, 60), {}, {count[0], count[1], count[2]}, bytes};
      for (int64_t& s : x.step) s = 16 * r.pick(0, r.pick(1, 40));
    }
    for (const Half& x : h) {
      // what is taken to be apart is so
      const bool told = rows_apart(x.rows());
      self = self && (!told || apart(x));
      told ? ++kept : ++refused;
    }
    if (!rows_apart(h[0].rows()) || !rows_apart(h[1].rows())) continue;
    pairs = pairs && (rows_meet(h[0].rows(), h[1].rows()) || !meet(h[0], h[1]));
  }
  check(self, "of other steps none that overlap are taken to be apart");
  check(pairs, "and no two that meet");
  check(kept > 1000 && refused > 1000, "of which many are apart and many are not");
}

void layouts_of_engines() {
  const int64_t N = 5, T = 16, H = 4, D = 256;
  const int64_t thd = T * H * D;
  auto half = [&](int64_t at, int64_t b, int64_t t, int64_t h) {
    return Half{at, {b, t, h}, {N, T, H}, D};
  };
  auto ok = [&](const Half& k, const Half& v) {
    return rows_apart(k.rows()) && rows_apart(v.rows()) && !rows_meet(k.rows(), v.rows());
  };
  check(ok(half(0, thd, H * D, D), half(N * thd, thd, H * D, D)), "halves of a layer");
  check(ok(half(0, 2 * thd, H * D, D), half(thd, 2 * thd, H * D, D)), "halves of each block");
  check(ok(half(0, 2 * thd, D, T * D), half(thd, 2 * thd, H * D, D)),
        "halves of each block, the heads before the tokens in one");
  check(ok(half(0, 2 * thd, 2 * D, 2 * T * D), half(D, 2 * thd, 2 * D, 2 * T * D)),
        "K and V side by side in each row");
  check(ok(half(0, 2 * thd, 2 * H * D, D), half(H * D, 2 * thd, 2 * H * D, D)),
        "K and V side by side in each token");
  check(!rows_apart(half(0, 0, H * D, D).rows()), "one block for all is not apart");
  check(!rows_apart(half(0, thd, 0, D).rows()), "nor is one token for all");
  check(!rows_apart(half(0, thd, H * D, 0).rows()), "nor one head for all");
  check(!rows_apart(half(0, thd - 16, H * D, D).rows()), "nor blocks that share their ends");
  const Half same = half(0, thd, H * D, D);
  check(rows_meet(same.rows(), same.rows()), "a cache meets itself");
  check(rows_meet(same.rows(), half(thd * (N - 1) + 16, thd, H * D, D).rows()),
        "and one that starts in its last block");
  check(!rows_meet(same.rows(), half(thd * N, thd, H * D, D).rows()), "but not one behind it");
  // blocks of 2 TiB, whose numbers leave 32 bits
  const int64_t far = int64_t(1) << 41;
  check(ok(half(0, far, H * D, D), half(far / 2, far, H * D, D)), "steps past 32 bits");
  check(!ok(half(0, far, H * D, D), half(far * (N - 1), far, H * D, D)), "and that meet there");
}

}  // namespace

int main() {
  views_of_dense_memory();
  steps_of_any_kind();
  layouts_of_engines();
  return failures ? 1 : 0;
}

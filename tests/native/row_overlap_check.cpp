// Host check of mw8::row_sets_meet and rows_apart (csrc/row_overlap.h) against
// bytes marked one by one, over random and nested layouts in a small memory,
// and over ones past 32 and 64 bits.  Prints "mismatches=<n> checked=<m>".
#include "row_overlap.h"

#include <cstdio>
#include <random>
#include <vector>

int main() {
  std::mt19937 rng(1);
  auto pick = [&](int lo, int hi) { return static_cast<int64_t>(std::uniform_int_distribution<int>(lo, hi)(rng)); };
  constexpr int kBytes = 4096, kMid = 1500;
  static char memory[kBytes];
  long long checked = 0, bad = 0, met = 0;
  auto marks = [&](const mw8::RowSet& r, std::vector<int>& m) {
    m.assign(kBytes, 0);
    for (int64_t i = 0; i < r.n_outer; ++i)
      for (int64_t j = 0; j < r.n_inner; ++j)
        for (int64_t b = 0; b < r.len; ++b) ++m[static_cast<const char*>(r.p) - memory + i * r.outer + j * r.inner + b];
  };
  std::vector<int> a, b;
  for (int it = 0; it < 300000; ++it) {
    mw8::RowSet w{memory + kMid + pick(-60, 60), pick(1, 8), pick(1, 5), pick(0, 60), pick(1, 5), pick(0, 60)};
    mw8::RowSet x{memory + kMid + pick(-60, 60), pick(0, 3) ? w.len : pick(1, 40), pick(0, 5), pick(-60, 60), pick(0, 5), pick(-60, 60)};
    if (pick(0, 2) == 0) x.outer = w.outer;  // views of one buffer
    if (pick(0, 2) == 0) x.inner = w.inner;
    if (pick(0, 3) == 0) w.outer = w.inner * pick(1, 6), x.outer = w.outer;
    marks(w, a);
    marks(x, b);
    bool twice = false, shared = false;
    for (int i = 0; i < kBytes; ++i) twice |= a[i] > 1, shared |= a[i] && b[i];
    // apart: no byte twice, and nested (rows that interleave count as overlapping)
    if (mw8::rows_apart(w) && twice) ++bad;
    if (!mw8::rows_apart(w)) continue;
    ++checked;
    met += shared;
    if (mw8::row_sets_meet(w, x) != shared) ++bad;
  }
  if (met < checked / 10 || met > checked * 9 / 10) ++bad;  // both answers are tried
  // far apart: token strides past 2^32 bytes, heads between them
  const int64_t far = int64_t{1} << 40;
  const mw8::RowSet q{reinterpret_cast<void*>(far), 256, 1 << 24, far, 8, 256};
  mw8::RowSet k = q;
  k.p = reinterpret_cast<void*>(far + 8 * 256), k.n_inner = 2;
  if (mw8::row_sets_meet(q, k)) ++bad;
  k.p = reinterpret_cast<void*>(far + 8 * 256 - 1);
  if (!mw8::row_sets_meet(q, k)) ++bad;
  std::printf("mismatches=%lld checked=%lld\n", bad, checked);
  return bad != 0;
}

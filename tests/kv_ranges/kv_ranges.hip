// CPU: the index arithmetic that the paged cache's kernels share with the host
// (srw_kv.hpp), over many calls.  Host code only: no kernel is built or launched.
//   kv_ranges rows    rows of k and v that a unit of 16 positions touches
//   kv_ranges spans   tiles and keys that rows see
#include <stdio.h>
#include <string.h>

#include <random>
#include <vector>

#include "srw_kv.hpp"

static long long failures = 0, checks = 0;
static void expect(bool ok, const char* what, long long a, long long b, long long c, long long d) {
  ++checks;
  if (!ok && ++failures <= 20) printf("FAIL %s: %lld %lld %lld %lld\n", what, a, b, c, d);
}

// Every unit of a sequence with n new tokens of len positions: the rows that are read
// lie in [row0, row0 + n), and every row that has a position in [0, len) is one unit's.
static void rows_of(int64_t row0, int n, int len) {
  const srw::KvSeq s{row0, n, len};
  std::vector<int> mine(n, 0);
  for (int64_t at = -2; at < n / 16 + 4; ++at) {
    srw::KvRun k;
    if (!srw::kv_run(s, at, k)) continue;
    expect(at >= 0 && at < n / 16 + 2, "unit", at, n, len, row0);
    expect(k.base % 16 == 0 && k.first >= 0 && k.first < k.last && k.last <= 16, "run", at, n, len, k.base);
    for (int i = 0; i < 16; ++i) {
      const int64_t row = k.row + srw::kv_in_run(k, i);
      expect(row >= row0 && row < row0 + n, "row", row, row0, n, len);
      if (i >= k.first && i < k.last) {
        expect(k.base + i == len - n + (row - row0), "position", k.base + i, row - row0, n, len);
        if (row >= row0 && row < row0 + n) ++mine[row - row0];
      }
    }
  }
  for (int i = 0; i < n; ++i) expect(mine[i] == 1, "once", i, n, len, mine[i]);
}

static void rows() {
  for (int n = 0; n <= 70; ++n)
    for (int len = 0; len <= 150; ++len)
      for (int64_t row0 : {int64_t{0}, int64_t{5}, int64_t{2147483000}}) rows_of(row0, n, len);
  std::mt19937 g(1);
  for (int i = 0; i < 2000; ++i) rows_of(g() % 100, g() % 3000, g() % 0x7fff0000u);
  rows_of(0, 3, 0x7fff0000);
  rows_of(0, 0, 0x7fff0000 - 5);
}

// Whether a token at position pos sees position j.
static bool sees(long long pos, long long j, long long window, long long sinks) {
  return j <= pos && (window == 0 || j > pos - window || j < sinks);
}

// Rows at positions [p_lo, p_hi]: every position of cap that one of them sees, among
// those in `probe`, lies in exactly one tile of the span, and kv_seen says who sees it.
static void span(int cap, int window, int sinks, int p_lo, int p_hi, const std::vector<int>& probe) {
  const srw::KvSpan s = srw::kv_span(cap, window, sinks, p_lo, p_hi);
  expect(s.tiles >= 0 && s.hi >= 0 && s.hi <= cap, "span", cap, window, p_lo, p_hi);
  for (int i = 0; i < s.tiles; i += s.tiles > 64 ? s.tiles / 32 : 1) {
    expect(s.key0(i) >= 0 && s.key0(i) < cap, "tile", s.key0(i), cap, p_lo, p_hi);
    if (i) expect(s.key0(i) > s.key0(i - 1), "order", i, s.key0(i), window, sinks);
  }
  for (const int j : probe) {
    if (j < 0 || j >= cap) continue;
    bool any = false;
    for (const int p : {p_lo, p_lo + (p_hi - p_lo) / 2, p_hi}) {
      const bool want = sees(p, j, window, sinks);
      any |= want;
      const int key0 = j / srw::kTile * srw::kTile;
      expect((srw::kv_seen(p, key0, window, sinks) >> (j - key0) & 1) == (want ? 1u : 0u), "seen", p, j, window, sinks);
    }
    if (!any) continue;
    const int t = j / srw::kTile;  // tile of the first tokens, or of the window
    const bool in = t < s.sink_tiles || (t - s.skip >= s.sink_tiles && t - s.skip < s.tiles);
    expect(in, "walked", j, p_lo, p_hi, window);
  }
}

static void spans() {
  constexpr int most = 0x7fffffff;
  std::mt19937 g(2);
  std::vector<int> all;
  for (int j = 0; j < 400; ++j) all.push_back(j);
  for (const int window : {0, 1, 2, 63, 64, 65, 130, 1000, most - 1, most})
    for (const int sinks : {0, 1, 4, 64, 70, most})
      for (int p_lo = -200; p_lo < 300; p_lo += 7)
        for (const int n : {0, 1, 15, 127})
          for (const int cap : {0, 16, 320, 400}) {
            if (sinks && !window) continue;
            span(cap, window, sinks, p_lo, p_lo + n, all);
          }
  // the ends of the range
  const int far = 0x7fff0000;
  for (int i = 0; i < 20000; ++i) {
    const int window = i % 3 == 0 ? most - g() % 3 : i % 3 == 1 ? 1 + g() % 5000 : 1 + g() % (most - 1);
    const int sinks = i % 2 ? g() % 100 : g() % most;
    const int n = g() % 128;
    const int p_lo = i % 5 == 0 ? -most + n + static_cast<int>(g() % 100) : static_cast<int>(g() % (far - 200)) - (i % 7 ? 0 : 100);
    const int cap = i % 4 ? far : 1 + g() % far;
    std::vector<int> probe{0, 1, sinks - 1, sinks, cap - 1, p_lo, p_lo + n};
    for (int k = 0; k < 40; ++k) {
      probe.push_back(p_lo >= 0 ? p_lo - static_cast<int>(g() % 200) : k);
      if (p_lo >= window) probe.push_back(p_lo - window + static_cast<int>(g() % 200) - 100);
    }
    span(cap, window, sinks, p_lo, p_lo + n, probe);
  }
}

int main(int argc, char** argv) {
  const char* what = argc > 1 ? argv[1] : "";
  if (!strcmp(what, "rows"))
    rows();
  else if (!strcmp(what, "spans"))
    spans();
  else
    return 2;
  printf("%s: %lld checks, %lld failures\n", what, checks, failures);
  return failures ? 1 : 0;
}

// CPU: the index arithmetic that the paged cache's kernels share with the host
// (srw_kv.hpp), over many calls.  Host code only: no kernel is built or launched.
//   kv_ranges rows    rows of k and v that a unit of 16 positions touches
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

int main(int argc, char** argv) {
  const char* what = argc > 1 ? argv[1] : "";
  if (!strcmp(what, "rows"))
    rows();
  else
    return 2;
  printf("%s: %lld checks, %lld failures\n", what, checks, failures);
  return failures ? 1 : 0;
}

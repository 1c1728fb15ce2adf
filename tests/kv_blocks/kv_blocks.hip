// CPU: whether the layers of two tensors meet (srw_kv.hpp), against every byte.  Host code
// only: no kernel is built or launched.
#include <stdio.h>

#include <random>
#include <vector>

#include "srw_kv.hpp"

int main() {
  std::mt19937 g(1);
  long long failures = 0, meet = 0, inside = 0;
  const int tries = 300000;
  for (int t = 0; t < tries; ++t) {
    auto one = [&] {
      srw::KvBlocks b;
      b.at = 1000 + g() % 60;
      b.bytes = g() % 12;
      b.n = 1 + g() % 6;
      b.stride = b.n > 1 ? b.bytes + g() % 25 : 0;
      return b;
    };
    const srw::KvBlocks a = one();
    srw::KvBlocks b = one();
    if (t % 2) b.stride = b.n > 1 && a.stride > b.bytes ? a.stride : b.stride;  // layers between each other
    std::vector<char> held(1500, 0);
    bool want = false;
    for (int64_t i = 0; i < a.n; ++i)
      for (int64_t k = 0; k < a.bytes; ++k) held[a.at + i * a.stride + k - 1000] = 1;
    for (int64_t i = 0; i < b.n; ++i)
      for (int64_t k = 0; k < b.bytes; ++k) want |= held[b.at + i * b.stride + k - 1000];
    const bool got = srw::kv_meet(a, b);
    meet += want;
    inside += !want && a.at < b.at + (b.n - 1) * b.stride + b.bytes && b.at < a.at + (a.n - 1) * a.stride + a.bytes;
    if (got != want && ++failures <= 20)
      printf("FAIL %d: [%lu %ld %ld %ld] [%lu %ld %ld %ld]\n", want, a.at, a.bytes, a.stride, a.n, b.at, b.bytes, b.stride, b.n);
  }
  printf("%d checks, %lld meet, %lld lie between, %lld failures\n", tries, meet, inside, failures);
  return failures || !meet || !inside;
}

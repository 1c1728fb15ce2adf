// CPU: the whole-number arithmetic that sampling shares with the host (srw_sample.hpp).
// Host code only: no kernel is built or launched.
//   sample_ranges shares    u and p times a sum
//   sample_ranges unders    the largest float32 under a number
//   sample_ranges octaves   octaves under R, over the range of logits and temperatures
#include <math.h>
#include <stdio.h>
#include <string.h>

#include <random>

#include "srw_sample.hpp"

static long long failures = 0, checks = 0;
static void expect(bool ok, const char* what, double a, unsigned long long b, unsigned long long c) {
  ++checks;
  if (!ok && ++failures <= 20) printf("FAIL %s: %.17g %llu %llu\n", what, a, b, c);
}

// f total in 128 bits: f = m 2^-s.
static void share(float f, uint64_t total) {
  int e;
  const float part = frexpf(f, &e);  // f = part 2^e, part of 24 bits in [1/2, 1)
  const unsigned __int128 product = static_cast<unsigned __int128>(static_cast<uint32_t>(ldexpf(part, 24))) * total;
  const int s = 24 - e;
  const unsigned __int128 whole = s < 128 ? product >> s : 0;
  const bool rest = (s < 128 ? whole << s : 0) != product;
  const uint64_t under = srw::share_of<false>(f, total), over = srw::share_of<true>(f, total);
  expect(under == static_cast<uint64_t>(whole), "under", f, total, under);
  expect(over == static_cast<uint64_t>(whole) + rest, "over", f, total, over);
  expect(under < total && over >= 1 && over <= total, "range", f, under, over);
}

static void shares() {
  std::mt19937_64 g(1);
  const float ends[] = {1e-45f, 3e-45f, 1.1754942e-38f, 1.1754944e-38f, 5.9604645e-8f, 0.25f, 0.5f, 0.99999994f, 0.1f,
                        5.421010862427522e-20f, 2.7105054e-20f, 1.0842022e-19f, 3.2311743e-27f, 6.4623485e-27f};
  for (int b = 0; b <= 62; ++b)
    for (const uint64_t t : {uint64_t{1} << b, (uint64_t{1} << b) + 1, (uint64_t{1} << b) - 1 + (b == 0)}) {
      for (const float f : ends) share(f, t ? t : 1);
      for (int i = 0; i < 2000; ++i) {
        const float f = ldexpf(static_cast<float>((g() >> 41) + 1), -24 - static_cast<int>(g() % 90));
        share(f < 1.f ? f : 0.5f, t ? t : 1);
      }
    }
  for (int i = 0; i < 2000000; ++i) share(static_cast<float>((g() >> 40) | 1) * 5.9604645e-8f, (g() >> (2 + g() % 60)) | 1);
}

// float_under(x): a float that is not above x, and the next one is.
static void under(double x) {
  const float f = srw::float_under(x), next = nextafterf(f, INFINITY);
  expect(static_cast<double>(f) <= x && static_cast<double>(next == 0.f ? 0.f : next) > x, "under", x, 0, 0);
  expect(f == f && srw::of_key(srw::key_of(f)) == f, "key", x, srw::key_of(f), 0);
}

static void unders() {
  std::mt19937_64 g(3);
  for (const double x : {0.0, -0.0, 1e-60, -1e-60, 1e-46, -1e-46, 7e-46, -7e-46, 1.4e-45, -1.4e-45, 2e-45, -2e-45, 1.1754943e-38,
                         -1.1754943e-38, 1.0, -1.0, 1.0000000001, -1.0000000001, 0.9999999999, 3.4028234663852886e38,
                         -3.4028234663852886e38, 3.4e38, 16777217.0, -16777217.0})
    under(x);
  for (int i = 0; i < 1000000; ++i) {
    const double x = ldexp(static_cast<double>(g() >> 11), -180 + static_cast<int>(g() % 250));
    under(x);
    under(-x);
  }
}

// 128 y = 128 (R - octaves) and up to a step beside it.
static void octave(int R, int octaves, int beside) {
  const int64_t y = 128 * (static_cast<int64_t>(R) - octaves) + beside;
  const int n = static_cast<int>(y);
  expect(srw::steps_under(R, n) == 128 * octaves - beside, "steps", R, octaves, beside);
  const uint64_t one = static_cast<uint64_t>(static_cast<uint32_t>(srw::at_octave(0x3ff00000, n, R))) << 32;
  const int64_t whole = y >= 0 ? y / 128 : -((127 - y) / 128);  // rounded down
  expect(__builtin_bit_cast(double, one) == ldexp(1.0, static_cast<int>(whole - R)), "high word", R, octaves, beside);
}

static void octaves() {
  std::mt19937_64 g(2);
  for (int b = 0; b <= 30; ++b)
    for (const int R : {1 << b, -(1 << b), (1 << b) - 1, 1 - (1 << b)})
      for (int o = 0; o < 1000; o += b < 24 ? 7 : 1)
        for (const int beside : {0, 1, 63, 64, 127}) octave(R, o, beside);
  for (int i = 0; i < 1000000; ++i)
    octave(static_cast<int>(g() % (1u << 31)) - (1 << 30), static_cast<int>(g() % 1000), static_cast<int>(g() % 128));
}

int main(int argc, char** argv) {
  if (argc < 2) return 2;
  if (!strcmp(argv[1], "shares")) shares();
  if (!strcmp(argv[1], "octaves")) octaves();
  if (!strcmp(argv[1], "unders")) unders();
  printf("%lld checks, %lld failures\n", checks, failures);
  return failures ? 1 : 0;
}

// srw_sample.hpp -- the whole-number arithmetic of sampling that host and device share
// (srw_sample.hip).
#pragma once

#include <math.h>
#include <stdint.h>

#include <hip/hip_runtime.h>

namespace srw {

// A number's place among all: larger logits have larger keys, -0 is 0, NaN the
// smallest.
__host__ __device__ inline uint32_t key_of(float l) {
  const uint32_t b = __builtin_bit_cast(uint32_t, l + 0.f);
  if (l != l) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__host__ __device__ inline float of_key(uint32_t k) {
  return k == 0 ? -INFINITY : __builtin_bit_cast(float, k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
// The largest float that is not above x.
__host__ __device__ inline float float_under(double x) {
  const float f = static_cast<float>(x);
  if (!(static_cast<double>(f) > x)) return f;
  return of_key(key_of(f) - (f == 0.f ? 2 : 1));  // (the key under 0's is -0's, which no number has)
}

// f times total, 0 < f < 1, rounded to the whole number below or (UP) above: f has 24
// bits, total 62 at most.
template <bool UP>
__host__ __device__ inline uint64_t share_of(float f, uint64_t total) {
  const uint32_t bits = __builtin_bit_cast(uint32_t, f), e = bits >> 23, m = (bits & 0x7fffffu) | (e ? 0x800000u : 0u);
  const int s = 150 - static_cast<int>(e ? e : 1);  // f = m 2^-s, s at least 24
  const uint64_t b = static_cast<uint64_t>(m) * static_cast<uint32_t>(total);
  const uint64_t high = static_cast<uint64_t>(m) * static_cast<uint32_t>(total >> 32) + (b >> 32);  // under 2^55
  const uint32_t low = static_cast<uint32_t>(b);  // m total = high 2^32 + low
  const int d = s < 32 ? 0 : s < 95 ? s - 32 : 63, l = s < 32 ? s : 32;
  const uint64_t whole = (high >> d) << (32 - l) | (static_cast<uint64_t>(low) >> l);
  const bool rest = (high & ((uint64_t{1} << d) - 1)) != 0 || (low & ((uint64_t{1} << l) - 1)) != 0;
  return UP ? whole + rest : whole;
}

// n: the low 32 bits of 128 y, a whole number; |y| and |R| up to 2^30.  128 (R - y), where
// y lies under 2^24 from R; and the high word of a double times 2^(y rounded down - R),
// where that is a double.  (128 R alone can pass 32 bits; what lies above them falls out
// of the difference.)
__host__ __device__ inline int steps_under(int R, int n) {
  return static_cast<int>(128u * static_cast<uint32_t>(R) - static_cast<uint32_t>(n));
}
__host__ __device__ inline int at_octave(int high, int n, int R) {
  return static_cast<int>(static_cast<uint32_t>(high) + (static_cast<uint32_t>((n >> 7) - R) << 20));
}

}  // namespace srw

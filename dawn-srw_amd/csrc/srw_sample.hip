// srw_sample.hip -- one token of every row of logits, from given random numbers.
//
// Of a row of logits l, with its largest M (NaN counts as -infinity) and a
// temperature t > 0, a token weighs w = exp((l - M) / t).  Tokens are ordered by
// their logits, the largest first, equal ones by index; top-k, top-p and min-p
// each keep a first part of that order, and the token drawn is the first, by
// index, at which the kept weights' running sum passes u times their sum.
//
// Weights are whole numbers W = round(2^q w), w from a polynomial in 64 bits (to
// 2^-46), q as large as V W < 2^62 allows: sums of them are exact, so no order of
// adding, no atomic and no split of the row changes what a row gives, and a
// border is where 64 bits put it.  What rounds to zero cannot be drawn and takes
// no part.
//
// Nothing is sorted.  One pass finds M, a second one counts (and, for top-p,
// sums) tokens by how far they lie under M, in 2 048 steps of equal width: the
// border of top-k or top-p lies in the first step at which the running count or
// sum reaches it.  The tokens down to that step, if there are no more than kList,
// become a list in LDS, on which the rest is done: the border's place within its
// step by digits of the logits' bits, and the draw by digits of the index.  Rows
// that keep more are walked again instead.

#include <math.h>

#include "srw_internal.hpp"
#include "srw_mfma_util.hpp"

namespace srw {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kSteps = 2048;   // of the distance under M
constexpr int kList = 4096;    // tokens that LDS holds

struct SampleArgs {
  const char* logits;
  int64_t stride;  // elements
  int32_t V, q;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* token;
  float* logprob;
};

// A number's place among all: larger logits have larger keys, -0 is 0, NaN the
// smallest.
__device__ inline uint32_t key_of(float l) {
  const uint32_t b = __float_as_uint(l + 0.f);
  if (l != l) return 0;
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ inline float of_key(uint32_t k) {
  return k == 0 ? -INFINITY : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// What a row's weights go by.
struct Weights {
  double M, c;  // largest logit, log2 e / t
  bool inf;     // M is infinite: its tokens weigh 1, all others nothing
  int q;
  // log2 of the weight
  __device__ double log2w(float l) const {
    if (inf) return l == INFINITY ? 0.0 : -INFINITY;
    return (static_cast<double>(l) - M) * c;
  }
  __device__ bool some(double y) const { return y > -(q + 1.0); }  // (false for NaN)
  // 2^y for y in (-q - 1, 0]: the exponential's series over half a unit of the
  // exponent, (ln 2 / 2)^12 / 12! = 6e-15 short at most
  __device__ static double weight(double y) {
    const double n = rint(y), r = y - n;
    double p = 4.4455382718708115e-10;
    p = fma(p, r, 7.0549116208011233e-09);
    p = fma(p, r, 1.0178086009239699e-07);
    p = fma(p, r, 1.3215486790144309e-06);
    p = fma(p, r, 1.5252733804059841e-05);
    p = fma(p, r, 1.5403530393381609e-04);
    p = fma(p, r, 1.3333558146428443e-03);
    p = fma(p, r, 9.6181291076284772e-03);
    p = fma(p, r, 5.5504108664821580e-02);
    p = fma(p, r, 2.4022650695910072e-01);
    p = fma(p, r, 6.9314718055994531e-01);
    p = fma(p, r, 1.0);
    return ldexp(p, static_cast<int>(n));
  }
  // round(2^q w), w <= 1: the low bits of a sum whose last place is 2^-q
  __device__ uint64_t whole(double w) const {
    return static_cast<uint64_t>(__double_as_longlong(w + ldexp(1.0, 52 - q))) & 0xfffffffffffffull;
  }
  __device__ uint64_t of(float l) const {
    const double y = log2w(l);
    return some(y) ? whole(weight(y)) : 0;
  }
};

template <typename T> struct Row {
  static constexpr int E = 16 / sizeof(T);  // logits of a vector
  const T* p;
  int V, off, n;  // the row begins off logits behind a 16-byte border; its vectors
  __device__ Row(const SampleArgs& a, int64_t b) {
    p = reinterpret_cast<const T*>(a.logits) + b * a.stride;
    V = a.V;
    off = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    n = (off + V + E - 1) / E;
  }
  // Vector v: logits E v - off ...; those outside the row as NaN.
  __device__ void get(int v, float (&x)[E]) const {
    const int i = v * E - off;
    if (i >= 0 && i + E <= V) {
      const u32x4_t w = *reinterpret_cast<const u32x4_t*>(p + i);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if constexpr (E == 4) {
          x[j] = __uint_as_float(w[j]);
        } else {
          x[2 * j] = lo_f32(w[j]);
          x[2 * j + 1] = hi_f32(w[j]);
        }
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        x[j] = __uint_as_float(0x7fc00000u);
        if (i + j >= 0 && i + j < V) {
          if constexpr (E == 4)
            x[j] = p[i + j];
          else
            x[j] = __uint_as_float(static_cast<uint32_t>(p[i + j]) << 16);
        }
      }
    }
  }
  // f(index, logit) of the vectors [v0, v1), one a lane, by the whole wave
  template <class F>
  __device__ void walk(int v0, int v1, F f) const {
    constexpr int U = 4;  // loads in flight
    for (int v = v0 + (threadIdx.x & 63); v < v1; v += 64 * U) {
      float x[U][E];
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (v + 64 * k < v1) get(v + 64 * k, x[k]);
#pragma unroll
      for (int k = 0; k < U; ++k)
        if (v + 64 * k < v1)
#pragma unroll
          for (int j = 0; j < E; ++j) f((v + 64 * k) * E - off + j, x[k][j]);
    }
  }
  // the part of the row that is this wave's
  template <class F>
  __device__ void mine(F f) const {
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = (n + kWaves - 1) / kWaves;
    walk(wave * per, (wave + 1) * per < n ? (wave + 1) * per : n, f);
  }
};

template <class T, class Op>
__device__ inline T wave_all(T v, Op op) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) v = op(v, __shfl_xor(v, w));
  return v;
}
// Sums over this lane and those before it.
template <class T>
__device__ inline T wave_scan(T v) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    const T o = __shfl_up(v, w);
    if (lane >= w) v += o;
  }
  return v;
}

struct Shared {
  uint32_t count[kSteps];
  unsigned long long mass[kSteps];
  unsigned long long list[kList];  // key << 32 | index
  unsigned long long wave_mass[kWaves];
  uint32_t wave_count[kWaves];
  float wave_max[kWaves];
  // a crossing: the bin, what lies before it and in it
  int bin;
  uint32_t before_n, in_n, listed, lo, hi;
  unsigned long long before_m, in_m;
};

__device__ inline uint64_t block_sum(Shared& s, uint64_t v) {
  const int wave = threadIdx.x >> 6;
  v = wave_all(v, [](uint64_t a, uint64_t b) { return a + b; });
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s.wave_mass[wave] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) v += s.wave_mass[w];
  __syncthreads();
  return v;
}

// The first of n = 256 or kSteps bins (of s.count and, with BY_MASS, s.mass) at
// which the running count (or mass) reaches target; nothing is written where it
// never does (s.bin = -1 before).  All threads; s is read after a barrier.
template <bool BY_MASS>
__device__ inline void crossing(Shared& s, int n, uint64_t target, uint32_t before_n, uint64_t before_m) {
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  constexpr int per = kSteps / kThreads;  // bins a thread
  uint32_t c[per], cs = 0;
  uint64_t m[per], ms = 0;
#pragma unroll
  for (int k = 0; k < per; ++k) {
    const int i = tid * per + k;
    c[k] = i < n ? s.count[i] : 0;
    m[k] = BY_MASS && i < n ? s.mass[i] : 0;
    cs += c[k];
    ms += m[k];
  }
  uint32_t cr = wave_scan(cs);
  uint64_t mr = BY_MASS ? wave_scan(ms) : 0;
  if (lane == 63) {
    s.wave_count[wave] = cr;
    if constexpr (BY_MASS) s.wave_mass[wave] = mr;
  }
  if (tid == 0) s.bin = -1;
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    before_n += s.wave_count[w];
    if constexpr (BY_MASS) before_m += s.wave_mass[w];
  }
  before_n += cr - cs;
  before_m += mr - ms;
#pragma unroll
  for (int k = 0; k < per; ++k) {
    const uint64_t was = BY_MASS ? before_m : before_n, is = BY_MASS ? before_m + m[k] : before_n + c[k];
    if (was < target && is >= target) {
      s.bin = tid * per + k;
      s.before_n = before_n;
      s.before_m = before_m;
      s.in_n = c[k];
      s.in_m = m[k];
    }
    before_n += c[k];
    before_m += m[k];
  }
  __syncthreads();
}

// Among candidates, the rank (the largest first, of `bits` bits) at which the
// running count (or mass) reaches target >= 1, with what lies before that rank and
// in it.  each(f) calls f(rank, mass) for every candidate of this thread.  There
// must be such a rank.
struct Found {
  uint32_t rank, before_n, in_n;
  uint64_t before_m, in_m;
};
template <bool BY_MASS, class Each>
__device__ inline Found select(Shared& s, int bits, uint64_t target, Each each) {
  Found f{0, 0, 0, 0, 0};
  int left = bits;
  while (left > 0) {
    const int d = left < 8 ? left : 8, shift = left - d;
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
    __syncthreads();
    each([&](uint32_t rank, uint64_t m) {
      if (left < 32 && rank >> left != f.rank) return;
      const int bin = (1 << d) - 1 - static_cast<int>(rank >> shift & ((1u << d) - 1));  // the largest first
      atomicAdd(&s.count[bin], 1u);
      if constexpr (BY_MASS) atomicAdd(&s.mass[bin], static_cast<unsigned long long>(m));
    });
    __syncthreads();
    crossing<BY_MASS>(s, 1 << d, target, f.before_n, f.before_m);
    f.rank = f.rank << d | static_cast<uint32_t>((1 << d) - 1 - s.bin);
    f.before_n = s.before_n;
    f.before_m = s.before_m;
    f.in_n = s.in_n;
    f.in_m = s.in_m;
    left = shift;
  }
  return f;
}

__device__ inline int bits_of(uint32_t most) { return most == 0 ? 1 : 32 - __clz(most); }

// A first part of the order: tokens of larger keys, and those of this key up to an
// index.
struct Cut {
  uint32_t key, index;
  __device__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= index); }
};

template <typename T>
__global__ __launch_bounds__(kThreads) void sample_kernel(SampleArgs a) {
  __shared__ Shared s;
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const Row<T> row(a, b);
  constexpr int E = Row<T>::E;
  const float t = a.temperature ? a.temperature[b] : a.temperature_all;
  const int k = a.top_k ? a.top_k[b] : a.top_k_all;
  const float p = a.top_p ? a.top_p[b] : a.top_p_all;
  float least = a.min_p ? a.min_p[b] : a.min_p_all;
  least = least > 0.f ? (least < 1.f ? least : 1.f) : 0.f;
  const float u = a.u[b];

  float m = -INFINITY;
  row.mine([&](int, float l) { m = fmaxf(m, l); });
  m = wave_all(m, [](float x, float y) { return fmaxf(x, y); });
  if (lane == 0) s.wave_max[wave] = m;
  if (tid == 0) {
    s.listed = 0;
    s.lo = 0xffffffffu;
    s.hi = 0;
  }
  for (int i = tid; i < kSteps; i += kThreads) {
    s.count[i] = 0;
    s.mass[i] = 0;
  }
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s.wave_max[w]);
  if (m == -INFINITY) {  // nothing to draw
    if (tid == 0) {
      a.token[b] = -1;
      if (a.logprob) a.logprob[b] = -INFINITY;
    }
    return;
  }
  const bool greedy = !(t > 0.f);
  if (greedy || (k == 1)) {
    row.mine([&](int i, float l) {
      if (l == m) atomicMin(&s.lo, static_cast<uint32_t>(i));
    });
    __syncthreads();
    if (tid == 0) {
      a.token[b] = s.lo;
      if (a.logprob) a.logprob[b] = 0.f;
    }
    return;
  }

  Weights wt;
  wt.M = m;
  wt.c = 1.4426950408889634 / static_cast<double>(t);
  wt.inf = m == INFINITY;
  wt.q = a.q;
  const bool by_k = k > 0 && k < a.V, by_p = p < 1.f;
  // steps under M: any way that never puts a smaller logit before a larger one does
  float scale = (kSteps - 1) / (static_cast<float>(a.q + 1) * 0.6931472f * t);
  scale = scale < 3e38f ? scale : 3e38f;
  auto step = [&](float l) {
    const float x = (m - l) * scale;
    return x < kSteps - 1 ? static_cast<int>(x) : kSteps - 1;
  };

  Cut cut{0, 0xffffffffu};  // all
  bool listed = false;      // the tokens of the cut, and some behind it, are a list
  // f(key, index, logit) of the list's tokens, or the row's, that weigh anything
  auto each_listed = [&](auto f) {
    for (uint32_t i = tid; i < s.listed; i += kThreads) {
      const uint64_t e = s.list[i];
      f(static_cast<uint32_t>(e >> 32), static_cast<uint32_t>(e), of_key(static_cast<uint32_t>(e >> 32)));
    }
  };
  auto each_in_row = [&](auto f) {
    row.mine([&](int i, float l) {
      if (wt.some(wt.log2w(l))) f(key_of(l), static_cast<uint32_t>(i), l);
    });
  };
  // the cut at which the running count or mass of the tokens with keys in [lo, hi] (of
  // the present cut) reaches target
  auto narrow = [&](auto by_mass, uint32_t lo, uint32_t hi, uint64_t target) {
    constexpr bool M = decltype(by_mass)::value;
    auto among = [&](auto each) {
      const Found f = select<M>(s, bits_of(hi - lo), target, [&](auto g) {
        each([&](uint32_t key, uint32_t i, float l) {
          if (key >= lo && key <= hi && cut.keeps(key, i)) g(key - lo, M ? wt.of(l) : 0);
        });
      });
      const uint32_t key = lo + f.rank;
      // equal ones: as many as it takes
      uint64_t n = target - (M ? f.before_m : f.before_n);
      if constexpr (M) {
        const uint64_t one = f.in_m / f.in_n;
        n = (n + one - 1) / one;
      }
      uint32_t index = cut.key == key ? cut.index : 0xffffffffu;
      if (n < f.in_n) {
        const uint32_t last = a.V - 1;
        const Found g = select<false>(s, bits_of(last), n, [&](auto h) {
          each([&](uint32_t ky, uint32_t i, float) {
            if (ky == key && cut.keeps(ky, i)) h(last - i, 0);
          });
        });
        index = last - g.rank;
      }
      cut = Cut{key, index};
    };
    if (listed)
      among(each_listed);
    else
      among(each_in_row);
  };

  if (by_k || by_p) {
    const bool sums = by_p && !by_k;
    row.mine([&](int, float l) {
      const double y = wt.log2w(l);
      if (wt.some(y)) {
        const int i = step(l);
        if (sums) {
          const uint64_t w = wt.whole(Weights::weight(y));
          atomicAdd(&s.mass[i], static_cast<unsigned long long>(w));
        }
        atomicAdd(&s.count[i], 1u);
      }
    });
    __syncthreads();
    uint64_t target = k;
    if (sums) {
      uint64_t all = 0;
      for (int i = tid; i < kSteps; i += kThreads) all += s.mass[i];
      all = block_sum(s, all);
      const double x = ceil(static_cast<double>(p) * static_cast<double>(all));
      target = x >= 1.0 ? static_cast<uint64_t>(x) : 1;
      target = target < all ? target : all;
      crossing<true>(s, kSteps, target, 0, 0);
    } else {
      crossing<false>(s, kSteps, target, 0, 0);
    }
    const int border = s.bin;
    const uint32_t before_n = s.before_n, in_n = s.in_n;
    const uint64_t before_m = s.before_m;
    if (border >= 0) {  // (fewer than k weigh anything: k keeps them all)
      listed = before_n + in_n <= kList;
      uint32_t lo = 0xffffffffu, hi = 0;
      row.mine([&](int i, float l) {
        if (!wt.some(wt.log2w(l))) return;
        const int at = step(l);
        if (at > border) return;
        const uint32_t key = key_of(l);
        if (at == border) {
          lo = key < lo ? key : lo;
          hi = key > hi ? key : hi;
        }
        if (listed) s.list[atomicAdd(&s.listed, 1u)] = static_cast<uint64_t>(key) << 32 | static_cast<uint32_t>(i);
      });
      lo = wave_all(lo, [](uint32_t x, uint32_t y) { return x < y ? x : y; });
      hi = wave_all(hi, [](uint32_t x, uint32_t y) { return x > y ? x : y; });
      if (lane == 0) {
        atomicMin(&s.lo, lo);
        atomicMax(&s.hi, hi);
      }
      __syncthreads();
      lo = s.lo;
      hi = s.hi;
      if (sums)
        narrow(std::true_type{}, lo, hi, target - before_m);
      else
        narrow(std::false_type{}, lo, hi, target - before_n);
    }
  }

  // top-p of what top-k left
  if (by_k && by_p) {
    uint64_t all = 0;
    auto add = [&](uint32_t key, uint32_t i, float l) {
      if (cut.keeps(key, i)) all += wt.of(l);
    };
    if (listed)
      each_listed(add);
    else
      each_in_row(add);
    all = block_sum(s, all);
    const double x = ceil(static_cast<double>(p) * static_cast<double>(all));
    uint64_t target = x >= 1.0 ? static_cast<uint64_t>(x) : 1;
    target = target < all ? target : all;
    narrow(std::true_type{}, cut.key, key_of(m), target);
  }

  // the draw
  auto weight_kept = [&](uint32_t key, uint32_t i, float l) -> uint64_t {
    if (!cut.keeps(key, i)) return 0;
    const double y = wt.log2w(l);
    if (!wt.some(y)) return 0;
    const double w = Weights::weight(y);
    return w >= least ? wt.whole(w) : 0;
  };
  auto want = [&](uint64_t total) {  // running sums over this are behind the draw
    const double x = u > 0.f ? static_cast<double>(u) * static_cast<double>(total) : 0.0;
    const uint64_t at = x < static_cast<double>(total) ? static_cast<uint64_t>(x) : total;
    return at < total ? at : total - 1;
  };
  auto done = [&](uint32_t index, float l, uint64_t total) {
    a.token[b] = index;
    if (a.logprob)
      a.logprob[b] = static_cast<float>(wt.log2w(l) * 0.6931471805599453 -
                                        log(ldexp(static_cast<double>(total), -wt.q)));
  };
  if (listed) {
    uint64_t total = 0;
    each_listed([&](uint32_t key, uint32_t i, float l) { total += weight_kept(key, i, l); });
    total = block_sum(s, total);
    const uint32_t last = a.V - 1;
    const Found f = select<true>(s, bits_of(last), want(total) + 1, [&](auto g) {
      each_listed([&](uint32_t key, uint32_t i, float l) {
        const uint64_t w = weight_kept(key, i, l);
        if (w) g(last - i, w);
      });
    });
    each_listed([&](uint32_t, uint32_t i, float l) {
      if (i == last - f.rank) done(i, l, total);
    });
    return;
  }
  int v0 = 0, v1 = row.n;
  uint64_t total = 0, at = 0;
  for (bool first = true; first || v1 - v0 > 64; first = false) {
    const int per = (v1 - v0 + kWaves - 1) / kWaves;
    const int w0 = v0 + wave * per, w1 = w0 + per < v1 ? w0 + per : v1;
    uint64_t sum = 0;
    row.walk(w0, w1, [&](int i, float l) { sum += weight_kept(key_of(l), static_cast<uint32_t>(i), l); });
    sum = wave_all(sum, [](uint64_t x, uint64_t y) { return x + y; });
    __syncthreads();
    if (lane == 0) s.wave_mass[wave] = sum;
    __syncthreads();
    if (first) {
      for (int w = 0; w < kWaves; ++w) total += s.wave_mass[w];
      at = want(total);
    }
    int w = 0;
    while (w < kWaves - 1 && at >= s.wave_mass[w]) at -= s.wave_mass[w++];
    v0 += w * per;
    v1 = v0 + per < v1 ? v0 + per : v1;
  }
  if (wave == 0) {
    float x[E];
    uint64_t w[E], sum = 0;
    const int v = v0 + lane;
    if (v < v1) row.get(v, x);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = v < v1 ? weight_kept(key_of(x[j]), static_cast<uint32_t>(v * E - row.off + j), x[j]) : 0;
      sum += w[j];
    }
    uint64_t run = wave_scan(sum) - sum;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (run <= at && at < run + w[j]) done(static_cast<uint32_t>(v * E - row.off + j), x[j], total);
      run += w[j];
    }
  }
}

srw_status_t check_sample(const srw_sample_t* d) {
  if (!d) return SRW_EINVAL;
  if (d->B < 0 || d->V < 1 || (d->dtype != SRW_F32 && d->dtype != SRW_BF16)) return SRW_EINVAL;
  if (d->B > (1 << 21) || d->V > (1 << 24)) return SRW_EUNSUPPORTED;  // (a launch has under 2^32 threads)
  if (d->B == 0) return SRW_OK;
  auto array = [](const void* p, size_t size, bool needed) {
    return p ? reinterpret_cast<uintptr_t>(p) % size == 0 : !needed;
  };
  if (!array(d->logits, d->dtype == SRW_F32 ? 4 : 2, true) || !array(d->u, 4, true) || !array(d->token, 8, true) ||
      !array(d->logprob, 4, false) || !array(d->temperature, 4, false) || !array(d->top_k, 4, false) ||
      !array(d->top_p, 4, false) || !array(d->min_p, 4, false))
    return SRW_EINVAL;
  if (d->B > 1 && d->row_stride < 0) return SRW_EINVAL;
  if (!d->temperature && !(d->temperature_all >= 0.f)) return SRW_EINVAL;
  if (!d->top_k && d->top_k_all < 0) return SRW_EINVAL;
  if (!d->top_p && !(d->top_p_all >= 0.f && d->top_p_all <= 1.f)) return SRW_EINVAL;
  if (!d->min_p && !(d->min_p_all >= 0.f && d->min_p_all <= 1.f)) return SRW_EINVAL;
  return SRW_OK;
}

}  // namespace
}  // namespace srw

extern "C" srw_status_t srw_sample(const srw_sample_t* d, void* stream) {
  const srw_status_t st = srw::check_sample(d);
  if (st != SRW_OK || d->B == 0) return st;
  srw::SampleArgs a{};
  a.logits = static_cast<const char*>(d->logits);
  a.stride = d->row_stride;
  a.V = static_cast<int32_t>(d->V);
  int bits = 0;  // V <= 2^bits
  while ((int64_t{1} << bits) < d->V) ++bits;
  a.q = 62 - bits < 51 ? 62 - bits : 51;
  a.u = d->u;
  a.temperature = d->temperature;
  a.top_p = d->top_p;
  a.min_p = d->min_p;
  a.top_k = d->top_k;
  a.temperature_all = d->temperature_all;
  a.top_p_all = d->top_p_all;
  a.min_p_all = d->min_p_all;
  a.top_k_all = d->top_k_all;
  a.token = d->token;
  a.logprob = d->logprob;
  (void)hipGetLastError();
  const dim3 grid(static_cast<unsigned>(d->B));
  if (d->dtype == SRW_F32)
    hipLaunchKernelGGL((srw::sample_kernel<float>), grid, dim3(srw::kThreads), 0, static_cast<hipStream_t>(stream), a);
  else
    hipLaunchKernelGGL((srw::sample_kernel<uint16_t>), grid, dim3(srw::kThreads), 0, static_cast<hipStream_t>(stream), a);
  return hipGetLastError() == hipSuccess ? SRW_OK : SRW_EHIP;
}

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
// Nothing is sorted.  One pass finds M.  A threshold that the border of top-k or
// top-p cannot lie above comes from counts or sums of tokens by how far they lie
// under M, in steps of 2^(1/64); the tokens down to it, if there are no more than
// kList, become a list that a workgroup holds in registers, and the rest is done on
// them: the border by digits of the logits' bits, the draw by digits of the index.
// Rows that keep more are walked again instead.

#include <math.h>

#include "srw_internal.hpp"
#include "srw_mfma_util.hpp"

namespace srw {
namespace {

constexpr int kSteps = 2048;   // of 2^(1/64) under M
constexpr int kList = 4096;    // tokens that a workgroup's registers hold
constexpr int kDigit = 9;      // bits of a select's pass

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
__device__ inline float float_under(double x) {  // the largest float that is not above x
  const float f = static_cast<float>(x);
  if (!(static_cast<double>(f) > x)) return f;
  return of_key(key_of(f) - 1);
}

// What a row's weights go by: log2 w = (l - M) c, c = log2 e / t.
struct Weights {
  double c, M, lowest, unit;  // lowest: what weighs less rounds to zero; unit 2^(52 - q)
  int q;
  const double* tab;                // 2^(j / 64)
  __device__ double log2w(float l) const { return (static_cast<double>(l) - M) * c; }
  // 64 log2 w to the nearest, in the low bits of a sum (of log2 w above -2^25)
  static constexpr double kMagic = 0x1.8p46;
  // round(2^q w): 2^(n / 64) from the table, the rest of the exponent, at most 1 / 128,
  // by a polynomial that is 1 at 0 and elsewhere 5e-15 off at most.  Garbage below
  // `lowest`.
  __device__ uint64_t whole(double y) const {
    const double t = y + kMagic;
    const int n = static_cast<int>(__double_as_longlong(t));
    const double r = y - (t - kMagic);
    double p = 0x1.3b2acb2c36b23p-7;
    p = fma(p, r, 0x1.c6b0b9214b9aep-5);
    p = fma(p, r, 0x1.ebfbdff82bb76p-3);
    p = fma(p, r, 0x1.62e42fefa2417p-1);
    p = fma(p, r, 1.0);
    p *= tab[n & 63];
    p = __hiloint2double(__double2hiint(p) + ((n >> 6) << 20), __double2loint(p));
    // the low bits of a sum whose last place is 2^-q
    return static_cast<uint64_t>(__double_as_longlong(p + unit)) & 0xfffffffffffffull;
  }
  // What a token adds to sums, down to the log2 weight `least` (false for NaN).
  __device__ uint64_t of(float l, double least) const {
    const double y = log2w(l);
    const uint64_t w = whole(y);
    return y >= least ? w : 0;
  }
  // steps of 2^(1/64) under M
  __device__ int step(double y) const {
    const int n = -static_cast<int>(__double_as_longlong(fmax(y, -40.0) + kMagic));
    return n < 0 ? 0 : n < kSteps ? n : kSteps - 1;
  }
};

template <typename T, int NT> struct Row {
  static constexpr int E = 16 / sizeof(T);  // logits of a vector
  const T* p;
  int V, off, n;  // the row begins off logits behind a 16-byte border; its vectors
  __device__ Row(const SampleArgs& a, int64_t b) {
    p = reinterpret_cast<const T*>(a.logits) + b * a.stride;
    V = a.V;
    off = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    n = (off + V + E - 1) / E;
  }
  __device__ float one(int i) const {
    if constexpr (E == 4)
      return p[i];
    else
      return __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
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
        if (i + j >= 0 && i + j < V) x[j] = one(i + j);
      }
    }
  }
  // f(index of the first, logits) of the vectors [v0, v1), one a lane, by the whole wave
  template <class F>
  __device__ void walk(int v0, int v1, F f) const {
    constexpr int U = 4;  // loads in flight
    int v = v0 + (threadIdx.x & 63);
    for (; v + 64 * (U - 1) < v1; v += 64 * U) {
      float x[U][E];
#pragma unroll
      for (int k = 0; k < U; ++k) get(v + 64 * k, x[k]);
#pragma unroll
      for (int k = 0; k < U; ++k) f((v + 64 * k) * E - off, x[k]);
    }
    for (; v < v1; v += 64) {
      float x[E];
      get(v, x);
      f(v * E - off, x);
    }
  }
  // the part of the row that is this wave's
  template <class F>
  __device__ void mine(F f) const {
    constexpr int kWaves = NT / 64;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per = (n + kWaves - 1) / kWaves;
    walk(wave * per, (wave + 1) * per < n ? (wave + 1) * per : n, f);
  }
};

// v of the lane that DPP control C names, 0 where there is none or MASK leaves the
// row of 16 out.
template <int C, int MASK>
__device__ inline uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), C, MASK, 0xf, false));
}
template <int C, int MASK>
__device__ inline uint64_t moved(uint64_t v) {
  return static_cast<uint64_t>(moved<C, MASK>(static_cast<uint32_t>(v >> 32))) << 32 |
         moved<C, MASK>(static_cast<uint32_t>(v));
}
// Sums over this lane and those before it: within rows of 16, then the rows.
template <class N>
__device__ inline N wave_scan(N v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
__device__ inline uint32_t last_lane(uint32_t v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ inline uint64_t last_lane(uint64_t v) {
  return static_cast<uint64_t>(last_lane(static_cast<uint32_t>(v >> 32))) << 32 | last_lane(static_cast<uint32_t>(v));
}
template <class N>
__device__ inline N wave_sum(N v) {
  return last_lane(wave_scan(v));
}
template <class N, class Op>
__device__ inline N wave_all(N v, Op op) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) v = op(v, __shfl_xor(v, w));
  return v;
}

struct Shared {
  double tab[64];
  unsigned long long mass[kSteps];
  uint32_t count[kSteps];
  unsigned long long list[kList];  // key << 32 | index
  unsigned long long wave_m[16];
  uint32_t wave_n[16];
  float wave_max[16];
  // a crossing: the bin (-1: none), what lies before it and in it
  int bin;
  uint32_t before_n, in_n, listed, lo, hi;
  unsigned long long before_m, in_m;
};

template <int NT>
__device__ inline uint64_t block_sum(Shared& s, uint64_t v) {
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) s.wave_m[threadIdx.x >> 6] = v;
  __syncthreads();
  v = 0;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) v += s.wave_m[w];
  __syncthreads();
  return v;
}

// The first of kSteps bins (of s.count, or BY_MASS of s.mass) at which the running
// count (or mass) reaches what target(total) says.
template <int NT, bool BY_MASS, class Target>
__device__ inline void crossing(Shared& s, Target target) {
  const int tid = threadIdx.x, wave = tid >> 6;
  constexpr int per = kSteps / NT;  // bins a thread
  uint64_t x[per], sum = 0;
#pragma unroll
  for (int k = 0; k < per; ++k) {
    x[k] = BY_MASS ? s.mass[tid * per + k] : s.count[tid * per + k];
    sum += x[k];
  }
  uint64_t run = wave_scan(sum);
  if ((tid & 63) == 63) s.wave_m[wave] = run;
  if (tid == 0) s.bin = -1;
  __syncthreads();
  uint64_t total = 0;
  run -= sum;
#pragma unroll
  for (int w = 0; w < NT / 64; ++w) {
    run += w < wave ? s.wave_m[w] : 0;
    total += s.wave_m[w];
  }
  const uint64_t t = target(total);
#pragma unroll
  for (int k = 0; k < per; ++k) {
    if (run < t && run + x[k] >= t) {
      s.bin = tid * per + k;
      s.before_m = run;
    }
    run += x[k];
  }
  __syncthreads();
}

// Among candidates, the rank (the largest first, of `bits` bits) at which the
// running count (or mass) reaches target >= 1, with what lies before that rank and
// in it.  each(f) calls f(rank, mass) for every candidate of this thread.  There
// must be such a rank.
struct Found {
  uint32_t rank, in_n;
  uint64_t before, in_m;
};
template <int NT, bool BY_MASS, class Each>
__device__ inline Found select(Shared& s, int bits, uint64_t target, Each each) {
  constexpr int kBins = 1 << kDigit, kEach = kBins / 64;
  auto place = [](int i) { return i + i / kEach; };  // (a lane's run of bins, over all banks)
  Found f{0, 0, 0, 0};
  int left = bits;
  while (left > 0) {
    const int d = left < kDigit ? left : kDigit, shift = left - d, last = (1 << d) - 1;
    for (int i = threadIdx.x; i < kBins + 64; i += NT) {
      s.count[i] = 0;
      if constexpr (BY_MASS) s.mass[i] = 0;
    }
    __syncthreads();
    each([&](uint32_t rank, uint64_t m) {
      if (left < 32 && rank >> left != f.rank) return;
      const int bin = place(last - static_cast<int>(rank >> shift & static_cast<uint32_t>(last)));  // the largest first
      atomicAdd(&s.count[bin], 1u);
      if constexpr (BY_MASS) atomicAdd(&s.mass[bin], static_cast<unsigned long long>(m));
    });
    __syncthreads();
    if (threadIdx.x < 64) {
      uint32_t c[kEach];
      uint64_t m[kEach], sum = 0;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        const int i = place(threadIdx.x * kEach + k);
        c[k] = s.count[i];
        m[k] = BY_MASS ? s.mass[i] : c[k];
        sum += m[k];
      }
      uint64_t run = f.before + wave_scan(sum) - sum;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        if (run < target && run + m[k] >= target) {
          s.bin = threadIdx.x * kEach + k;
          s.before_m = run;
          s.in_n = c[k];
          s.in_m = m[k];
        }
        run += m[k];
      }
    }
    __syncthreads();
    f.rank = f.rank << d | static_cast<uint32_t>(last - s.bin);
    f.before = s.before_m;
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

template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
  constexpr int kWaves = NT / 64, kEach = kList / NT;  // kEach: a thread's tokens of a list
  constexpr bool kWhole = NT == 256;                   // every row is its own list
  using R = Row<T, NT>;
  constexpr int E = R::E;
  __shared__ Shared s;
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const R row(a, b);
  const float t = a.temperature ? a.temperature[b] : a.temperature_all;
  const int k = a.top_k ? a.top_k[b] : a.top_k_all;
  const float p = a.top_p ? a.top_p[b] : a.top_p_all;
  float least = a.min_p ? a.min_p[b] : a.min_p_all;
  least = least > 0.f ? (least < 1.f ? least : 1.f) : 0.f;
  const float u = a.u[b];

  if (tid < 64) s.tab[tid] = exp2(tid / 64.0);
  if (tid == 0) {
    s.listed = 0;
    s.lo = 0xffffffffu;
    s.hi = 0;
  }
  auto clear = [&] {
    for (int i = tid; i < kSteps; i += NT) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
  };
  clear();
  float mine = -INFINITY;  // the thread's largest
  row.mine([&](int, const float(&x)[E]) {
#pragma unroll
    for (int j = 0; j < E; ++j) mine = fmaxf(mine, x[j]);
  });
  const float wm = wave_all(mine, [](float x, float y) { return fmaxf(x, y); });
  if (lane == 0) s.wave_max[wave] = wm;
  __syncthreads();
  float m = s.wave_max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, s.wave_max[w]);
  if (m == -INFINITY) {  // nothing to draw
    if (tid == 0) {
      a.token[b] = -1;
      if (a.logprob) a.logprob[b] = -INFINITY;
    }
    return;
  }
  if (!(t > 0.f) || k == 1) {  // the first of the largest
    uint32_t first = 0xffffffffu;
    if (mine == m)
      row.mine([&](int i, const float(&x)[E]) {
#pragma unroll
        for (int j = E - 1; j >= 0; --j)
          if (x[j] == m && static_cast<uint32_t>(i + j) < first) first = i + j;
      });
    if (first != 0xffffffffu) atomicMin(&s.lo, first);
    __syncthreads();
    if (tid == 0) {
      a.token[b] = s.lo;
      if (a.logprob) a.logprob[b] = 0.f;
    }
    return;
  }

  // The first token, by index, at which the running sum of f(index, logit) passes
  // at(total): its index goes to done.  Every wave sums a part of the row, then of the
  // part in which that is, until one wave holds the rest.
  auto draw_in_row = [&](auto f, auto at_of, auto done) {
    int v0 = 0, v1 = row.n;
    uint64_t total = 0, at = 0;
    for (bool first = true; first || v1 - v0 > 64; first = false) {
      const int per = (v1 - v0 + kWaves - 1) / kWaves;
      const int w0 = v0 + wave * per, w1 = w0 + per < v1 ? w0 + per : v1;
      uint64_t sum = 0;
      row.walk(w0, w1, [&](int i, const float(&x)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j) sum += f(i + j, x[j]);
      });
      sum = wave_sum(sum);
      __syncthreads();
      if (lane == 0) s.wave_m[wave] = sum;
      __syncthreads();
      if (first) {
        for (int w = 0; w < kWaves; ++w) total += s.wave_m[w];
        at = at_of(total);
      }
      int w = 0;
      while (w < kWaves - 1 && at >= s.wave_m[w]) at -= s.wave_m[w++];
      v0 += w * per;
      v1 = v0 + per < v1 ? v0 + per : v1;
    }
    if (wave != 0) return;
    float x[E];
    uint64_t w[E], sum = 0;
    const int v = v0 + lane;
    if (v < v1) row.get(v, x);
#pragma unroll
    for (int j = 0; j < E; ++j) {
      w[j] = v < v1 ? f(v * E - row.off + j, x[j]) : 0;
      sum += w[j];
    }
    uint64_t run = wave_scan(sum) - sum;
#pragma unroll
    for (int j = 0; j < E; ++j) {
      if (run <= at && at < run + w[j]) done(v * E - row.off + j, x[j], total);
      run += w[j];
    }
  };
  auto share = [&](uint64_t total, double of) -> uint64_t {  // the place of a draw in [0, total)
    const double x = u > 0.f ? static_cast<double>(u) * of : 0.0;
    const uint64_t at = x < of ? static_cast<uint64_t>(x) : total;
    return at < total ? at : total - 1;
  };
  auto part = [&](uint64_t total) -> uint64_t {  // what top-p's run has to reach
    const double x = ceil(static_cast<double>(p) * static_cast<double>(total));
    const uint64_t y = x >= 1.0 ? static_cast<uint64_t>(x) : 1;
    return y < total ? y : total;
  };
  const bool by_k = k > 0 && k < a.V, by_p = p < 1.f;

  if (m == INFINITY) {  // its tokens weigh the same, all others nothing
    uint64_t kept = 0;
    draw_in_row([&](int, float l) -> uint64_t { return l == INFINITY; },
                [&](uint64_t total) {
                  kept = by_k && k < static_cast<int64_t>(total) ? k : total;
                  if (by_p) kept = part(kept);
                  return share(kept, static_cast<double>(kept));
                },
                [&](int i, float, uint64_t) {
                  a.token[b] = i;
                  if (a.logprob) a.logprob[b] = static_cast<float>(-log(static_cast<double>(kept)));
                });
    return;
  }

  Weights wt;
  wt.c = 1.4426950408889634 / static_cast<double>(t);
  wt.M = m;
  wt.q = a.q;
  wt.lowest = -(a.q + 1.0);
  wt.unit = ldexp(1.0, 52 - a.q);
  wt.tab = s.tab;
  double floor_y = wt.lowest;  // of what can be drawn
  if (least > 0.f) floor_y = fmax(floor_y, log2(static_cast<double>(least)));
  const uint32_t key_m = key_of(m);

  auto at_of = [&](uint64_t total) { return share(total, static_cast<double>(total)); };
  auto done = [&](int index, float l, uint64_t total) {
    a.token[b] = index;
    if (a.logprob)
      a.logprob[b] = static_cast<float>(wt.log2w(l) * 0.6931471805599453 -
                                        log(ldexp(static_cast<double>(total), -wt.q)));
  };

  // -- the list ----------------------------------------------------------------------
  Cut cut{0, 0xffffffffu};  // all
  uint32_t key[kEach], index[kEach];
  int n = 0;                // tokens of the list, kEach threads apart
  auto each_listed = [&](auto f) {  // f(key, index, e)
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (tid + e * NT < n) f(key[e], index[e]);
  };
  auto each_in_row = [&](auto f) {
    row.mine([&](int i, const float(&x)[E]) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (wt.log2w(x[j]) >= wt.lowest) f(key_of(x[j]), static_cast<uint32_t>(i + j));
    });
  };
  // the cut at which the running count or mass of the tokens of the present cut with
  // keys in [lo, hi] reaches target
  auto narrow = [&](auto by_mass, auto each, uint32_t lo, uint32_t hi, uint64_t target) {
    constexpr bool BM = decltype(by_mass)::value;
    const Found f = select<NT, BM>(s, bits_of(hi - lo), target, [&](auto g) {
      each([&](uint32_t ky, uint32_t i) {
        if (ky >= lo && ky <= hi && cut.keeps(ky, i)) g(ky - lo, BM ? wt.of(of_key(ky), wt.lowest) : 0);
      });
    });
    const uint32_t border = lo + f.rank;
    // equal ones: as many as it takes
    uint64_t take = target - f.before;
    if constexpr (BM) {
      const uint64_t one = f.in_m / f.in_n;
      take = (take + one - 1) / one;
    }
    uint32_t to = cut.key == border ? cut.index : 0xffffffffu;
    if (take < f.in_n) {
      const uint32_t last = a.V - 1;
      const Found g = select<NT, false>(s, bits_of(last), take, [&](auto h) {
        each([&](uint32_t ky, uint32_t i) {
          if (ky == border && cut.keeps(ky, i)) h(last - i, 0);
        });
      });
      to = last - g.rank;
    }
    cut = Cut{border, to};
  };
  // the row's tokens that `wanted` names become the list; whether it holds them
  auto collect = [&](auto wanted) -> bool {
    row.mine([&](int i, const float(&x)[E]) {
      bool any = false;
#pragma unroll
      for (int j = 0; j < E; ++j) any |= wanted(x[j]);
      if (!any) return;
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (wanted(x[j])) {
          const uint32_t at = atomicAdd(&s.listed, 1u);
          if (at < kList) s.list[at] = static_cast<uint64_t>(key_of(x[j])) << 32 | static_cast<uint32_t>(i + j);
        }
    });
    __syncthreads();
    n = static_cast<int>(s.listed);
    const bool fits = n <= kList;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (fits && tid + e * NT < n) {
        const uint64_t x = s.list[tid + e * NT];
        key[e] = static_cast<uint32_t>(x >> 32);
        index[e] = static_cast<uint32_t>(x);
      }
    __syncthreads();
    if (tid == 0) s.listed = 0;
    __syncthreads();
    if (!fits) n = 0;
    return fits;
  };
  auto under = [&](double steps) { return float_under(static_cast<double>(m) - steps / (64.0 * wt.c)); };

  bool listed = kWhole;  // all that the cut keeps is in the list
  if constexpr (kWhole) {
    n = a.V;
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (tid + e * NT < n) {
        key[e] = key_of(row.one(tid + e * NT));
        index[e] = tid + e * NT;
        if (!(wt.log2w(of_key(key[e])) >= wt.lowest)) key[e] = 0;
      }
    if (by_k) {
      uint64_t weigh = 0;
      each_listed([&](uint32_t ky, uint32_t) { weigh += ky != 0; });
      weigh = block_sum<NT>(s, weigh);
      if (k < static_cast<int64_t>(weigh)) narrow(std::false_type{}, each_listed, 1, key_m, k);
    }
  } else if (by_k || by_p) {
    const bool sums = by_p && !by_k;
    // Top-k of up to NT: where the threads' largest tokens count k, so many lie above.
    const bool by_threads = by_k && k <= NT;
    auto count = [&](float l) {
      const double y = wt.log2w(l);
      if (y >= wt.lowest) atomicAdd(&s.count[wt.step(y)], 1u);
    };
    if (by_threads)
      count(mine);
    else
      row.mine([&](int, const float(&x)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j) {
          if (sums) {
            const double y = wt.log2w(x[j]);
            const uint64_t w = wt.whole(y);
            if (y >= wt.lowest) atomicAdd(&s.mass[wt.step(y)], static_cast<unsigned long long>(w));
          } else {
            count(x[j]);
          }
        }
      });
    __syncthreads();
    uint64_t target = k;
    if (sums)
      crossing<NT, true>(s, [&](uint64_t total) { return target = part(total); });
    else
      crossing<NT, false>(s, [&](uint64_t) { return target; });
    int border = s.bin;
    if (by_threads && border < 0) border = kSteps - 1;
    if (border >= 0) {  // (fewer than k weigh anything: k keeps them all)
      // (half a step more than the border's, for roundings)
      const float from = border == kSteps - 1 ? under(64.0 * (a.q + 2)) : under(border + 1.0);
      const uint64_t before = s.before_m;
      listed = collect([&](float l) { return l >= from; });
      if (listed) {
        uint64_t weigh = 0;
        each_listed([&](uint32_t ky, uint32_t) { weigh += wt.log2w(of_key(ky)) >= wt.lowest; });
        if (sums) {
          narrow(std::true_type{}, each_listed, key_of(from), key_m, target);
        } else {
          weigh = block_sum<NT>(s, weigh);
          if (k < static_cast<int64_t>(weigh)) narrow(std::false_type{}, each_listed, key_of(from), key_m, target);
        }
      } else if (!by_threads &&
                 collect([&](float l) {
                   if (!(l >= from)) return false;
                   const double y = wt.log2w(l);
                   return y >= wt.lowest && wt.step(y) == border;
                 })) {
        // the border's step alone
        uint32_t lo = 0xffffffffu, hi = 0;
        each_listed([&](uint32_t ky, uint32_t) {
          lo = ky < lo ? ky : lo;
          hi = ky > hi ? ky : hi;
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
          narrow(std::true_type{}, each_listed, lo, hi, target - before);
        else
          narrow(std::false_type{}, each_listed, lo, hi, target - before);
      } else {
        uint64_t weigh = 0;
        each_in_row([&](uint32_t, uint32_t) { ++weigh; });
        weigh = block_sum<NT>(s, weigh);
        if (sums)
          narrow(std::true_type{}, each_in_row, 0, key_m, target);
        else if (k < static_cast<int64_t>(weigh))
          narrow(std::false_type{}, each_in_row, 0, key_m, target);
      }
    }
  }

  // top-p of what top-k left, or of a row that is its own list
  if (by_p && (by_k || kWhole)) {
    uint64_t all = 0;
    auto add = [&](uint32_t ky, uint32_t i) {
      if (cut.keeps(ky, i)) all += wt.of(of_key(ky), wt.lowest);
    };
    if (listed) {
      each_listed(add);
      all = block_sum<NT>(s, all);
      narrow(std::true_type{}, each_listed, cut.key, key_m, part(all));
    } else if constexpr (!kWhole) {
      each_in_row(add);
      all = block_sum<NT>(s, all);
      narrow(std::true_type{}, each_in_row, cut.key, key_m, part(all));
    }
  }

  // -- the draw ----------------------------------------------------------------------
  if (listed) {
    uint64_t w[kEach], total = 0;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      w[e] = 0;
      if (tid + e * NT < n && cut.keeps(key[e], index[e])) w[e] = wt.of(of_key(key[e]), floor_y);
      total += w[e];
    }
    total = block_sum<NT>(s, total);
    const uint32_t last = a.V - 1;
    const Found f = select<NT, true>(s, bits_of(last), at_of(total) + 1, [&](auto g) {
#pragma unroll
      for (int e = 0; e < kEach; ++e)
        if (w[e]) g(last - index[e], w[e]);
    });
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (w[e] && index[e] == last - f.rank) done(index[e], of_key(key[e]), total);
  } else if constexpr (!kWhole) {
    if (cut.key == 0) {
      draw_in_row([&](int, float l) { return wt.of(l, floor_y); }, at_of, done);
    } else {
      const float border = of_key(cut.key);
      const int to = cut.index > 0x7fffffffu ? 0x7fffffff : static_cast<int>(cut.index);
      draw_in_row([&](int i, float l) { return l > border || (l == border && i <= to) ? wt.of(l, floor_y) : 0; }, at_of,
                  done);
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
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (d->V <= srw::kList) {
    if (d->dtype == SRW_F32)
      hipLaunchKernelGGL((srw::sample_kernel<float, 256>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((srw::sample_kernel<uint16_t, 256>), grid, dim3(256), 0, s, a);
  } else if (d->dtype == SRW_F32) {
    hipLaunchKernelGGL((srw::sample_kernel<float, 1024>), grid, dim3(1024), 0, s, a);
  } else {
    hipLaunchKernelGGL((srw::sample_kernel<uint16_t, 1024>), grid, dim3(1024), 0, s, a);
  }
  return hipGetLastError() == hipSuccess ? SRW_OK : SRW_EHIP;
}

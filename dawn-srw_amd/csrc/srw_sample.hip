// srw_sample.hip -- one token of every row of logits, from given random numbers.
//
// Of a row of logits l, with its largest M (NaN counts as -infinity) and a
// temperature t > 0, a token weighs w = exp((l - M) / t).  Tokens are ordered by
// their logits, the largest first, equal ones by index; top-k, top-p and min-p
// each keep a first part of that order, and the token drawn is the first, by
// index, at which the kept weights' running sum passes u times their sum.
//
// With y = l log2 e / t, weights are whole numbers W = round(2^(q + y - R)), from a
// polynomial in 64 bits (to 2^-40), R a whole number not under M's y and q as large as
// V W < 2^62 allows, 51 at most: sums of them are exact, so no order of adding and no
// atomic changes what a row gives.  What rounds to zero cannot be drawn and takes no part.
// Rows that need the sum of all logits take it by parts of 8 192 from the first on,
// wherever the row lies, each part over its own R; a part's sum enters the row's rounded
// down to the row's units, and a draw that falls into a part finds its token in the part's.
//
// Nothing is sorted.  A threshold that the border of top-k or top-p cannot lie above
// is found first; the tokens down to it, if there are no more than kList, become a
// list in LDS, and the rest is done on them: borders by digits of the logits' bits,
// the draw by digits of the index.
//
// * Top-k of up to 1 024: the threads' largest logits are counted by steps of
//   2^(1/32); where k of them lie above, so many tokens do.  A larger k: all logits are.
// * Top-p, and rows without either: sample_parts_kernel has summed each part of 8 192
//   logits, for top-p by steps of 2^(1/16).  Of top-p rows that keep more than kList the tokens of the
//   border's step alone become the list; the draw finds its part by the parts' sums and
//   walks that one.  Where min-p lies above the border's step its tokens are the list.
//
// A row of up to 2 048 logits (1 024 by top-k) is its own list.
//
// Measured (calls that follow each other, us): 64 rows of 1 000 float32 by top-p 10.9; one
// row of 30 000 float32, every rule on, 11.3; 64 rows of 32 000 float32 with top-k 11.6 (34
// with k of 2 000), top-p 28, top-p and min-p 21, min-p 13.4, from the whole distribution
// 14, greedy 7.8; 192 rows of 131 073 bf16 with top-p 65 to 67 (one read of them: 9.8); 512
// rows of 100 003 from the whole distribution 54 to 59 in float32 (39.7), and 51 to 56 in
// bf16, by the 64-bit operations of the sums.  A single row is a chain of
// about twenty steps of a workgroup that each wait for memory or a barrier.
//
// A workgroup of sixteen waves has a CU's vector units to itself, and an instruction
// of all of them takes it 16 cycles (24 in 64 bits): what is done for the row as a
// whole is left to one wave, lists are dense so that the waves behind their end have
// nothing to do, and loops over the row test a vector before they look at its logits.

#include <math.h>

#include "srw_internal.hpp"
#include "srw_mfma_util.hpp"
#include "srw_sample.hpp"

namespace srw {
namespace {

constexpr int kSteps = 1024;   // of 2^(1/32) under 2^R
constexpr int kCoarse = 512;   // of 2^(1/16), what parts are summed by
constexpr int kList = 4096;    // tokens of a list
constexpr int kOwnList = 2048; // logits of a row that is its own list, at most
constexpr int kFew = 128;      // tokens that are compared each with each
constexpr int kPart = 8192;    // logits of a part
constexpr int kDigit = 9, kBins = 1 << kDigit;  // bits of a select's pass
constexpr int kMostParts = (1 << 24) / kPart;

struct SampleArgs {
  const char* logits;
  int64_t stride;  // elements
  int32_t V, q, parts;
  const float *u, *temperature, *top_p, *min_p;
  const int32_t* top_k;
  float temperature_all, top_p_all, min_p_all;
  int32_t top_k_all;
  int64_t* token;
  float* logprob;
  // of every row and part: its largest logit, its sum, and for top-p the steps' running
  // sums
  float* part_max;
  unsigned long long *part_sum, *part_steps;
};

// A row's parameters.
struct Rules {
  float t, p, least;
  int k;
  bool greedy, by_k, by_p;
  __device__ __forceinline__ Rules(const SampleArgs& a, int64_t b) {
    t = a.temperature ? a.temperature[b] : a.temperature_all;
    k = a.top_k ? a.top_k[b] : a.top_k_all;
    p = a.top_p ? a.top_p[b] : a.top_p_all;
    least = a.min_p ? a.min_p[b] : a.min_p_all;
    least = least > 0.f ? (least < 1.f ? least : 1.f) : 0.f;
    greedy = !(t > 0.f) || k == 1;
    by_k = k > 0 && k < a.V;
    by_p = p < 1.f;
  }
  // whether the parts' sums are asked for
  __device__ __forceinline__ bool by_parts() const { return !greedy && !by_k && (by_p || least == 0.f); }
};

// 2^(j / 128).
__device__ __forceinline__ void fill_table(double* tab) {
  if (threadIdx.x < 128) tab[threadIdx.x] = exp2(static_cast<int>(threadIdx.x) / 128.0);
}

// What the weights of a row, or of a part, go by.  The same roundings wherever a weight
// is worked out (no contraction): sums of some tokens and of all agree to the last unit.
struct Weights {
  double c, per, unit;  // log2 e / t, and its inverse; 2^(52 - q)
  const double* tab;  // 2^(j / 128)
  int R;
  float lowest;       // smaller logits weigh nothing; above -infinity

  // Whether 2^30 and more lies under M's y: the next smaller logit is 2^6 octaves away
  // and weighs nothing.
  __device__ __forceinline__ static bool peaked(float m, double c) {
    return !(fabs(static_cast<double>(m) * c) < 1073741824.0);
  }
  __device__ __forceinline__ void begin(float t, int q, const double* table) {
    c = 1.4426950408889634 / static_cast<double>(t);
    per = fmin(static_cast<double>(t) * 0.6931471805599453, 1e300);
    unit = ldexp(1.0, 52 - q);
    tab = table;
  }
  __device__ __forceinline__ void set(float m, int q) {
    R = static_cast<int>(ceil(static_cast<double>(m) * c));
    lowest = static_cast<float>(fmax((R - q - 1.0) * per, -3.4028234663852886e38));
  }
  // 128 y to the nearest, in the low bits of a sum
  static constexpr double kMagic = 0x1.8p45;
  __device__ __forceinline__ static int n_of(double t) { return static_cast<int>(__double_as_longlong(t)); }
  __device__ __forceinline__ double sum_of(float l) const {
#pragma clang fp contract(off)
    return static_cast<double>(l) * c + kMagic;
  }
  // W, for logits that weigh something (garbage for others): 2^(n / 128) from the
  // table, the rest of the exponent, at most 1 / 256, by a polynomial that is 1 at 0 and
  // elsewhere 6e-13 off at most.
  __device__ __forceinline__ uint64_t whole(float l) const {
#pragma clang fp contract(off)
    const double y = static_cast<double>(l) * c, t = y + kMagic;
    const int n = n_of(t);
    const double r = y - (t - kMagic);
    double p = fma(0x1.c6b095a17a14dp-5, r, 0x1.ebfbeebe2d1a2p-3);
    p = fma(p, r, 0x1.62e42fefa39efp-1);
    p = fma(p, r, 1.0) * tab[n & 127];
    p = __hiloint2double(at_octave(__double2hiint(p), n, R), __double2loint(p));
    // the low bits of a sum whose last place is 2^-q
    return static_cast<uint64_t>(__double_as_longlong(p + unit)) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ uint64_t of(float l, float least) const {
    const uint64_t w = whole(l);
    return l >= least ? w : 0;
  }
  // steps of 2^(1/32) under 2^R
  __device__ __forceinline__ int step(float l) const {
    const int n = steps_under(R, n_of(sum_of(l)));
    return n < 4 * kSteps ? n >> 2 : kSteps - 1;
  }
};

// log2 x of x in [2^-100, 2^63] (min-p's share, sums in units of 2^R): float32's, mended by
// what it is off.
__device__ __forceinline__ double log2_of(double x, const double* tab) {
  const float l = __builtin_amdgcn_logf(static_cast<float>(x));
  Weights w;
  w.tab = tab;
  const double y = l, t = y + Weights::kMagic;
  const int n = Weights::n_of(t);
  const double r = y - (t - Weights::kMagic);
  double p = fma(0x1.c6b095a17a14dp-5, r, 0x1.ebfbeebe2d1a2p-3);
  p = fma(p, r, 0x1.62e42fefa39efp-1);
  p = fma(p, r, 1.0) * tab[n & 127];
  p = __hiloint2double(at_octave(__double2hiint(p), n, 0), __double2loint(p));  // 2^l
  const double e = (x - p) / p;                                                   // some 1e-7
  return y + e * (1.0 - 0.5 * e) * 1.4426950408889634;
}

// A row: vectors of 16 bytes, the first and the last of them partly outside of it.
template <typename T, int NT> struct Row {
  static constexpr int E = 16 / sizeof(T);  // logits of a vector
  static constexpr int kWaves = NT / 64, kAhead = 8;
  const T* p;
  int V, off, n;  // the row begins off logits behind a 16-byte border; its vectors
  __device__ __forceinline__ Row(const SampleArgs& a, int64_t b) {
    p = reinterpret_cast<const T*>(a.logits) + b * a.stride;
    V = a.V;
    off = static_cast<int>(reinterpret_cast<uintptr_t>(p) % 16 / sizeof(T));
    n = (off + V + E - 1) / E;
  }
  __device__ __forceinline__ float one(int i) const {
    if constexpr (E == 4)
      return p[i];
    else
      return __uint_as_float(static_cast<uint32_t>(p[i]) << 16);
  }
  __device__ __forceinline__ const u32x4_t* at(int v) const { return reinterpret_cast<const u32x4_t*>(p + (v * E - off)); }
  __device__ __forceinline__ static u32x4_t nothing() {
    constexpr uint32_t nan = E == 4 ? 0x7fc00000u : 0x7fc07fc0u;
    return u32x4_t{nan, nan, nan, nan};
  }
  // w with the logit of index i in its place j.
  __device__ __forceinline__ void put(u32x4_t& w, int j, int i) const {
    if constexpr (E == 4)
      w[j] = __float_as_uint(p[i]);
    else
      w[j / 2] = j & 1 ? (w[j / 2] & 0xffffu) | static_cast<uint32_t>(p[i]) << 16 : (w[j / 2] & 0xffff0000u) | p[i];
  }
  // Vector v + lane: logits E (v + lane) - off ...; those outside the row, and those of
  // vectors from `end` on, as NaN.
  __device__ __forceinline__ u32x4_t raw(int v, int end) const {
    const int lane = threadIdx.x & 63, i = (v + lane) * E - off;
    if (v * E >= off && (v + 64) * E - off <= V && v + 64 <= end) return *at(v + lane);
    u32x4_t w = nothing();
    if (v + lane >= end) return w;
    if (i >= 0 && i + E <= V) return *at(v + lane);
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (i + j >= 0 && i + j < V) put(w, j, i + j);
    return w;
  }
  // a, the first `off` logits of it those of b.
  __device__ __forceinline__ u32x4_t headed(u32x4_t a, u32x4_t b) const {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t of_b;
      if constexpr (E == 4)
        of_b = k < off ? 0xffffffffu : 0u;
      else
        of_b = (2 * k < off ? 0xffffu : 0u) | (2 * k + 1 < off ? 0xffff0000u : 0u);
      a[k] = (b[k] & of_b) | (a[k] & ~of_b);
    }
    return a;
  }
  // A lane's share of a part's logits, in any order.  The part's vectors are those from
  // part kPart / E on; its first holds the last `off` logits of the part before, in whose
  // places its own last ones are put, which lie in the vector behind.
  template <int kHeld>
  __device__ __forceinline__ void share(int part, u32x4_t (&held)[kHeld]) const {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int v0 = part * (kPart / E) + wave * 64 * kHeld, begin = part * kPart;
#pragma unroll
    for (int k = 0; k < kHeld; ++k) held[k] = raw(v0 + 64 * k, n);
    if (wave > 0 || off == 0) return;
    u32x4_t last = nothing();
    const int i = begin + kPart - off;
    if (i + E <= V) {
      last = *at(v0 + kPart / E);
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (j < off && i + j < V) put(last, j, i + j);
    }
    if (lane == 0) held[0] = headed(held[0], last);
  }
  __device__ __forceinline__ static void wide(u32x4_t w, float (&x)[E]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (E == 4) {
        x[j] = __uint_as_float(w[j]);
      } else {
        x[2 * j] = lo_f32(w[j]);
        x[2 * j + 1] = hi_f32(w[j]);
      }
    }
  }
  // f(index of the first, logits) of the vectors [from, to) (n of two and more), one a
  // lane: the runs of 64 at from, from + 64 step, ..., those of a wave.  AHEAD loads are on
  // their way together (one takes about a microsecond where another XCD's kernel, or none,
  // has read the row before), and f stands once: a vector comes out of the registers by
  // its number.  The logits of a first or last vector that is partly outside of the row
  // come one a lane, with NaN beside each, to the wave that asks for that end.
  template <int AHEAD, class F>
  __device__ __forceinline__ void walk(int from, int to, int step, bool head, bool tail, F f) const {
    const int lane = threadIdx.x & 63;
    int edge = -1;  // its index
    if (head && off > 0 && lane < E - off) edge = lane;
    const int behind = (n - 1) * E - off + lane - 32;
    if (tail && n * E - off > V && lane >= 32 && behind < V) edge = behind;
    bool more = __ballot(edge >= 0) != 0;
    const float x0 = edge >= 0 ? one(edge) : __uint_as_float(0x7fc00000u);
    from = from < first() ? first() : from;
    to = to > end() ? end() : to;
#pragma unroll 1
    for (; from < to || more; from += 64 * step * AHEAD) {
      typedef uint32_t held_t __attribute__((ext_vector_type(4 * AHEAD)));
      held_t held = {};
      if (from < to) {
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
          const int v = from + 64 * step * k + lane;
          const u32x4_t w = *at(v < to ? v : to - 1);
#pragma unroll
          for (int j = 0; j < 4; ++j) held[4 * k + j] = w[j];
        }
      }
#pragma unroll 1
      for (int k = 0; k < AHEAD; ++k) {
        const int v = from + 64 * step * k;
        float x[E];
        int i;
        if (v < to) {
          wide(u32x4_t{held[4 * k], held[4 * k + 1], held[4 * k + 2], held[4 * k + 3]}, x);
          i = (v + lane) * E - off;
          if (v + 64 > to && v + lane >= to) wide(nothing(), x);
        } else if (more) {
          wide(nothing(), x);
          x[0] = x0;
          i = edge;
          more = false;
        } else {
          break;
        }
        f(i, x);
      }
    }
  }
  // vectors that are in the row as a whole
  __device__ __forceinline__ int first() const { return off > 0 ? 1 : 0; }
  __device__ __forceinline__ int end() const { return n * E - off > V ? n - 1 : n; }
  // A wave's part of [from, to), a run of vectors.
  template <int AHEAD = kAhead, class F>
  __device__ __forceinline__ void part(int wave, int from, int to, F f) const {
    const int per = (to - from + kWaves - 1) / kWaves, v0 = from + wave * per, v1 = v0 + per < to ? v0 + per : to;
    if (v0 < v1) walk<AHEAD>(v0, v1, 1, v0 == 0, v1 == n, f);
  }
  // The largest logit of the thread's share of the row.
  __device__ __forceinline__ float largest() const {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float m = -INFINITY;
    if (threadIdx.x < E) {  // those of a first and last vector that are partly outside
      const int i = threadIdx.x, j = (n - 1) * E - off + i;
      if (off > 0 && i < E - off) m = one(i);
      if (n * E - off > V && j < V) m = fmaxf(m, one(j));
    }
    const int last = end();
#pragma unroll 1
    for (int from = first() + 64 * wave; from < last; from += 64 * kWaves * kAhead) {
      u32x4_t w[kAhead];
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        const int v = from + 64 * kWaves * k + lane;
        w[k] = *at(v < last ? v : last - 1);
      }
#pragma unroll
      for (int k = 0; k < kAhead; ++k) {
        float x[E];
        wide(w[k], x);
        float top = x[0];
#pragma unroll
        for (int j = 1; j < E; ++j) top = fmaxf(top, x[j]);
        // (a token is one thread's alone: top-k counts threads)
        m = fmaxf(m, from + 64 * kWaves * k + lane < last ? top : -INFINITY);
      }
    }
    return m;
  }
  // f(index, logit, lanes) for each logit of a vector of the thread's share that lies in
  // [from, to] on some lanes.  (Two instructions a logit where none does.)
  template <class F>
  __device__ __forceinline__ void between(float from, float to, F f) const {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), last = end();
    if (wave == 0) {  // of a first and last vector that are partly outside, one a lane
      int edge = -1;
      if (off > 0 && lane < E - off) edge = lane;
      const int behind = (n - 1) * E - off + lane - 32;
      if (n * E - off > V && lane >= 32 && behind < V) edge = behind;
      const float x = edge >= 0 ? one(edge) : __uint_as_float(0x7fc00000u);
      const uint64_t hits = __ballot(x >= from && x <= to);
      if (hits) f(edge, x, hits);
    }
    constexpr int kSome = 4;  // and as many on their way behind them
    u32x4_t w[kSome], next[kSome];
    auto fetch = [&](int from) {
#pragma unroll
      for (int k = 0; k < kSome; ++k) {
        const int v = from + 64 * kWaves * k + lane;
        next[k] = __builtin_nontemporal_load(at(v < last ? v : last - 1));
      }
    };
    int v0 = first() + 64 * wave;
    if (v0 < last) fetch(v0);
#pragma unroll 1
    for (; v0 < last; v0 += 64 * kWaves * kSome) {
#pragma unroll
      for (int k = 0; k < kSome; ++k) w[k] = next[k];
      if (v0 + 64 * kWaves * kSome < last) fetch(v0 + 64 * kWaves * kSome);
#pragma unroll
      for (int k = 0; k < kSome; ++k) {
        const int v = v0 + 64 * kWaves * k + lane;
        if (v0 + 64 * kWaves * k >= last) break;
        float x[E];
        wide(w[k], x);
        const uint64_t in = __ballot(v < last);
        uint64_t hits[E], any = 0;
#pragma unroll
        for (int j = 0; j < E; ++j) {
          hits[j] = __ballot(__builtin_amdgcn_fmed3f(x[j], from, to) == x[j]) & in;
          any |= hits[j];
        }
        if (any)
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (hits[j]) f(v * E - off + j, x[j], hits[j]);
      }
    }
  }
};

// v of the lane that DPP control C names, 0 where there is none or MASK leaves the
// row of 16 out.
template <int C, int MASK>
__device__ __forceinline__ uint32_t moved(uint32_t v) {
  return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(v), C, MASK, 0xf, false));
}
template <int C, int MASK>
__device__ __forceinline__ uint64_t moved(uint64_t v) {
  return static_cast<uint64_t>(moved<C, MASK>(static_cast<uint32_t>(v >> 32))) << 32 |
         moved<C, MASK>(static_cast<uint32_t>(v));
}
// Sums over this lane and those before it: within rows of 16, then the rows.
template <class N>
__device__ __forceinline__ N wave_scan(N v) {
  v += moved<0x111, 0xf>(v);
  v += moved<0x112, 0xf>(v);
  v += moved<0x114, 0xf>(v);
  v += moved<0x118, 0xf>(v);
  v += moved<0x142, 0xa>(v);
  v += moved<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t last_lane(uint32_t v) { return __builtin_amdgcn_readlane(v, 63); }
__device__ __forceinline__ uint64_t last_lane(uint64_t v) {
  return static_cast<uint64_t>(last_lane(static_cast<uint32_t>(v >> 32))) << 32 | last_lane(static_cast<uint32_t>(v));
}
__device__ __forceinline__ uint64_t lane_of(uint64_t v, int lane) {
  return static_cast<uint64_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v >> 32), lane)) << 32 |
         static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<uint32_t>(v), lane));
}
template <class N>
__device__ __forceinline__ N wave_sum(N v) {
  return last_lane(wave_scan(v));
}
template <class N, class Op>
__device__ __forceinline__ N wave_all(N v, Op op) {
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) v = op(v, __shfl_xor(v, w));
  return v;
}

// WHAT a kernel's rows are: any; each its own list; each drawn from its whole
// distribution.
enum { kAnyRow, kListRow, kWholeRow };
template <int WHAT> struct Shared {
  static constexpr int kListed = WHAT == kWholeRow ? 1 : WHAT == kListRow ? kOwnList : kList;
  static constexpr int kParts = WHAT == kListRow ? 1 : kMostParts;
  double tab[128];
  union {
    unsigned long long list[kListed];  // key << 32 | index
    unsigned long long steps[WHAT == kAnyRow ? 2 : 1][kCoarse];  // of the row's parts, half of them each
  };
  unsigned long long weight[kListed];  // of the list's tokens
  static constexpr int kMass = WHAT == kListRow ? kSteps : kBins;
  uint32_t count[kSteps + 64];
  unsigned long long mass[kMass + 64];
  float part_max[kParts];
  float under[kParts];  // octaves of a part's R under the row's; 1e9: it weighs nothing
  unsigned long long kept[kParts];  // of each part, in its units
  unsigned long long few_rank[kFew], few_mass[kFew], few_run[kFew];
  unsigned long long wave_m[16];
  float wave_max[16];
  // a crossing: the bin (-1: none), what lies before it and in it
  int bin, part;
  uint32_t in_n, few, first;
  unsigned long long before, rank, at;
  unsigned long long total;
  float guess;
};

// Every wave's number, on all lanes: each of the first NT / 64 lanes its own.
template <int NT, class S>
__device__ __forceinline__ uint64_t of_waves(S& s, uint64_t v) {
  if ((threadIdx.x & 63) == 0) s.wave_m[threadIdx.x >> 6] = v;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  v = lane < NT / 64 ? s.wave_m[lane] : 0;
  __syncthreads();
  return v;
}
template <int NT, class S>
__device__ __forceinline__ uint64_t block_sum(S& s, uint64_t v) {
  return wave_sum(of_waves<NT>(s, wave_sum(v)));
}

// The first step at which s.count's running sum reaches target.
template <int NT, class S>
__device__ __forceinline__ void crossing(S& s, uint32_t target) {
  static_assert(NT == kSteps);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t c = s.count[threadIdx.x];
  uint32_t run = wave_scan(c);
  if (threadIdx.x == 0) s.bin = -1;
  const uint32_t waves = wave_scan(static_cast<uint32_t>(of_waves<NT>(s, last_lane(run))));
  run += (wave > 0 ? __builtin_amdgcn_readlane(waves, wave > 0 ? wave - 1 : 0) : 0) - c;
  if (run < target && run + c >= target) {
    s.bin = threadIdx.x;
    s.before = run;
  }
  __syncthreads();
}

// Among candidates of different ranks (of `bits` bits), the one at which the running
// mass, the largest rank first, reaches target >= 1; there must be one.  each(f) calls
// f(rank, mass) for every candidate of this thread, of which there are no more than n.
// A pass takes a digit; where no more than 64 candidates share the digits up to the
// border's, one wave compares each with each.  With `coarse` (COARSE: it may be) the first
// pass goes by step_of(rank), which orders as the ranks do: the first digit of logits of a few octaves
// has a few values, and atomics on few bins wait for each other (64 rows of 1 000 by
// top-p 11.8 us without, 10.9 with; of 2 000 15.8 and 14.0).
template <int NT, bool COARSE, class S, class Each, class Step>
__device__ __forceinline__ uint64_t select(S& s, int bits, uint64_t target, uint32_t n, bool coarse, Step step_of, Each each) {
  const int lane = threadIdx.x & 63;
  uint64_t rank = 0, before = 0;
  int left = bits, step = -1;
  auto clear = [&](int bins) {
    for (int i = threadIdx.x; i < bins + 64; i += NT) {
      s.count[i] = 0;
      s.mass[i] = 0;
    }
  };
  // the bin in which the target falls, by wave 0: a lane a run of kEach
  auto cross = [&](auto each_of, auto place) {
    constexpr int kEach = decltype(each_of)::value;
    if (threadIdx.x < 64) {
      uint64_t m[kEach], sum = 0;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        m[k] = s.mass[place(lane * kEach + k)];
        sum += m[k];
      }
      uint64_t run = before + wave_scan(sum) - sum;
#pragma unroll
      for (int k = 0; k < kEach; ++k) {
        if (run < target && run + m[k] >= target) {
          s.bin = lane * kEach + k;
          s.before = run;
          s.in_n = s.count[place(lane * kEach + k)];
        }
        run += m[k];
      }
    }
    __syncthreads();
    before = s.before;
    n = s.in_n;
  };
  if (COARSE && coarse && n > 64) {
    auto place = [](int i) { return i + i / (kSteps / 64); };
    clear(kSteps);
    __syncthreads();
    each([&](uint64_t r, uint64_t m) {
      const int bin = place(step_of(r));
      atomicAdd(&s.count[bin], 1u);
      atomicAdd(&s.mass[bin], static_cast<unsigned long long>(m));
    });
    __syncthreads();
    cross(std::integral_constant<int, kSteps / 64>{}, place);
    step = s.bin;
  }
  constexpr int kEach = kBins / 64;
  auto place = [](int i) { return i + i / kEach; };  // (a lane's run of bins, over all banks)
#pragma unroll 1
  for (;;) {
    if (threadIdx.x == 0) s.few = 0;
    if (threadIdx.x < 64) s.few_run[threadIdx.x] = 0;
    if (n <= 64) {
      __syncthreads();
      each([&](uint64_t r, uint64_t m) {
        if ((left < 64 && r >> left != rank) || (COARSE && step >= 0 && step_of(r) != step)) return;
        const uint32_t at = atomicAdd(&s.few, 1u);
        s.few_rank[at] = r;
        s.few_mass[at] = m;
      });
      __syncthreads();
      // a lane for each, a wave for some of those that it is compared with
      const int c = static_cast<int>(s.few), wave = threadIdx.x >> 6;
      const uint64_t r = s.few_rank[lane], m = s.few_mass[lane];  // (garbage behind the last)
      uint64_t run = 0;
#pragma unroll 2
      for (int j = wave; j < c; j += NT / 64) run += s.few_rank[j] > r ? s.few_mass[j] : 0;
      if (lane < c && run) atomicAdd(&s.few_run[lane], static_cast<unsigned long long>(run));
      __syncthreads();
      if (threadIdx.x < 64) {
        run = before + s.few_run[lane];
        if (lane < c && run < target && run + m >= target) s.rank = r;
      }
      __syncthreads();
      return s.rank;
    }
    const int d = left < kDigit ? left : kDigit, shift = left - d, last = (1 << d) - 1;
    clear(kBins);
    __syncthreads();
    each([&](uint64_t r, uint64_t m) {
      if (r >> left != rank || (COARSE && step >= 0 && step_of(r) != step)) return;
      const int bin = place(last - static_cast<int>(static_cast<uint32_t>(r >> shift) & static_cast<uint32_t>(last)));
      atomicAdd(&s.count[bin], 1u);
      atomicAdd(&s.mass[bin], static_cast<unsigned long long>(m));
    });
    __syncthreads();
    cross(std::integral_constant<int, kEach>{}, place);
    rank = rank << d | static_cast<uint32_t>(last - s.bin);
    left = shift;
    if (left == 0) return rank;
  }
}

__device__ __forceinline__ int first_of(uint64_t lanes) { return __builtin_ctzll(lanes); }
__device__ __forceinline__ int bits_of(uint32_t most) { return most == 0 ? 1 : 32 - __clz(most); }

// A first part of the order: tokens of larger keys, and those of this key up to an
// index.
struct Cut {
  uint32_t key, index;
  __device__ __forceinline__ bool keeps(uint32_t k, uint32_t i) const { return k > key || (k == key && i <= index); }
};

// The largest logit and the sum of weights of a row's part of kPart logits, and, for
// top-p, its sums by steps.  A lane holds its 32 logits in registers.  Bound by the
// memory for whole rows of float32 (512 rows of 100 003: 48.7 us, 4.2 TB/s), by the ten
// operations in 64 bits of a weight, as many others and an LDS atomic for top-p (192 rows
// of 131 073 bf16: 29 us, 1.7 TB/s).  256 threads, or 512 where there are too few parts to
// fill the card with those (64 rows of 32 000 by top-p: the call 29.7 and 28.3 us; 256 rows
// 47.0 and 46.3; 512 rows of 100 003 from the whole distribution 58 and 65, and 80 with
// 1 024; 192 rows of 131 073 bf16 66, 67 and 75).
template <typename T, int NT>
__global__ __launch_bounds__(NT) void sample_parts_kernel(SampleArgs a) {
  using R = Row<T, NT>;
  constexpr int E = R::E, kHeld = kPart / NT / E;  // vectors of a lane
  constexpr int kWaves = NT / 64;
  __shared__ double tab[128];
  __shared__ unsigned long long hist[kSteps], wave_sums[kWaves];
  __shared__ float wave_max[kWaves];
  const int64_t b = blockIdx.x / a.parts;
  const int part = blockIdx.x % a.parts;
  const Rules rules(a, b);
  if (!rules.by_parts()) return;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const R row(a, b);
  u32x4_t held[kHeld];
  row.share(part, held);
  fill_table(tab);
  if (rules.by_p)
    for (int i = tid; i < kSteps; i += NT) hist[i] = 0;
  float m = -INFINITY, x[E];
#pragma unroll
  for (int k = 0; k < kHeld; ++k) {
    R::wide(held[k], x);
#pragma unroll
    for (int j = 0; j < E; ++j) m = fmaxf(m, x[j]);
  }
  m = wave_all(m, [](float u, float v) { return fmaxf(u, v); });
  if (lane == 0) wave_max[wave] = m;
  __syncthreads();
  m = wave_max[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, wave_max[w]);
  const int64_t at = b * a.parts + part;
  Weights wt;
  wt.begin(rules.t, a.q, tab);
  const bool nothing = Weights::peaked(m, wt.c) || m == -INFINITY;  // (the row's draw does not ask)
  if (!nothing) wt.set(m, a.q);
  uint64_t sum = 0;
  if (!nothing) {
    if (rules.by_p) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        R::wide(held[k], x);
#pragma unroll
        for (int j = 0; j < E; ++j) {
          const uint64_t w = wt.whole(x[j]);
          if (x[j] >= wt.lowest) atomicAdd(&hist[wt.step(x[j])], static_cast<unsigned long long>(w));
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        R::wide(held[k], x);
#pragma unroll
        for (int j = 0; j < E; ++j) sum += wt.of(x[j], wt.lowest);
        __builtin_amdgcn_sched_barrier(0);
      }
      sum = wave_sum(sum);
      if (lane == 0) wave_sums[wave] = sum;
    }
  }
  if (tid == 0) a.part_max[at] = m;
  __syncthreads();
  if (rules.by_p) {
    // running sums: what a border leaves of a part is one number; a thread two of the
    // coarse steps
    uint64_t s0 = 0, s1 = 0;
    if (tid < kCoarse / 2) {
      s0 = hist[4 * tid] + hist[4 * tid + 1];
      s1 = hist[4 * tid + 2] + hist[4 * tid + 3];
    }
    uint64_t run = wave_scan(s0 + s1);
    if (lane == 63) wave_sums[wave] = run;
    __syncthreads();
    if (tid < kCoarse / 2) {
      for (int w = 0; w < wave; ++w) run += wave_sums[w];
      *reinterpret_cast<ulonglong2*>(&a.part_steps[at * kCoarse + 2 * tid]) = make_ulonglong2(run - s1, run);
    }
  } else if (tid == 0) {
    sum = 0;
    for (int w = 0; w < kWaves; ++w) sum += wave_sums[w];
    a.part_sum[at] = nothing ? 0 : sum;
  }
}

template <typename T, int NT, int WHAT>
__global__ __launch_bounds__(NT) void sample_kernel(SampleArgs a) {
  constexpr int kWaves = NT / 64;
  constexpr bool kWhole = WHAT == kListRow;
  using R = Row<T, NT>;
  constexpr int E = R::E, kShift = E == 8 ? 16 : 0;  // bits of keys that say nothing
  __shared__ Shared<WHAT> s;
  const int64_t b = blockIdx.x;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const R row(a, b);
  const Rules rules(a, b);
  const int k = rules.k;
  const bool by_k = rules.by_k, by_p = rules.by_p, by_parts = !kWhole && rules.by_parts();
  const float u = a.u[b];
  const float* part_max = a.part_max + b * a.parts;

  fill_table(s.tab);
  if (tid == 0) s.first = 0xffffffffu;
  if constexpr (WHAT == kAnyRow) s.count[tid] = 0;
  float mine = -INFINITY;  // the thread's largest
  if (by_parts) {
    for (int i = tid; i < a.parts; i += NT) {
      const float x = part_max[i];
      if (!by_p) s.kept[i] = a.part_sum[b * a.parts + i];
      s.part_max[i] = x;
      mine = fmaxf(mine, x);
    }
  } else if constexpr (kWhole) {
    for (int i = tid; i < a.V; i += NT) mine = fmaxf(mine, row.one(i));
  } else {
    mine = row.largest();
  }
  const float wm = wave_all(mine, [](float x, float y) { return fmaxf(x, y); });
  if (lane == 0) s.wave_max[wave] = wm;
  __syncthreads();
  const float m = wave_all(s.wave_max[lane % kWaves], [](float x, float y) { return fmaxf(x, y); });
  if (m == -INFINITY) {  // nothing to draw
    if (tid == 0) {
      a.token[b] = -1;
      if (a.logprob) a.logprob[b] = -INFINITY;
    }
    return;
  }
  if (rules.greedy) {  // the first of the largest
    if constexpr (kWhole) {
      for (int i = tid; i < a.V; i += NT)
        if (row.one(i) == m) atomicMin(&s.first, static_cast<uint32_t>(i));
    } else {
      row.part(wave, 0, row.n, [&](int i, const float(&x)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (x[j] == m) atomicMin(&s.first, static_cast<uint32_t>(i + j));
      });
    }
    __syncthreads();
    if (tid == 0) {
      a.token[b] = s.first;
      if (a.logprob) a.logprob[b] = 0.f;
    }
    return;
  }
  const uint32_t key_m = key_of(m), last = a.V - 1;
  const int index_bits = bits_of(last);
  Weights wt;
  wt.begin(rules.t, a.q, s.tab);
  wt.lowest = m;
  wt.R = 0;
  const bool peaked = Weights::peaked(m, wt.c);  // the largest weigh the same, all others nothing
  if (!peaked) wt.set(m, a.q);
  float floor_l = wt.lowest;  // of what can be drawn
  if (rules.least > 0.f && !peaked) {
    const double x = m + log2_of(fmax(static_cast<double>(rules.least), 0x1p-100), s.tab) * wt.per;
    floor_l = fmaxf(floor_l, -float_under(fmin(-x, 3.4028234663852886e38)));  // (the smallest float that is not below x)
  }
  // (sums are all lanes': the scalar unit takes their shares)
  auto part = [&](uint64_t total) -> uint64_t {  // what top-p's run has to reach
    return rules.p > 0.f ? share_of<true>(rules.p, lane_of(total, 0)) : 1;
  };
  auto place = [&](uint64_t total) -> uint64_t {  // of the draw in [0, total)
    total = lane_of(total, 0);
    return !(u > 0.f) ? 0 : u < 1.f ? share_of<false>(u, total) : total - 1;
  };
  // The token and the logarithm of its share: weight and total in one unit, the total
  // also in units of 2^R.
  auto done = [&](int i, float l, double weight, double total, double total_r) {
    a.token[b] = i;
    if (!a.logprob) return;
    double log2p = 0.0;
    if (weight != total)
      log2p = (peaked ? 0.0 : static_cast<double>(l) * wt.c - wt.R) - log2_of(total_r, s.tab);
    a.logprob[b] = static_cast<float>(log2p * 0.6931471805599453);
  };
  auto under_of = [&](float pm) -> float {
    if (pm == -INFINITY || Weights::peaked(pm, wt.c)) return 1e9f;
    return static_cast<float>(fmin(wt.R - ceil(static_cast<double>(pm) * wt.c), 1e9));
  };
  const uint32_t key_floor = key_of(floor_l);
  const double per_unit = peaked ? 1.0 : ldexp(1.0, -a.q);

  // -- the list: what the first border is decided on ------------------------------------
  Cut cut{0, 0xffffffffu};    // all
  bool listed = kWhole;       // all that the cut keeps are in the list
  bool first_cut = false, counts = true, from_list = true;
  int n = 0, border = -1;
  uint32_t lo = 0, hi = key_m;  // keys from here on, up to there
  uint64_t target = k;
  if constexpr (WHAT == kWholeRow) {
    from_list = false;
  } else if constexpr (kWhole) {
    n = a.V;
    for (int i = tid; i < n; i += NT) {
      const float l = row.one(i);
      s.list[i] = l >= wt.lowest ? static_cast<uint64_t>(key_of(l)) << 32 | static_cast<uint32_t>(i) : 0;
    }
    __syncthreads();
    first_cut = by_k;
  } else if (!peaked && (by_k || by_p || rules.least > 0.f)) {
    const bool by_threads = by_k && k <= NT;
    bool all = true, band = false;  // what the list may be: all from the border's step on, that step alone
    float from = floor_l, to = INFINITY;
    int wide = 2;                   // the steps are of 2^wide / 128
    uint64_t before = 0;
    if (by_k) {
      if (by_threads) {
        if (mine >= wt.lowest) atomicAdd(&s.count[wt.step(mine)], 1u);
      } else {
        row.part(wave, 0, row.n, [&](int, const float(&x)[E]) {
#pragma unroll
          for (int j = 0; j < E; ++j)
            if (x[j] >= wt.lowest) atomicAdd(&s.count[wt.step(x[j])], 1u);
        });
      }
      __syncthreads();
      crossing<NT>(s, static_cast<uint32_t>(k));
      border = s.bin;
      before = s.before;
      if (by_threads && border < 0) border = kSteps - 1;
      band = !by_threads;
      all = first_cut = border >= 0;  // (fewer than k weigh anything: k keeps them all)
    } else if (by_p) {
      // the parts' sums by steps, shifted to the row's R
      for (int p = tid; p < a.parts; p += NT) s.under[p] = under_of(s.part_max[p]);
      __syncthreads();
      // the running sums, shifted to the row's R
      constexpr int kSome = 8, kOf = NT / kCoarse;  // loads on their way together; threads of a step
      const int i = tid & (kCoarse - 1);
      uint64_t sum = 0;
#pragma unroll 1
      for (int p0 = tid / kCoarse; p0 < a.parts; p0 += kSome * kOf) {
        unsigned long long w[kSome];
        int down[kSome];
#pragma unroll
        for (int j = 0; j < kSome; ++j) {
          const int p = p0 + j * kOf < a.parts ? p0 + j * kOf : p0;
          down[j] = static_cast<int>(fminf(s.under[p], 63.f));
          // (the last step holds all that lies lower)
          const int at = i == kCoarse - 1 ? i : i - 16 * down[j];
          if (at < 0 || p0 + j * kOf >= a.parts) down[j] = 63;
          w[j] = a.part_steps[(b * a.parts + p) * kCoarse + (at < 0 ? 0 : at)];
        }
#pragma unroll
        for (int j = 0; j < kSome; ++j) sum += w[j] >> down[j];
      }
      s.steps[tid / kCoarse][i] = sum;
      __syncthreads();
      const uint64_t goal = part(s.steps[0][kCoarse - 1] + s.steps[1][kCoarse - 1]);
      if (tid < kCoarse) {
        const uint64_t here = s.steps[0][i] + s.steps[1][i], over = i > 0 ? s.steps[0][i - 1] + s.steps[1][i - 1] : 0;
        if (here >= goal && over < goal) {
          s.bin = i;
          s.before = over;
          // (about as many tokens, were they half as heavy again as the border's)
          s.guess = static_cast<float>(here) * __builtin_amdgcn_exp2f((i + 1) * 0.0625f - a.q) * 0.5f;
        }
      }
      __syncthreads();
      border = s.bin;
      before = s.before;
      wide = 3;
      counts = false;
      first_cut = true;
      band = true;
      all = s.guess <= kFew;
      target = goal;
    }
    if (border >= 0) {
      // logits of the steps up to the border's, and of the border's, with a little room
      // for roundings
      const double low = 1 << wide, first_n = low * border;  // n of its first, under 128 R
      const bool lowest_step = border == (wide == 2 ? kSteps : kCoarse) - 1;
      from = lowest_step ? wt.lowest : fmaxf(wt.lowest, float_under((wt.R - (first_n + low) * 0.0078125) * wt.per));
      to = -float_under(-(wt.R - (first_n - 1.0) * 0.0078125) * wt.per);
      if (by_p && !by_k && floor_l > to) {  // min-p leaves less than top-p: no border of its own
        from = floor_l;
        all = true;
        band = first_cut = false;
      } else if (by_p && !by_k && lowest_step) {
        // the last step's sums count what lies under the row's lowest and weighs nothing in
        // the row's units, and a list of it could be empty: the border is found on the row
        all = band = false;
      }
    }
    // gathers the tokens from `from` on (first all, then the border's step alone)
    from_list = false;
#pragma unroll 1
    for (int attempt = all ? 0 : 1; attempt < (band ? 2 : 1) && !from_list && (all || band); ++attempt) {
      const bool alone = attempt == 1;
      const float most = alone ? to : INFINITY;
      // (what is not of the step that stands alone leaves a hole)
      auto entry = [&](float l, uint32_t i) -> uint64_t {
        const bool of = !alone || (l >= wt.lowest && (wide == 2 ? wt.step(l) : wt.step(l) >> 1) == border);
        return of ? static_cast<uint64_t>(key_of(l)) << 32 | i : 0;
      };
      if (tid == 0) s.few = 0;
      __syncthreads();
      // first into places of the wave's own (in s.weight), then together
      constexpr int kSlots = kList / kWaves;
      unsigned long long* slots = s.weight + kSlots * wave;
      int mine_n = 0;
      row.between(from, most, [&](int i, float l, uint64_t mask) {
        const int before = mine_n;
        mine_n += __popcll(mask);
        if (mine_n > kSlots) return;
        if (mask >> lane & 1)
          slots[__builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(mask >> 32),
                                          __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(mask), before))] =
              static_cast<uint64_t>(__float_as_uint(l)) << 32 | static_cast<uint32_t>(i);
      });
      const uint32_t counted = static_cast<uint32_t>(of_waves<NT>(s, static_cast<uint64_t>(mine_n)));
      const uint32_t places = wave_scan(counted);
      const bool fits = !__ballot(counted > kSlots);
      n = static_cast<int>(last_lane(places));
      if (fits) {
        const int at = static_cast<int>(__builtin_amdgcn_readlane(places, wave)) - mine_n;
        for (int i = lane; i < mine_n; i += 64) {
          const uint64_t x = slots[i];
          s.list[at + i] = entry(__uint_as_float(static_cast<uint32_t>(x >> 32)), static_cast<uint32_t>(x));
        }
      } else if (by_parts && n <= kList) {
        // Which wave meets a token goes by the row's address; whether there is a list must
        // not: top-p sums a list in the row's units and other tokens in their parts'.
        for (int i = tid; i < a.V; i += NT) {
          const float l = row.one(i);
          if (l >= from && l <= most) s.list[atomicAdd(&s.few, 1u)] = entry(l, static_cast<uint32_t>(i));
        }
      } else {
        n = kList + 1;
      }
      __syncthreads();
      if (n <= kList) {
        from_list = true;
        listed = !alone;
        if (alone) target -= before;
        lo = first_cut ? key_of(from) : 0;
        hi = first_cut && alone && key_of(to) < hi ? key_of(to) : hi;
      }
    }
  }

  if constexpr (WHAT != kWholeRow) {
    if (kWhole || from_list) {  // weights, for every look at the list
      for (int i = tid; i < n; i += NT) {
        const float l = of_key(static_cast<uint32_t>(s.list[i] >> 32));
        s.weight[i] = peaked ? l >= wt.lowest : wt.of(l, wt.lowest);
      }
    }
    // f(key, index, weight) of the list's tokens, or the row's, of the cut, from lo on
    auto each = [&](bool in_list, auto f) {
      if (kWhole || in_list) {
#pragma unroll 1
        for (int i = tid; i < n; i += NT) {  // (a thread's own)
          const uint64_t x = s.list[i];
          const uint32_t ky = static_cast<uint32_t>(x >> 32), at = static_cast<uint32_t>(x);
          if (ky != 0 && ky >= lo && cut.keeps(ky, at)) f(ky, at, s.weight[i]);
        }
      } else if constexpr (!kWhole) {  // (four loads ahead: with eight registers spill)
        row.template part<4>(wave, 0, row.n, [&](int i, const float(&x)[E]) {
#pragma unroll 1
          for (int j = 0; j < E; ++j) {
            float l = x[0];
#pragma unroll
            for (int c = 1; c < E; ++c) l = j == c ? x[c] : l;
            const uint32_t ky = key_of(l), at = static_cast<uint32_t>(i + j);
            if (l >= wt.lowest && ky >= lo && cut.keeps(ky, at)) f(ky, at, peaked ? 1 : wt.whole(l));
          }
        });
      }
    };
    // Few tokens: each is compared with each, a lane for each and a pair of waves for some
    // of those that it is compared with; once in the order, once by index.
    if (listed && n <= kFew) {
      if (tid < kFew) s.few_rank[tid] = s.few_run[tid] = s.mass[tid] = 0;
      __syncthreads();
      constexpr int kOf = NT / kFew;
      const int e = tid & (kFew - 1), slice = tid / kFew;
      const uint64_t x = e < n ? s.list[e] : 0, place_of = x ^ 0xffffffffu;
      uint64_t rank = 0, before = 0;
#pragma unroll 2
      for (int j = slice; j < n; j += kOf) {
        const bool over = (s.list[j] ^ 0xffffffffu) > place_of;
        rank += over;
        before += over ? s.weight[j] : 0;
      }
      if (rank) {
        atomicAdd(&s.few_rank[e], static_cast<unsigned long long>(rank));
        atomicAdd(&s.few_run[e], static_cast<unsigned long long>(before));
      }
      __syncthreads();
      uint64_t total = 0;
      if (wave == 0) {
        constexpr int kEach = kFew / 64;
        uint64_t w[kEach], sum = 0;
#pragma unroll
        for (int h = 0; h < kEach; ++h) {
          const int i = lane + 64 * h;
          w[h] = i < n && (!by_k || s.few_rank[i] < static_cast<uint64_t>(k)) ? s.weight[i] : 0;
          sum += w[h];
        }
        if (by_p && !by_parts) target = part(wave_sum(sum));
        sum = 0;
#pragma unroll
        for (int h = 0; h < kEach; ++h) {
          const int i = lane + 64 * h;
          if (by_p && s.few_run[i] >= target) w[h] = 0;
          if (static_cast<uint32_t>(s.list[i] >> 32) < key_floor) w[h] = 0;
          s.few_mass[i] = w[h];
          sum += w[h];
        }
        total = wave_sum(sum);
        if (lane == 0) s.total = total;
      }
      __syncthreads();
      const uint32_t index = static_cast<uint32_t>(x);
      before = 0;
#pragma unroll 2
      for (int j = slice; j < n; j += kOf) before += static_cast<uint32_t>(s.list[j]) < index ? s.few_mass[j] : 0;
      if (before) atomicAdd(&s.mass[e], static_cast<unsigned long long>(before));
      __syncthreads();
      if (tid < kFew) {
        total = s.total;
        const uint64_t at = place(total), own = s.few_mass[e];
        before = s.mass[e];
        if (e < n && before <= at && at < before + own)
          done(index, of_key(static_cast<uint32_t>(x >> 32)), static_cast<double>(own), static_cast<double>(total),
               static_cast<double>(total) * per_unit);
      }
      return;
    }
    // Three selects, each on what the one before left: top-k's or top-p's border, top-p's
    // behind top-k's, the draw (of a list; a row's has walks of its own below).
#pragma unroll 1
    for (int stage = 0; stage < 3; ++stage) {
      const bool draw = stage == 2;
      bool ones = false, in_list = listed;
      if (stage == 0) {
        if (!first_cut) continue;
        ones = counts;
        in_list = from_list;
      } else if (stage == 1 ? !by_p || by_parts || (peaked && !kWhole) : !listed) {
        continue;
      }
      if (stage > 0) lo = cut.key > lo ? cut.key : lo;
      if (draw) lo = key_floor > lo ? key_floor : lo;
      uint64_t total = 0;
      each(in_list, [&](uint32_t, uint32_t, uint64_t w) { total += ones ? 1 : w; });
      total = block_sum<NT>(s, total);
      if (stage == 0) {
        if (counts && target >= total && in_list == listed) continue;  // k keeps them all
        if (!counts && !in_list) target = part(total);  // (top-p on the row: all in its units)
        target = target < total ? target : total;       // (a border's step, by roundings)
      } else {
        target = draw ? place(total) + 1 : part(total);
      }
      const uint32_t lowest = lo >> kShift;
      const int bits = draw ? index_bits : bits_of((hi >> kShift) - lowest) + index_bits;
      auto step_of = [&](uint64_t r) { return wt.step(of_key((lowest + static_cast<uint32_t>(r >> index_bits)) << kShift)); };
      const uint64_t r = select<NT, kWhole>(s, bits, target, in_list ? n : a.V, !draw && !peaked, step_of, [&](auto g) {
        each(in_list, [&](uint32_t ky, uint32_t i, uint64_t w) {
          if (ones) w = 1;
          if (w) g(static_cast<uint64_t>(draw ? 0 : (ky >> kShift) - lowest) << index_bits | (last - i), w);
        });
      });
      const uint32_t at = last - (static_cast<uint32_t>(r) & ((1u << index_bits) - 1));
      if (!draw) {
        uint32_t ky = (lowest + static_cast<uint32_t>(r >> index_bits)) << kShift;
        if (kShift > 0 && !(ky & 0x80000000u)) ky |= (1u << kShift) - 1;  // (a negative number's)
        cut = Cut{ky, at};
        hi = key_m;
      } else if (tid == 0) {
        const float l = row.one(at);
        done(at, l, static_cast<double>(peaked ? 1 : wt.whole(l)), static_cast<double>(total),
             static_cast<double>(total) * per_unit);
      }
    }
  }
  if constexpr (!kWhole) {
    if (listed) return;
    const float key_l = cut.key ? of_key(cut.key) : -INFINITY;
    const uint32_t to = cut.index;
    int begin = 0, v0 = 0, v1 = row.n;  // of a part: its first logit, and its vectors
    uint64_t at = 0;
    double total = 0.0, total_r = 0.0;
    bool need_total = true;
    if (by_parts && !peaked && (by_p ? from_list && floor_l <= key_l : rules.least == 0.f)) {
      // The parts' sums of what is kept: of top-p the steps before the border's, and of
      // its step what the cut keeps.
      __syncthreads();
      if (WHAT == kAnyRow && by_p) {
        for (int p = tid; p < a.parts; p += NT) {
          const int end = border - 16 * static_cast<int>(fminf(s.under[p], 63.f));
          s.kept[p] = end > 0 ? a.part_steps[(b * a.parts + p) * kCoarse + end - 1] : 0;
        }
        __syncthreads();
        for (int i = tid; i < n; i += NT) {
          const uint64_t x = s.list[i];
          const uint32_t ky = static_cast<uint32_t>(x >> 32), index = static_cast<uint32_t>(x);
          if (ky == 0 || !cut.keeps(ky, index)) continue;
          const int p = static_cast<int>(index) / kPart;
          Weights w = wt;
          w.set(s.part_max[p], a.q);
          atomicAdd(&s.kept[p], static_cast<unsigned long long>(w.of(of_key(ky), w.lowest)));
        }
        __syncthreads();
      }
      if (wave == 0) {
        int under = 0;
        auto kept_of = [&](int p) -> uint64_t {  // in the row's units
          const uint64_t x = p < a.parts ? s.kept[p] : 0;
          under = x ? static_cast<int>(fminf(under_of(s.part_max[p]), 63.f)) : 0;
          return x >> under;
        };
        uint64_t sum = 0;
        for (int p0 = 0; p0 < a.parts; p0 += 64) sum += wave_sum(kept_of(p0 + lane));
        uint64_t place_in = place(sum);
#pragma unroll 1
        for (int p0 = 0; p0 < a.parts; p0 += 64) {
          const uint64_t v = kept_of(p0 + lane), to_here = wave_scan(v);
          const uint64_t over = __ballot(to_here > place_in);
          if (over) {
            if (lane == first_of(over)) {
              s.part = p0 + lane;
              s.at = (place_in - (to_here - v)) << under;  // (the first of the part's units that are this one of the row's)
            }
            break;
          }
          place_in -= last_lane(to_here);
        }
        if (lane == 0) s.total = sum;
      }
      __syncthreads();
      at = s.at;
      total = static_cast<double>(s.total);
      total_r = total * per_unit;
      begin = s.part * kPart;
      v0 = begin / E;
      v1 = v0 + kPart / E < row.n ? v0 + kPart / E : row.n;
      need_total = false;
    }
    // The draw: every wave sums what its part of the row keeps, then of the part in
    // which the draw lies, until one step of a wave holds the rest.
    Weights w = wt;  // in the units of the row, or of its part
    const bool by_part = !need_total;
    if (by_part) w.set(s.part_max[s.part], a.q);
    // (the part's sum counts what weighs something in the part's units, under the row's
    // lowest too: a draw that falls into its part finds a token there.  Of top-p the cut lies
    // above the row's lowest and min-p's.)
    const float low = fmaxf(by_part ? key_l : fmaxf(floor_l, key_l), w.lowest);
    auto weight = [&](float l, int i) -> uint64_t {
      uint64_t x = w.whole(l);
      if (peaked) x = 1;
      return l >= low && (l != key_l || static_cast<uint32_t>(i) <= to) ? x : 0;
    };
    // the wave in whose part the draw lies, with the draw's place there
    auto pick = [&](uint64_t sum) -> int {
      const uint64_t sums = of_waves<NT>(s, wave_sum(sum)), run = wave_scan(sums);
      if (need_total) {
        uint64_t kept = last_lane(run);
        if (peaked) {  // (top-k and top-p count, and the first ones by index are kept)
          if (by_k && k < static_cast<int64_t>(kept)) kept = k;
          if (by_p) kept = part(kept);
        }
        at = place(kept);
        total = static_cast<double>(kept);
        total_r = total * per_unit;
        need_total = false;
      }
      const int w = first_of(__ballot(run > at) | 1ull << 63) & (kWaves - 1);  // (there is one)
      at -= lane_of(run, w) - lane_of(sums, w);
      return w;
    };
    constexpr int kFewer = E == 8 ? 4 : 8;  // loads ahead (eight of bf16: registers spill)
    constexpr int kHeld = kPart / E / NT, kMost = kHeld * NT;  // vectors of a lane, of a workgroup
#pragma unroll 1
    while (v1 - v0 > kMost) {
      const int per = (v1 - v0 + kWaves - 1) / kWaves;
      uint64_t sum = 0;
      row.template part<kFewer>(wave, v0, v1, [&](int i, const float(&x)[E]) {
#pragma unroll
        for (int j = 0; j < E; ++j) sum += weight(x[j], i + j);
      });
      v0 += pick(sum) * per;
      v1 = v0 + per < v1 ? v0 + per : v1;
    }
    uint64_t of[kHeld], sum = 0;
    u32x4_t held[kHeld];
    const int mine0 = v0 + wave * 64 * kHeld;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) held[h] = row.raw(mine0 + 64 * h, v1);
    // (a part that begins inside of a vector: that vector's first logits are of the part
    // before, and as many of its own lie behind its vectors, one a lane of the last wave)
    const int behind = begin + kPart - row.off + lane;
    const bool ends = by_part && row.off > 0 && wave == kWaves - 1;
    const float x_behind = ends && lane < row.off && behind < a.V ? row.one(behind) : __uint_as_float(0x7fc00000u);
    if (wave == 0 && begin > 0 && lane == 0) held[0] = row.headed(held[0], R::nothing());
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      float x[E];
      R::wide(held[h], x);
      of[h] = 0;
#pragma unroll
      for (int j = 0; j < E; ++j) of[h] += weight(x[j], (mine0 + 64 * h + lane) * E - row.off + j);
      sum += of[h];
    }
    if (ends) sum += weight(x_behind, behind);
    if (pick(sum) != wave) return;
    // of the wave's vectors that with the draw, and the lane's place in front of it
    uint64_t run = 0, before = 0, in = 0;
    u32x4_t it = held[0];
    int i = 0;
    bool found = false;
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
      const uint64_t to_here = run + wave_scan(of[h]), all = last_lane(to_here);
      if (!found && all > at) {
        found = true;
        it = held[h];
        i = (mine0 + 64 * h + lane) * E - row.off;
        before = to_here - of[h];
        in = of[h];
      }
      run = all;
    }
    if (!found && ends) {  // one of those behind
      found = true;
      it = R::nothing();
      it[0] = E == 8 ? __float_as_uint(x_behind) >> 16 | 0x7fc00000u : __float_as_uint(x_behind);
      i = behind;
      in = weight(x_behind, behind);
      before = run + wave_scan(in) - in;
    }
    if (found && before <= at && at < before + in) {
#pragma unroll 1
      for (int j = 0; j < E; ++j) {  // (once in the code: one lane's few logits)
        const int d = j / (E / 4);
        uint32_t bits = d < 2 ? (d == 0 ? it[0] : it[1]) : d == 2 ? it[2] : it[3];
        if (E == 8) bits = j & 1 ? bits & 0xffff0000u : bits << 16;
        const float l = __uint_as_float(bits);
        const uint64_t y = weight(l, i + j);
        if (before <= at && at < before + y)
          done(i + j, l, ldexp(static_cast<double>(y), w.R - wt.R), total, total_r);
        before += y;
      }
    }
  }
}

// Whether rows are their own lists.  Top-k's threshold makes short lists of longer rows:
// 64 rows of 300 | 1 000 | 2 000 float32 take 8.3 | 10.6 | 13.5 us by top-k as their own
// lists and 9.0 | 8.8 | 9.2 by a threshold (512 rows of 1 000: 12.7 and 16.7), by top-p
// 8.3 | 10.7 | 13.9 and, of parts, 21 | 25 | 25.  A list of 4 096 leaves room for one
// workgroup a CU.
bool own_list(const srw_sample_t& d) { return d.V <= (d.top_k || d.top_k_all > 0 ? kOwnList / 2 : kOwnList); }
// Parts of a row (0: it is its own list).
int64_t parts_of(const srw_sample_t& d) { return own_list(d) ? 0 : (d.V + kPart - 1) / kPart; }
// Whether a row may ask for its parts' sums.
bool by_parts(const srw_sample_t& d) {
  if (own_list(d)) return false;
  if (!d.temperature && !(d.temperature_all > 0.f)) return false;
  const bool by_p = d.top_p || d.top_p_all < 1.f, whole = d.min_p || d.min_p_all == 0.f;
  return (d.top_k || d.top_k_all == 0 || d.top_k_all >= d.V) && (by_p || whole);
}
// Whether no row can do otherwise, and for its sums alone.
bool only_whole(const srw_sample_t& d) {
  return by_parts(d) && !d.temperature && !d.top_k && !d.top_p && d.top_p_all >= 1.f && !d.min_p && d.min_p_all == 0.f;
}
struct Workspace {
  size_t max, sum, steps, bytes;  // offsets, and the whole
};
Workspace workspace_of(const srw_sample_t& d) {
  Workspace w{};
  if (!by_parts(d)) return w;
  const size_t n = static_cast<size_t>(d.B) * parts_of(d);
  const bool by_p = d.top_p || d.top_p_all < 1.f;
  w.sum = (n * 4 + 255) & ~size_t{255};
  w.steps = (w.sum + n * 8 + 255) & ~size_t{255};
  w.bytes = w.steps + (by_p ? n * kCoarse * 8 : 0);
  return w;
}

srw_status_t check_sample(const srw_sample_t* d) {
  if (!d) return SRW_EINVAL;
  if (d->B < 0 || d->V < 1 || (d->dtype != SRW_F32 && d->dtype != SRW_BF16)) return SRW_EINVAL;
  if (d->B > (1 << 21) || d->V > (1 << 24)) return SRW_EUNSUPPORTED;  // (a launch has under 2^32 threads)
  if (d->B == 0) return SRW_OK;
  if (d->B * parts_of(*d) >= (1 << 24)) return SRW_EUNSUPPORTED;
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

extern "C" {

srw_status_t srw_sample_workspace_size(const srw_sample_t* d, size_t* bytes) {
  const srw_status_t st = srw::check_sample(d);
  if (st != SRW_OK) return st;
  if (!bytes) return SRW_EINVAL;
  *bytes = d->B == 0 ? 0 : srw::workspace_of(*d).bytes;
  return SRW_OK;
}

srw_status_t srw_sample(const srw_sample_t* d, void* workspace, size_t workspace_bytes, void* stream) {
  const srw_status_t st = srw::check_sample(d);
  if (st != SRW_OK || d->B == 0) return st;
  const srw::Workspace w = srw::workspace_of(*d);
  if (w.bytes > 0 && (!workspace || reinterpret_cast<uintptr_t>(workspace) % 16 || workspace_bytes < w.bytes))
    return SRW_EWORKSPACE;
  srw::SampleArgs a{};
  a.logits = static_cast<const char*>(d->logits);
  a.stride = d->B > 1 ? d->row_stride : 0;
  a.V = static_cast<int32_t>(d->V);
  int bits = 0;  // V <= 2^bits
  while ((int64_t{1} << bits) < d->V) ++bits;
  a.q = 62 - bits < 51 ? 62 - bits : 51;
  a.parts = static_cast<int32_t>(srw::parts_of(*d));
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
  char* ws = static_cast<char*>(workspace);
  a.part_max = reinterpret_cast<float*>(ws + w.max);
  a.part_sum = reinterpret_cast<unsigned long long*>(ws + w.sum);
  a.part_steps = reinterpret_cast<unsigned long long*>(ws + w.steps);
  (void)hipGetLastError();
  const dim3 grid(static_cast<unsigned>(d->B)), parts(static_cast<unsigned>(d->B * a.parts));
  const hipStream_t s = static_cast<hipStream_t>(stream);
  auto launch = [&](auto logit) {
    using T = decltype(logit);
    if (w.bytes > 0 && parts.x <= 512)
      hipLaunchKernelGGL((srw::sample_parts_kernel<T, 512>), parts, dim3(512), 0, s, a);
    else if (w.bytes > 0)
      hipLaunchKernelGGL((srw::sample_parts_kernel<T, 256>), parts, dim3(256), 0, s, a);
    if (srw::own_list(*d))
      hipLaunchKernelGGL((srw::sample_kernel<T, 512, srw::kListRow>), grid, dim3(512), 0, s, a);
    else if (srw::only_whole(*d))
      hipLaunchKernelGGL((srw::sample_kernel<T, 256, srw::kWholeRow>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((srw::sample_kernel<T, 1024, srw::kAnyRow>), grid, dim3(1024), 0, s, a);
  };
  if (d->dtype == SRW_F32)
    launch(float{});
  else
    launch(uint16_t{});
  return hipGetLastError() == hipSuccess ? SRW_OK : SRW_EHIP;
}

}  // extern "C"

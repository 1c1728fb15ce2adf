// srw_attn.hip -- attention of new tokens over the paged key/value cache.
//
//   out[t] = sum_j p[t,j] v[j],  p = softmax_j(scale q[t] . k[j])
//   over the positions j that the token at position i sees:
//   j <= i, and with a window j > i - window or j < sinks.
//
// Both kernels walk a sequence's visible positions in tiles of 64 with a
// running maximum m and sum l (scores in units of log2): S^T = K Q^T, p =
// 2^(s - m), O^T += V^T P^T.  Tokens lie along a matrix product's columns, so
// a token's maximum, sum and rescaling are numbers of its own lanes, and the
// score accumulators are, rounded to bf16, the second product's operand as
// they stand: which key a row of the first product holds is chosen so that
// the eight k-slots of a lane are consecutive positions of the value page.
// All heads of a group share one pass over their key head's pages.
//
// 8-bit pages: the codes are bf16 numbers exactly, so both products run on the
// codes.  A key's scale multiplies its score, a value's scale goes into the
// exponent,
//   w[j] = 2^(s[j] + log2 vs[j] - m),  l = sum_j w[j] / vs[j],
// so that m follows the weights that the second product reads.  (A weight under
// 2^-126 is lost to l: one of a key whose value scale is 2^-d times that of the
// key that m follows, and which so weighs less than 2^(d - 126) of it.)
//
// The matrix cores read weights in bf16.  The kernel for few rows, bound by
// memory, gives them in two parts (bf16 of w and of what is left, 16 bits in
// all), the one for many rows rounds them once; everything else is float32.
//
// m is raised only when an exponent passes it by more than 8: weights then stay
// under 2^8 and their sum far inside float32, and the accumulators are rescaled
// a few times a row instead of once a tile.
//
// What a token must not see is left out by selects, not by adding numbers;
// positions without a page (a table entry that names none, as for positions
// that a window has left behind) are not seen, and value bytes that no token
// of a tile sees are cleared before the product, since 0 x NaN is NaN.  A token
// that sees nothing gets zeros.
//
// Scores beyond +-4096, whose last bits are no longer small beside 1, and values
// that are not finite are rare, and the loops carry nothing for them: a wave that
// ends with either goes over its tiles again (careful_rows).

#include <float.h>
#include <math.h>

#include "srw_kv.hpp"

namespace srw {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr float kLazy = 8.f;       // log2 of the largest weight before m is raised
constexpr float kLowest = -FLT_MAX;  // m of a row that has seen nothing, or scores of -inf only
constexpr float kLarge = 4096.f;      // an m whose last bit, 2^-11, moves a weight by under 2e-4

struct AttnArgs {
  KvView kv;
  const uint16_t* q;
  uint16_t* out;
  float* part;    // [S][T Hq][DH]: unnormalised partial outputs
  float2* ml;     // [S][T Hq]: (m, l)
  int64_t q_token, q_head;
  int Hq, G, window, sinks;
  float sc;       // scale log2 e
  int S, least;   // splits of a row tile's key tiles, of so many at least
};

__device__ inline KvSpan span_of(const AttnArgs& a, int p_lo, int p_hi) {
  return kv_span(a.kv.cap, a.window, a.sinks, p_lo, p_hi);
}

// Tiles of a split, of the row tile's own number: a table far wider than a
// sequence leaves no long split behind.
__device__ inline int per_split(const AttnArgs& a, int tiles) {
  const int per = (tiles + a.S - 1) / a.S;
  return per > a.least ? per : a.least;
}

// The sequence and the tile of R rows (token, head of the group) of workgroup
// `at`.  start(b) = cu[b] G / R + b leaves room for a last, partial tile; a
// sequence's last tiles, which see most, come first.
struct Tile {
  int64_t b;
  KvSeq sq;
  int r0, r1;  // r0 = -1: none
};
template <int R>
__device__ inline Tile tile_of(const AttnArgs& a, int64_t at) {
  Tile t;
  int64_t rt;
  if (a.kv.cu) {
    auto start = [&](int64_t i) { return static_cast<int64_t>(a.kv.cu[i]) * a.G / R + i; };
    t.b = kv_find(a.kv.B, at, start);
    rt = at - start(t.b);
  } else {
    const int per = (a.G + R - 1) / R;
    t.b = at / per;
    rt = at % per;
  }
  t.b = __builtin_amdgcn_readfirstlane(static_cast<int>(t.b));
  t.sq = kv_seq(a.kv, t.b);
  const int rows = t.sq.n * a.G, rts = (rows + R - 1) / R;
  t.r0 = rt < 0 || rt >= rts ? -1 : (rts - 1 - static_cast<int>(rt)) * R;
  t.r1 = t.r0 + R < rows ? t.r0 + R : rows;
  return t;
}

__device__ inline f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}
// All ones where bit n of w is set, else zero; v there, else -inf.
template <int N>
__device__ inline uint32_t bit_mask(uint32_t w) {
  return static_cast<uint32_t>(__builtin_amdgcn_sbfe(static_cast<int>(w), N, 1));
}
template <int N>
__device__ inline float only(uint32_t w, float v) {
  const uint32_t m = bit_mask<N>(w);
  return __uint_as_float((__float_as_uint(v) & m) | (0xff800000u & ~m));
}
// t[j] += (of in lane j of the lane's row of 16) * s[j], j = J0 .. J0 + 7, as
// one instruction each: the compiler folds a row broadcast into a multiply or
// a subtraction, but not into a multiply-add.  (Two wait states lie between a
// register's write and its broadcast; one after a transcendental.)
template <int J0>
__device__ inline void fma_lanes8(float* t, float of, const float* s) {
  asm volatile(
      "s_nop 1\n\t"
      "v_fmac_f32_dpp %0, %8, %9 row_newbcast:%c17 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %1, %8, %10 row_newbcast:%c18 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %2, %8, %11 row_newbcast:%c19 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %3, %8, %12 row_newbcast:%c20 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %4, %8, %13 row_newbcast:%c21 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %5, %8, %14 row_newbcast:%c22 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %6, %8, %15 row_newbcast:%c23 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %7, %8, %16 row_newbcast:%c24 row_mask:0xf bank_mask:0xf"
      : "+v"(t[0]), "+v"(t[1]), "+v"(t[2]), "+v"(t[3]), "+v"(t[4]), "+v"(t[5]), "+v"(t[6]), "+v"(t[7])
      : "v"(of), "v"(s[0]), "v"(s[1]), "v"(s[2]), "v"(s[3]), "v"(s[4]), "v"(s[5]), "v"(s[6]), "v"(s[7]), "n"(J0),
        "n"(J0 + 1), "n"(J0 + 2), "n"(J0 + 3), "n"(J0 + 4), "n"(J0 + 5), "n"(J0 + 6), "n"(J0 + 7));
}
// l += (of in lane j of the lane's row of 16) * t[j], j = 0 .. 15.
__device__ inline void sum_lanes16(float& l, float of, const float* t) {
  asm volatile(
      "s_nop 1\n\t"
      "v_fmac_f32_dpp %0, %1, %2 row_newbcast:0 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %3 row_newbcast:1 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %4 row_newbcast:2 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %5 row_newbcast:3 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %6 row_newbcast:4 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %7 row_newbcast:5 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %8 row_newbcast:6 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %9 row_newbcast:7 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %10 row_newbcast:8 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %11 row_newbcast:9 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %12 row_newbcast:10 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %13 row_newbcast:11 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %14 row_newbcast:12 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %15 row_newbcast:13 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %16 row_newbcast:14 row_mask:0xf bank_mask:0xf\n\t"
      "v_fmac_f32_dpp %0, %1, %17 row_newbcast:15 row_mask:0xf bank_mask:0xf"
      : "+v"(l)
      : "v"(of), "v"(t[0]), "v"(t[1]), "v"(t[2]), "v"(t[3]), "v"(t[4]), "v"(t[5]), "v"(t[6]), "v"(t[7]), "v"(t[8]),
        "v"(t[9]), "v"(t[10]), "v"(t[11]), "v"(t[12]), "v"(t[13]), "v"(t[14]), "v"(t[15]));
}
// Matrix accumulators that inline assembly reads next: the compiler does not
// count the wait states of their last product (at most 18) for it.
__device__ inline void settled(f32x4_t (&a)[4]) {
  asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a[0]), "+v"(a[1]), "+v"(a[2]), "+v"(a[3]));
}
// A value's scale in the exponent: its log2 and its inverse.  A scale of zero
// stands for values of zero and takes 2^-100.  The smallest that kv_write gives
// other values is 2^-100 / 448, above 2^-109: smaller ones are taken for that,
// so that the inverses' sums stay in float32.  NaN stays.
__device__ inline void in_exponent(float vs, float& lv, float& rv) {
  constexpr float least = 1.5407439555097887e-33f;  // 2^-109
  const float x = vs == 0.f ? 7.888609052210118e-31f : vs < least ? least : vs;
  lv = __builtin_amdgcn_logf(x);
  rv = __builtin_amdgcn_rcpf(x);
}
// What sums under the maximum m are worth under mn, which is not lower.
__device__ inline float lowered(float m, float mn) { return m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn); }
__device__ inline u32x4_t ld16(const void* p) { return *static_cast<const u32x4_t*>(p); }

// The largest magnitude among bf16 pairs, as bits: 0x7f80 and above is not
// finite.
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
__device__ inline u16x2_t most16(u16x2_t m, u32x4_t x) {
#pragma unroll
  for (int u = 0; u < 4; ++u)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2_t, x[u] & 0x7fff7fffu));
  return m;
}
__device__ inline bool not_finite(u16x2_t m) { return m[0] >= 0x7f80 || m[1] >= 0x7f80; }
// Numbers that are not finite as zeros.
__device__ inline u32x4_t finite16(u32x4_t x) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const uint32_t top = ((x[u] & 0x7f807f80u) + 0x00800080u) >> 15 & 0x00010001u;
    x[u] &= ~((top << 16) - top);
  }
  return x;
}
// 1 for each of two bf16 numbers that a test of its bits holds for, else 0.
template <class Test>
__device__ inline uint32_t ones16(uint32_t w, Test test) {
  return (test(w & 0xffffu) ? 0x3f80u : 0u) | (test(w >> 16) ? 0x3f800000u : 0u);
}

template <class F, int... J>
__device__ inline void each16(F f, std::integer_sequence<int, J...>) {
  (f(std::integral_constant<int, J>{}), ...);
}
template <class F>
__device__ inline void for16(F f) {
  each16(f, std::make_integer_sequence<int, 16>{});
}

template <int ND>
__device__ inline void rescale(f32x4_t (&o)[ND], float w) {
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 4; ++v) o[d][v] *= w;
}
__device__ inline float largest16(const float (&t)[16]) {
  float r = t[0];
#pragma unroll
  for (int j = 1; j < 16; ++j) r = fmaxf(r, t[j]);
  return r;
}

// The scores of a tile become weights.  A lane holds 16 scores of one token (of
// lane & 15), those of the keys 16 g + j, g = lane >> 4, as acc[j / 4][j % 4];
// scales of the tile's key k lie in lane k.  whole: every token sees every
// key, else bit j of `mine` says whether the lane's token sees key 16 g + j.
// pf gets the weights rounded to bf16, with TWO pl what the rounding left.
// CAREFUL: for scores of any size (careful_again).  Scores are rounded, and
// compared over m or the largest of them, before value scales come in.
template <int KIND, int ND, bool TWO, bool CAREFUL = false>
__device__ inline void weigh(f32x4_t (&acc)[4], float sc, float ksl, float lvl, float rvl, bool whole, uint32_t mine,
                             float& m, float& l, f32x4_t (&o)[ND], u32x4_t (&pf)[2], u32x4_t (&pl)[2]) {
  // exponents, over m (0 while the token has seen nothing)
  float t[16];
  auto mx = [](float u, float w) { return fmaxf(u, w); };
  auto mask = [&] {
    if (whole) return;
    for16([&](auto jt) {
      constexpr int j = decltype(jt)::value;
      t[j] = only<j>(mine, t[j]);
    });
  };
  const float mu = m == kLowest ? 0.f : m;
  if constexpr (CAREFUL) {
    for16([&](auto jt) {
      constexpr int j = decltype(jt)::value;
      t[j] = acc[j >> 2][j & 3] * (KIND == SRW_KV_BF16 ? sc : row_lane<j>(ksl));
    });
    mask();
    float mt = join32(join16(largest16(t), mx), mx);
    const float r = fabsf(m) <= kLarge ? m : fmaxf(m, mt), rz = r == kLowest ? 0.f : r;
    for16([&](auto jt) {
      constexpr int j = decltype(jt)::value;
      t[j] -= rz;
      if constexpr (KIND != SRW_KV_BF16) t[j] += row_lane<j>(lvl);
    });
    mask();
    mt = join32(join16(largest16(t), mx), mx);
    // (a large r does not resolve what value scales add)
    const float up = !(fabsf(r) <= kLarge) ? 0.f : m == kLowest ? mt : fmaxf(mt, 0.f);
    const float w = __builtin_amdgcn_exp2f((m == r ? 0.f : m - r) - up);
    m = r + up;
    l *= w;
    rescale(o, w);
#pragma unroll
    for (int j = 0; j < 16; ++j) t[j] -= up;
  } else {
    if constexpr (KIND == SRW_KV_BF16) {
#pragma unroll
      for (int j = 0; j < 16; ++j) t[j] = fmaf(acc[j >> 2][j & 3], sc, -mu);
    } else {
      float s[16];
      settled(acc);
      for16([&](auto jt) {
        constexpr int j = decltype(jt)::value;
        s[j] = acc[j >> 2][j & 3];
        t[j] = row_lane<j>(lvl) - mu;
      });
      fma_lanes8<0>(t, ksl, s);
      fma_lanes8<8>(t + 8, ksl, s + 8);
    }
    mask();
    float mt = largest16(t);
    if (__any(mt > (m == kLowest ? kLowest : kLazy))) {
      mt = join32(join16(mt, mx), mx);
      const float mn = fmaxf(mu + mt, m), up = mn - mu;
      const float w = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= w;
      rescale(o, w);
#pragma unroll
      for (int j = 0; j < 16; ++j) t[j] -= up;
    }
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) t[j] = __builtin_amdgcn_exp2f(t[j]);
  if constexpr (KIND == SRW_KV_BF16) {
#pragma unroll
    for (int j = 0; j < 16; ++j) l += t[j];
  } else if (whole) {
    sum_lanes16(l, rvl, t);
  } else {  // the scale of a key that is not seen may be anything
    for16([&](auto jt) {
      constexpr int j = decltype(jt)::value;
      l += __uint_as_float(__float_as_uint(row_lane<j>(rvl) * t[j]) & bit_mask<j>(mine));
    });
  }
#pragma unroll
  for (int st = 0; st < 2; ++st)
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const float p0 = t[8 * st + 2 * u], p1 = t[8 * st + 2 * u + 1];
      const uint32_t hi = pack_bf16(p0, p1);
      pf[st][u] = hi;
      if constexpr (TWO) pl[st][u] = pack_bf16(p0 - lo_f32(hi), p1 - hi_f32(hi));
    }
}

// A wave's rows, up to 16 from r0 on, over the tiles first, first + step, ... < end
// of a span, for scores and values of any size: straight from memory, a fragment
// at a time.  Values that are not finite are kept out of the products; where there
// are any, a second pass adds them to the rows that see them.
template <int KIND, int DH>
__device__ inline void careful_rows(const AttnArgs& a, const Tile& tl, const KvSpan& sp, int h, int r0, int r1, int first,
                                    int end, int step, float& m, float& l, f32x4_t (&o)[DH / 16]) {
  constexpr int ES = kv_bytes<KIND>();
  constexpr int ND = DH / 16;
  int lane = threadIdx.x & 63;
  asm volatile("" : "+v"(lane));  // nothing here is worked out before it is needed
  const int col = lane & 15, g = lane >> 4;
  const KvSeq& sq = tl.sq;
  const int P = a.kv.P, fr = r0 + col;
  const bool in = fr < r1;
  const int tok = in ? fr / a.G : 0, pos = in ? sq.len - sq.n + tok : -1;
  const uint16_t* src = a.q + (sq.row0 + tok) * a.q_token + (h * a.G + (in ? fr - tok * a.G : 0)) * a.q_head;
  // the keys of lane group g in the tile at key0: which the lane's token sees (bit j:
  // key 16 g + j), which any row does, and their values
  uint32_t mine, seen;
  const char* vsrc;
  auto values_of = [&](int key0) {
    const int kv = key0 + 16 * g;
    const int pv = kv < sp.hi ? kv_page(a.kv, tl.b, kv) : -1;
    mine = pv < 0 ? 0u : static_cast<uint32_t>(kv_seen(pos, key0, a.window, a.sinks) >> (16 * g)) & 0xffffu;
    seen = mine;
    for (int w = 1; w < 16; w <<= 1) seen |= __shfl_xor(seen, w);
    const int64_t hv = static_cast<int64_t>(pv < 0 ? 0 : pv) * a.kv.H + h;
    vsrc = a.kv.v + ((hv * DH + col) * P + (kv & (P - 1))) * ES;
    return hv * P + (kv & (P - 1)) + col;  // (of the scales)
  };
  auto value = [&](int d, int st) {  // of the keys that some row sees
    const char* at = vsrc + static_cast<int64_t>(16 * d) * P * ES;
    u32x4_t v;
    if constexpr (KIND == SRW_KV_BF16) {
      v = ld16(at + 16 * st);
    } else {
      const uint2 raw = *reinterpret_cast<const uint2*>(at + 8 * st);
      v = widen8<KIND>(raw.x, raw.y);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t two = seen >> (8 * st + 2 * u);
      v[u] &= (two & 1 ? 0x0000ffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
    }
    return v;
  };
  m = kLowest;
  l = 0.f;
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  u16x2_t most = {0, 0};
  for (int i = first; i < end; i += step) {
    const int key0 = sp.key0(i);
    // (rows of the first product as in attn_rows_kernel)
    const int kk = key0 + 16 * (col >> 2);
    int pk = kk < sp.hi ? kv_page(a.kv, tl.b, kk) : -1;
    pk = pk < 0 ? 0 : pk;
    const int64_t hk = static_cast<int64_t>(pk) * a.kv.H + h;
    const char* ksrc = a.kv.k + (hk * P + (kk & (P - 1)) + (col & 3)) * (DH * ES) + 16 * g;
    f32x4_t acc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      acc[t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < DH * ES / 64; ++j) {
        const u32x4_t k = ld16(ksrc + 4 * t * (DH * ES) + 64 * j);
        if constexpr (KIND == SRW_KV_BF16) {
          acc[t] = mfma16(k, in ? ld16(src + 32 * j + 8 * g) : u32x4_t{0, 0, 0, 0}, acc[t]);
        } else {
#pragma unroll
          for (int s = 0; s < 2; ++s)
            acc[t] = mfma16(widen8<KIND>(k[2 * s], k[2 * s + 1]),
                            in ? ld16(src + 64 * j + 16 * g + 8 * s) : u32x4_t{0, 0, 0, 0}, acc[t]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    const int64_t scale_at = values_of(key0);
    float ksl = 0.f, lvl = 0.f, rvl = 0.f;
    if constexpr (KIND != SRW_KV_BF16) {
      ksl = a.kv.ks[scale_at] * a.sc;
      in_exponent(a.kv.vs[scale_at], lvl, rvl);
    }
    u32x4_t pf[2], pl[2];
    weigh<KIND, ND, true, true>(acc, a.sc, ksl, lvl, rvl, false, mine, m, l, o, pf, pl);
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        u32x4_t v = value(d, st);
        if constexpr (KIND != SRW_KV_INT8) {
          most = most16(most, v);
          v = finite16(v);
        }
        o[d] = mfma16(v, pl[st], mfma16(v, pf[st], o[d]));
        __builtin_amdgcn_sched_barrier(0);
      }
  }
  if (KIND == SRW_KV_INT8 || !__any(not_finite(most))) return;
  for (int i = first; i < end; i += step) {
    values_of(sp.key0(i));
    // a row gets each kind of number that is not finite which it sees: how many there
    // are is a product of zeros and ones
    auto add = [&](auto test, float x) {
#pragma unroll
      for (int d = 0; d < ND; ++d) {
        f32x4_t n = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          u32x4_t is = value(d, st), sees;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            is[u] = ones16(is[u], test);
            const uint32_t two = mine >> (8 * st + 2 * u);
            sees[u] = (two & 1 ? 0x3f80u : 0u) | (two & 2 ? 0x3f800000u : 0u);
          }
          n = mfma16(is, sees, n);
        }
#pragma unroll
        for (int r = 0; r < 4; ++r) o[d][r] += n[r] > 0.f ? x : 0.f;
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    add([](uint32_t b) { return b == 0x7f80u; }, INFINITY);
    add([](uint32_t b) { return b == 0xff80u; }, -INFINITY);
    add([](uint32_t b) { return (b & 0x7fffu) > 0x7f80u; }, __uint_as_float(0x7fc00000u));
  }
}

// Whether a wave's rows have to be walked again, by careful_rows: m is so large
// that a product (exact) and m (rounded) do not cancel, that 2^(product - m) could
// be anything and log2 vs is lost beside m; or a sum is not finite, as such weights
// or values leave it (an infinity times what is left of a weight, zero or negative,
// is NaN, and so is zero times one that a row does not see).
template <int ND>
__device__ inline bool careful_again(float m, float l, const f32x4_t (&o)[ND]) {
  f32x4_t none = {l * 0.f, 0.f, 0.f, 0.f};  // NaN once a sum is not finite
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 4; ++v) none[v] = fmaf(o[d][v], 0.f, none[v]);
  const bool odd = none[0] + none[1] + none[2] + none[3] != 0.f;
  return __any(odd || (fabsf(m) > kLarge && m != kLowest));
}

// -- few rows: single tokens, short chunks -----------------------------------
//
// A workgroup takes up to 16 NQ rows (token, head of the group) of one
// sequence and key head; its four waves take every fourth tile of its split,
// each with its own m, l and O, and join in LDS at the end.  Bound by the
// pages' bytes: a wave loads both operands' fragments straight into
// registers, 16 bytes a lane, no barrier in the loop.  Measured: 32 sequences
// of 4 000 to 32 000 positions, 32 heads on 8 of 128, fp8, in 260 us, 4.7 TB/s (a
// large copy's traffic: 4.9); 64 sequences of up to 512, 6 heads of 64, int8, in 9.
//
// Waves on a SIMD that its registers are kept for (32 sequences of 18 000
// positions, fp8, head_dim 128: 276 us with three, 281 with two).
template <int KIND, int DH, int NQ> constexpr int rows_waves() {
  return NQ > 1 ? 1 : DH == 64 ? 4 : KIND == SRW_KV_BF16 ? 2 : 3;
}
template <int KIND, int DH, int NQ>
__global__ __launch_bounds__(256, (rows_waves<KIND, DH, NQ>())) void attn_rows_kernel(AttnArgs a) {
  constexpr int ES = kv_bytes<KIND>();
  constexpr int NPC = DH * ES / 64;  // 16-byte pieces of a key a lane
  constexpr int NS = DH / 32;        // k-steps of the first product
  constexpr int ND = DH / 16;
  __shared__ float sm[4][16 * NQ], sl[4][16 * NQ];
  __shared__ float so[4][16 * NQ][DH + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int split = blockIdx.z, h = blockIdx.y;
  const Tile tl = tile_of<16 * NQ>(a, blockIdx.x);
  if (tl.r0 < 0) return;
  const int64_t b = tl.b;
  const KvSeq sq = tl.sq;
  const int r0 = tl.r0, r1 = tl.r1;
  const int P = a.kv.P;
  const int p_lo = sq.len - sq.n + r0 / a.G, p_hi = sq.len - sq.n + (r1 - 1) / a.G;
  const KvSpan sp = span_of(a, p_lo, p_hi);
  const int per = per_split(a, sp.tiles);
  const int i0 = split * per;
  const int i1 = i0 + per < sp.tiles ? i0 + per : sp.tiles;

  u32x4_t q[NQ][NS];
  int pos[NQ];
  float m[NQ], l[NQ];
  f32x4_t o[NQ][ND];
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const int fr = r0 + 16 * x + col;
    const bool in = fr < r1;
    const int tok = in ? fr / a.G : 0;
    pos[x] = in ? sq.len - sq.n + tok : -1;
    const uint16_t* src = a.q + (sq.row0 + tok) * a.q_token + (h * a.G + (in ? fr - tok * a.G : 0)) * a.q_head;
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      // the dims of this step's slots, as the key pieces below hold them
      const int d = ES == 2 ? 32 * s + 8 * g : 64 * (s / 2) + 16 * g + 8 * (s & 1);
      q[x][s] = in ? ld16(src + d) : u32x4_t{0, 0, 0, 0};
    }
  }

#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    m[x] = kLowest;
    l[x] = 0.f;
#pragma unroll
    for (int d = 0; d < ND; ++d) o[x][d] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  for (int i = i0 + wave; i < i1; i += 4) {
    const int key0 = sp.key0(i);
    // rows of the first product: row 4 u + v of its tile t is key 16 u + 4 t
    // + v, so lane (col, g) loads keys of group col / 4 and its score
    // registers, like its k-slots of the second product, are those of group g
    const int kk = key0 + 16 * (col >> 2), kv = key0 + 16 * g;
    int pk = kk < sp.hi ? kv_page(a.kv, b, kk) : -1, pv = kv < sp.hi ? kv_page(a.kv, b, kv) : -1;
    const bool have = pv >= 0;
    pk = pk < 0 ? 0 : pk;
    pv = pv < 0 ? 0 : pv;
    const int64_t hk = static_cast<int64_t>(pk) * a.kv.H + h, hv = static_cast<int64_t>(pv) * a.kv.H + h;
    const char* ksrc = a.kv.k + (hk * P + (kk & (P - 1)) + (col & 3)) * (DH * ES) + 16 * g;
    const char* vsrc = a.kv.v + ((hv * DH + col) * P + (kv & (P - 1))) * ES;
    u32x4_t kf[4][NPC], vf[ND][ES];
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int j = 0; j < NPC; ++j) kf[t][j] = ld16(ksrc + 4 * t * (DH * ES) + 64 * j);
    float ksl = 0.f, lvl = 0.f, rvl = 0.f;
    if constexpr (KIND != SRW_KV_BF16) {
      ksl = a.kv.ks[hv * P + (kv & (P - 1)) + col] * a.sc;
      in_exponent(a.kv.vs[hv * P + (kv & (P - 1)) + col], lvl, rvl);
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int j = 0; j < ES; ++j) vf[d][j] = ld16(vsrc + static_cast<int64_t>(16 * d) * P * ES + 16 * j);

    f32x4_t acc[NQ][4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      u32x4_t kb[NS];
#pragma unroll
      for (int j = 0; j < NPC; ++j) {
        if constexpr (KIND == SRW_KV_BF16) {
          kb[j] = kf[t][j];
        } else {
          kb[2 * j] = widen8<KIND>(kf[t][j][0], kf[t][j][1]);
          kb[2 * j + 1] = widen8<KIND>(kf[t][j][2], kf[t][j][3]);
        }
      }
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        acc[x][t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s) acc[x][t] = mfma16(kb[s], q[x][s], acc[x][t]);
      }
    }
    // every row sees every key of the tile?
    const bool whole = __all(have) && key0 + kTile - 1 <= p_lo &&
                       (a.window == 0 || key0 > p_hi - a.window || key0 + kTile <= a.sinks);
    uint32_t seen = 0;  // bit j: some row of the tile sees the lane's key kv + j
    u32x4_t pf[NQ][2], pl[NQ][2];
#pragma unroll
    for (int x = 0; x < NQ; ++x) {
      uint32_t mine = 0xffffu;
      if (!whole) {
        mine = have ? static_cast<uint32_t>(kv_seen(pos[x], key0, a.window, a.sinks) >> (16 * g)) & 0xffffu : 0u;
        seen |= mine;
      }
      weigh<KIND, ND, true>(acc[x], a.sc, ksl, lvl, rvl, whole, mine, m[x], l[x], o[x], pf[x], pl[x]);
    }
    if (!whole && KIND != SRW_KV_INT8) {
      for (int w = 1; w < 16; w <<= 1) seen |= __shfl_xor(seen, w);  // over the columns: keys that some row sees
#pragma unroll
      for (int u = 0; u < 4 * ES; ++u) {  // a dword's keys
        uint32_t keep;
        if constexpr (ES == 2) {
          const uint32_t two = seen >> (2 * u);
          keep = (two & 1 ? 0x0000ffffu : 0u) | (two & 2 ? 0xffff0000u : 0u);
        } else {
          keep = ((seen >> (4 * u) & 15u) * 0x00204081u & 0x01010101u) * 0xffu;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) vf[d][u / 4][u % 4] &= keep;
      }
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
#pragma unroll
      for (int st = 0; st < 2; ++st) {
        u32x4_t vb;
        if constexpr (KIND == SRW_KV_BF16)
          vb = vf[d][st];
        else
          vb = widen8<KIND>(vf[d][0][2 * st], vf[d][0][2 * st + 1]);
#pragma unroll
        for (int x = 0; x < NQ; ++x) o[x][d] = mfma16(vb, pl[x][st], mfma16(vb, pf[x][st], o[x][d]));
      }
    }
  }

#pragma unroll
  for (int x = 0; x < NQ; ++x)
    if (careful_again(m[x], l[x], o[x])) careful_rows<KIND, DH>(a, tl, sp, h, r0 + 16 * x, r1, i0 + wave, i1, 4, m[x], l[x], o[x]);

  // join the four waves
  auto sum = [](float u, float w) { return u + w; };
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    l[x] = join32(join16(l[x], sum), sum);
    if (g == 0) {
      sm[wave][16 * x + col] = m[x];
      sl[wave][16 * x + col] = l[x];
    }
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<f32x4_t*>(&so[wave][16 * x + col][16 * d + 4 * g]) = o[x][d];
  }
  __syncthreads();
  // thread (r, c): DH / 16 consecutive dims of a row, 16 rows a pass
#pragma unroll
  for (int x = 0; x < NQ; ++x) {
    const int r = 16 * x + (threadIdx.x >> 4), c = (threadIdx.x & 15) * ND;
    const int fr = r0 + r;
    if (fr < r1) {
      float mm = sm[0][r];
#pragma unroll
      for (int w = 1; w < 4; ++w) mm = fmaxf(mm, sm[w][r]);
      float ll = 0.f, ov[ND];
#pragma unroll
      for (int d = 0; d < ND; ++d) ov[d] = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        // (a wave without visible keys has l = 0)
        const float e = lowered(sm[w][r], mm);
        ll += sl[w][r] * e;
#pragma unroll
        for (int d = 0; d < ND; ++d) ov[d] += so[w][r][c + d] * e;
      }
      const int tok = fr / a.G;
      const int64_t row = (sq.row0 + tok) * a.Hq + h * a.G + (fr - tok * a.G);
      if (a.S == 1) {
        const float inv = ll == 0.f ? 0.f : 1.f / ll;
        uint32_t w[ND / 2];
#pragma unroll
        for (int d = 0; d < ND / 2; ++d) w[d] = pack_bf16(ov[2 * d] * inv, ov[2 * d + 1] * inv);
        if constexpr (ND == 8)
          *reinterpret_cast<uint4*>(a.out + row * DH + c) = make_uint4(w[0], w[1], w[2], w[3]);
        else
          *reinterpret_cast<uint2*>(a.out + row * DH + c) = make_uint2(w[0], w[1]);
      } else {
        const int64_t at = split * (a.kv.T * a.Hq) + row;
        if (ll != 0.f) {
#pragma unroll
          for (int d = 0; d < ND; d += 4)
            *reinterpret_cast<f32x4_t*>(a.part + at * DH + c + d) = f32x4_t{ov[d], ov[d + 1], ov[d + 2], ov[d + 3]};
        }
        if (c == 0) a.ml[at] = make_float2(mm, ll);
      }
    }
  }
}

// Joins the splits.  Groups of DH / 4 lanes; W of them take a row's splits in
// turn, each with four loads in flight, and join in LDS: one for few splits (no
// LDS), four for more, all of a workgroup of 1024 for the many splits of up to
// 256 rows (6 rows of 160 splits: 23 us with the attention before it, 30 with
// four groups; 360 of 35: 21, and 17 with four; 128 tokens of 6 heads over 4 000
// positions in 8 splits: 14 with one group, 23 with all).
template <int DH, int W, int TH>
__global__ __launch_bounds__(TH) void attn_join_kernel(const float* part, const float2* ml, uint16_t* out, int64_t rows,
                                                       int S) {
  constexpr int L = DH / 4, N = TH / L;  // lanes a group, groups
  const int c = threadIdx.x % L, first = threadIdx.x / L / W * W, grp = threadIdx.x / L - first;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * (N / W) + first / W;
  const int64_t row = at < rows ? at : rows - 1;
  float m = kLowest, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;
  for (int s0 = grp; s0 < S; s0 += W * U) {
    float2 x[U];
    f32x4_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + W * u < S ? s0 + W * u : s0;
      x[u] = ml[s * rows + row];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {  // a split without visible keys wrote no output
      const int s = s0 + W * u < S ? s0 + W * u : s0;
      if (x[u].y != 0.f) v[u] = *reinterpret_cast<const f32x4_t*>(part + (s * rows + row) * DH + 4 * c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (s0 + W * u >= S || x[u].y == 0.f) continue;
      const float mn = fmaxf(m, x[u].x);
      const float e0 = lowered(m, mn), e1 = lowered(x[u].x, mn);
      m = mn;
      l = l * e0 + x[u].y * e1;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = o[k] * e0 + v[u][k] * e1;
    }
  }
  if constexpr (W > 1) {
    __shared__ float sm[N], sl[N];
    __shared__ f32x4_t so[N][L];
    if (c == 0) {
      sm[first + grp] = m;
      sl[first + grp] = l;
    }
    so[first + grp][c] = o;
    __syncthreads();
    if (grp != 0) return;
    m = sm[first];
    l = 0.f;
#pragma unroll
    for (int g = 1; g < W; ++g) m = fmaxf(m, sm[first + g]);
    o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int g = 0; g < W; ++g) {
      const float e = lowered(sm[first + g], m);
      l += sl[first + g] * e;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] += so[first + g][c][k] * e;
    }
  }
  if (at >= rows) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  *reinterpret_cast<uint2*>(out + row * DH + 4 * c) =
      make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
}

// -- many rows: chunks of prompts ---------------------------------------------
//
// 128 rows a workgroup, 16 to each of eight waves; a tile's keys and values go
// through LDS once for all of them, two stages deep.  bf16 pages are copied
// there directly (global_load_lds), 8-bit ones are widened on the way.  16-byte
// pieces of a row are XOR-swizzled by the row so that the 16 lanes of a
// fragment read cover all banks.
//
// Vector work fills it most: a score takes 4 (bf16) or 5 (8 bits) instructions
// and an exponential, which costs 2.5 of them, against 4 head_dim products.  Of a
// long chunk's SIMD cycles the vector ALU is active for 70%, the matrix cores for
// 29%; the LDS, whose every fragment feeds one product, is for 44% of a CU's.  None
// is full: a wave alone issues a vector instruction every 8 cycles, half the SIMD's
// rate, and matrix instructions run beside other waves' vector ones; so what counts
// is waves on a SIMD, and with 16 rows a wave (at most 128 registers) four fit,
// where 32 rows (240 registers at head_dim 128) left two.
//
// Measured: 2 048 tokens of 32 heads over 30 011 positions of 8, int8, head_dim
// 128, in 1 400 to 1 430 us, 0.73 PFLOP/s (32 rows a wave: 1 363, but calls of few tiles
// twice as long); 8 prompts of 512 of 6 heads of 64, bf16, in 14 us (39 so).
template <int DH> __device__ inline int k_swz(int row) {
  // a fragment's 16 rows are 16 u + 4 t + v, u, v = 0 .. 3
  return DH == 64 ? (row >> 1 & 1) | (row >> 3 & 6) : (row & 3) | (row >> 2 & 12);
}
// (the lanes of one LDS access may be of two neighbouring g, columns 0-3 and
// 12-15 of one and 4-11 of the other, whose pieces differ in bits 1 and 2: bit 0
// tells those columns apart)
__device__ inline int v_swz(int row) { return ((row >> 2 ^ row >> 3) & 1) | (row & 2) | (row >> 1 & 4); }

template <int KIND, int DH>
__global__ __launch_bounds__(512, 4) void attn_tile_kernel(AttnArgs a) {
  constexpr int ES = kv_bytes<KIND>();
  constexpr int NS = DH / 32, ND = DH / 16;
  constexpr int NP = DH / 8;               // pieces of a key row
  constexpr int kStage = kTile * DH * 2;   // bytes of a tile's keys (or values) in LDS
  constexpr int NI = kStage / 8192;        // 16-byte pieces a thread of either
  constexpr bool Q8 = KIND != SRW_KV_BF16;
  constexpr int kBatch = DH == 64 ? 8 : 4;  // fragments read together
  __shared__ __align__(16) char kl[2][kStage];
  __shared__ __align__(16) char vl[2][kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int g = lane >> 4;
  const int h = blockIdx.y, split = blockIdx.z;
  const int P = a.kv.P;
  const Tile tl = tile_of<128>(a, blockIdx.x);
  if (tl.r0 < 0) return;
  const int64_t b = tl.b;
  const KvSeq sq = tl.sq;
  const int r0 = tl.r0, r1 = tl.r1;
  const KvSpan sp = span_of(a, sq.len - sq.n + r0 / a.G, sq.len - sq.n + (r1 - 1) / a.G);
  const int per = per_split(a, sp.tiles);
  const int i0 = split * per;
  const int i1 = i0 + per < sp.tiles ? i0 + per : sp.tiles;

  // this wave's rows
  const int w0 = r0 + 16 * wave, w1 = w0 + 16 < r1 ? w0 + 16 : r1;
  const bool active = w0 < r1;
  const int p_lo = sq.len - sq.n + w0 / a.G, p_hi = sq.len - sq.n + (w1 - 1) / a.G;
  // (the loop has no registers to keep a row's place: it is worked out again
  // where it is needed)
  struct Place {
    bool in;
    int tok, head, pos;
  };
  auto place = [&] {
    int c = threadIdx.x & 15;
    asm volatile("" : "+v"(c));
    Place p;
    p.in = w0 + c < r1;
    p.tok = p.in ? (w0 + c) / a.G : 0;
    p.head = h * a.G + (p.in ? w0 + c - p.tok * a.G : 0);
    p.pos = p.in ? sq.len - sq.n + p.tok : -1;
    return p;
  };
  u32x4_t q[NS];
  {
    const Place p = place();
    const bool in = p.in;
    const int tok = p.tok, head = p.head;
    const uint16_t* src = a.q + (sq.row0 + tok) * a.q_token + head * a.q_head + 8 * g;
#pragma unroll
    for (int s = 0; s < NS; ++s) q[s] = in ? ld16(src + 32 * s) : u32x4_t{0, 0, 0, 0};
  }
  float m = kLowest, l = 0.f;
  f32x4_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d) o[d] = f32x4_t{0.f, 0.f, 0.f, 0.f};

  // At head_dim 128 the loop has no registers for addresses that it could keep:
  // they are worked out from the lane again (one that was spilled cost a wait for
  // the tile's loads in flight: a tenth of a call over small pages).
  auto fresh = [](int x) {
    if constexpr (DH == 128) asm volatile("" : "+v"(x));
    return x;
  };
  // Slots: pages of 64 and more hold whole tiles (one page each), at slot0 of
  // theirs; smaller ones start with one.  Where tiles lie is worked out 16 at a
  // time, a lane for each group of 16 positions: lane 4 n + u has the byte offset
  // of the page of tile ib + n's positions 16 u .. (of page 0 where they have
  // none), and bit 4 n + u of `have` says whether there is one.  (Done a tile at
  // a time by every wave, on the scalar unit that the whole CU shares, it cost
  // as much as the products.)
  const bool one = P >= kTile;
  const int64_t page_bytes = static_cast<int64_t>(a.kv.H) * P * DH * ES, head_at = static_cast<int64_t>(h) * P * DH * ES;
  const char* kbase = a.kv.k + head_at;
  const char* vbase = a.kv.v + head_at;
  int ib = i0, off_lo = 0, off_hi = 0;
  uint64_t have = 0;
  auto locate = [&] {
    int ln = lane;  // (once in 16 tiles: not worth a register either)
    asm volatile("" : "+v"(ln));
    const int i = ib + (ln >> 2), at = sp.key0(i) + 16 * (ln & 3);
    const int id = i < i1 && at < sp.hi ? kv_page(a.kv, b, at) : -1;
    have = __ballot(id >= 0);
    const int64_t off = (id < 0 ? 0 : id) * page_bytes;
    off_lo = static_cast<int>(off);
    off_hi = static_cast<int>(off >> 32);
  };
  if (i0 < i1) locate();
  u32x4_t rk, rv;               // 8-bit tiles on their way
  float ksn = 0.f, vsn = 0.f;   // scales of key `lane`
  int havn = 0;                 // bit u: positions 16 u .. have a page
  // Where a thread's pieces lie in a page, from its first slot of the tile.
  // 8 bits: 16 codes, of keys 16 dims of a position (the wave's positions in one
  // group of 16), of values 16 positions of a dim; at head_dim 64 the first four
  // waves take the keys, the others the values.  (bf16: a wave's second key
  // pieces are four positions, and four rows of the same swizzle, behind its
  // first.)
  auto key_at = [&]() -> uint32_t {
    const int tx = fresh(threadIdx.x);
    if constexpr (Q8) return (tx / (NP / 2) & (P - 1)) * DH + 16 * (tx % (NP / 2));
    const int row = (wave * NI * 64 + (tx & 63)) / NP;
    return ((row & (P - 1)) * DH + 8 * ((tx & 63) % NP ^ k_swz<DH>(row))) * ES;
  };
  auto value_at = [&](int n) -> uint32_t {
    const int tx = fresh(threadIdx.x);
    if constexpr (Q8) return ((tx >> 2) - (DH == 64 && wave >= 4 ? 64 : 0)) * P + ((16 * (tx & 3)) & (P - 1));
    const int row = ((wave * NI + n) * 64 + (tx & 63)) / 8;
    return (row * P + ((8 * ((tx & 7) ^ v_swz(row))) & (P - 1))) * ES;
  };
  uint32_t kat0 = 0, vat0[NI];
  if constexpr (DH == 64) {
    kat0 = key_at();
#pragma unroll
    for (int n = 0; n < NI; ++n) vat0[n] = value_at(n);
  }
  auto fetch = [&](int i, int stage) {
    uint32_t kat = kat0, vat[NI];
    if constexpr (DH == 128) kat = key_at();
#pragma unroll
    for (int n = 0; n < NI; ++n) vat[n] = DH == 64 ? vat0[n] : value_at(n);
    const int at = 4 * (i - ib), slot0 = sp.key0(i) & (P - 1);
    havn = static_cast<int>(have >> at) & 15;
    auto page = [&](int u) -> int64_t {  // of group u, the same for the whole wave
      const uint32_t lo = __builtin_amdgcn_readlane(off_lo, at + u), hi = __builtin_amdgcn_readlane(off_hi, at + u);
      return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
    };
    auto page_of_lane = [&](int u) -> int64_t {
      const uint32_t lo = __shfl(off_lo, at + u), hi = __shfl(off_hi, at + u);
      return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
    };
    const int64_t page0 = one ? page(0) : 0;
    if constexpr (!Q8) {
      const int ku = wave * NI * 64 / NP >> 4;  // (a wave's keys are of one group)
      const char* src = kbase + (one ? page0 : page(ku)) + slot0 * (DH * ES);
#pragma unroll
      for (int n = 0; n < NI; ++n)
        g2lds16(src + n * (64 / NP * DH * ES) + kat, kl[stage] + 16 * (wave * NI + n) * 64);
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int first = (wave * NI + n) * 64;
        if (one) {
          g2lds16(vbase + page0 + slot0 * ES + vat[n], vl[stage] + 16 * first);
        } else {
          const int ln = fresh(lane), group = ((ln & 7) ^ v_swz((first + ln) / 8)) >> 1;
          g2lds16(vbase + page_of_lane(group) + vat[n], vl[stage] + 16 * first);
        }
      }
    } else {
      if (DH == 128 || wave < 4) {
        const char* src = kbase + (one ? page0 : page(wave * 64 / (NP / 2) >> 4)) + slot0 * DH;
        rk = ld16(src + kat);
      }
      if (DH == 128 || wave >= 4) {
        if (one)
          rv = ld16(vbase + page0 + slot0 + vat[0]);
        else
          rv = ld16(vbase + page_of_lane(lane & 3) + vat[0]);
      }
      if (one) {
        const int64_t first = (page0 >> (DH == 64 ? 6 : 7)) + (h * P + slot0);
        int at4 = 4 * (threadIdx.x & 63);
        asm volatile("" : "+v"(at4));
        ksn = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(a.kv.ks + first) + static_cast<uint32_t>(at4));
        vsn = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(a.kv.vs + first) + static_cast<uint32_t>(at4));
      } else {
        const int64_t first = (page_of_lane(g) >> (DH == 64 ? 6 : 7)) + (h * P + (lane & (P - 1)));
        ksn = a.kv.ks[first];
        vsn = a.kv.vs[first];
      }
    }
  };
  // positions of the tile at key0 that some row of the workgroup sees; hav: its
  // groups that have pages
  auto seen_by_any = [&](int key0, int hav) {
    uint64_t keys = low_bits(sp.hi - key0);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (!(hav >> u & 1)) keys &= ~(0xffffull << (16 * u));
    if (key0 < sp.lo) keys &= ~low_bits(sp.lo - key0) | low_bits(a.sinks - key0);
    return keys;
  };
  auto settle = [&](int key0, int stage) {  // 8 bits: widen into LDS
    if constexpr (Q8) {
      const int tx = fresh(threadIdx.x);
      if (DH == 128 || wave < 4) {
        const int row = tx / (NP / 2), pc = tx % (NP / 2);
#pragma unroll
        for (int u = 0; u < 2; ++u)
          *reinterpret_cast<u32x4_t*>(kl[stage] + row * (DH * 2) + 16 * ((2 * pc + u) ^ k_swz<DH>(row))) =
              widen8<KIND>(rk[2 * u], rk[2 * u + 1]);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (DH == 128 || wave >= 4) {
        const int row = (tx >> 2) - (DH == 64 ? 64 : 0), pc = tx & 3;
        const bool late = row & 2;  // (its pieces meet those of row - 2 in other banks)
        if (KIND == SRW_KV_FP8 && (havn != 15 || sp.hi - key0 < kTile || key0 < sp.lo)) {
          // codes of positions that no row sees may be NaN's
          const uint32_t bits = static_cast<uint32_t>(seen_by_any(key0, havn) >> (16 * pc));
#pragma unroll
          for (int u = 0; u < 4; ++u) rv[u] &= ((bits >> (4 * u) & 15u) * 0x00204081u & 0x01010101u) * 0xffu;
        }
        const u32x4_t x = late ? u32x4_t{rv[2], rv[3], rv[0], rv[1]} : rv;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          *reinterpret_cast<u32x4_t*>(vl[stage] + row * 128 + 16 * ((2 * pc + (u ^ (late ? 1 : 0))) ^ v_swz(row))) =
              widen8<KIND>(x[2 * u], x[2 * u + 1]);
      }
    }
  };

  if (i0 < i1) fetch(i0, 0);
  for (int i = i0; i < i1; ++i) {
    const int stage = (i - i0) & 1;
    const int key0 = sp.key0(i);
    settle(key0, stage);
    wait_vm0();
    __syncthreads();
    const int hav = havn;
    float ksl = 0.f, lvl = 0.f, rvl = 0.f;
    if constexpr (Q8) {
      ksl = ksn * a.sc;
      in_exponent(vsn, lvl, rvl);
    }
    if (i + 1 < i1) {
      if (i + 1 - ib == 16) {
        ib += 16;
        locate();
      }
      fetch(i + 1, stage ^ 1);
    }
    if (!active || key0 > p_hi) continue;

    // fragments are read several at a time, so that products wait for LDS a few
    // times and not for each of them
    const int fl = lane, fc = fl & 15, fg = fl >> 4;
    f32x4_t acc[4];
#pragma unroll
    for (int t0 = 0; t0 < 4; t0 += kBatch / NS) {
      u32x4_t kf[kBatch / NS][NS];
#pragma unroll
      for (int t = 0; t < kBatch / NS; ++t) {
        // row 4 u + v of product t0 + t holds key 16 u + 4 (t0 + t) + v
        const int row = 16 * (fc >> 2) + 4 * (t0 + t) + (fc & 3);
#pragma unroll
        for (int s = 0; s < NS; ++s) kf[t][s] = ld16(kl[stage] + row * (DH * 2) + 16 * ((4 * s + fg) ^ k_swz<DH>(row)));
      }
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < kBatch / NS; ++t) {
        acc[t0 + t] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int s = 0; s < NS; ++s) acc[t0 + t] = mfma16(kf[t][s], q[s], acc[t0 + t]);
      }
    }
    const bool whole = hav == 15 && sp.hi - key0 >= kTile && key0 + kTile - 1 <= p_lo &&
                       (a.window == 0 || key0 > p_hi - a.window || key0 + kTile <= a.sinks);
    uint64_t keys = ~0ull;
    uint32_t mine = 0xffffu;
    if (!whole) {
      keys = seen_by_any(key0, hav);
      mine = static_cast<uint32_t>((kv_seen(place().pos, key0, a.window, a.sinks) & keys) >> (16 * g)) & 0xffffu;
    }
    u32x4_t pf[2], pl[2];
    weigh<KIND, ND, false>(acc, a.sc, ksl, lvl, rvl, whole, mine, m, l, o, pf, pl);
#pragma unroll
    for (int d0 = 0; d0 < ND; d0 += kBatch / 2) {
      u32x4_t vf[kBatch / 2][2];
#pragma unroll
      for (int d = 0; d < kBatch / 2; ++d)
#pragma unroll
        for (int st = 0; st < 2; ++st)
          vf[d][st] = ld16(vl[stage] + (16 * (d0 + d) + fc) * 128 + 16 * ((2 * fg + st) ^ v_swz(fc)));
      __builtin_amdgcn_sched_barrier(0);
      if (KIND == SRW_KV_BF16 && keys != ~0ull) {  // values that no row sees
#pragma unroll
        for (int st = 0; st < 2; ++st) {
          const uint32_t bits = static_cast<uint32_t>(keys >> (16 * g + 8 * st)) & 0xffu;
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const uint32_t keep = (bits >> (2 * u) & 1 ? 0x0000ffffu : 0u) | (bits >> (2 * u + 1) & 1 ? 0xffff0000u : 0u);
#pragma unroll
            for (int d = 0; d < kBatch / 2; ++d) vf[d][st][u] &= keep;
          }
        }
      }
#pragma unroll
      for (int st = 0; st < 2; ++st)
#pragma unroll
        for (int d = 0; d < kBatch / 2; ++d) o[d0 + d] = mfma16(vf[d][st], pf[st], o[d0 + d]);
    }
  }
  if (!active) return;
  if (careful_again(m, l, o)) careful_rows<KIND, DH>(a, tl, sp, h, w0, r1, i0, i1, 1, m, l, o);
  auto sum = [](float u, float w) { return u + w; };
  l = join32(join16(l, sum), sum);
  const Place p = place();
  if (!p.in) return;
  const int64_t row = (sq.row0 + p.tok) * a.Hq + p.head;
  if (a.S == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < ND; ++d)
      *reinterpret_cast<uint2*>(a.out + row * DH + 16 * d + 4 * g) =
          make_uint2(pack_bf16(o[d][0] * inv, o[d][1] * inv), pack_bf16(o[d][2] * inv, o[d][3] * inv));
  } else {
    const int64_t at = split * (a.kv.T * a.Hq) + row;
    if (l != 0.f) {
#pragma unroll
      for (int d = 0; d < ND; ++d) *reinterpret_cast<f32x4_t*>(a.part + at * DH + 16 * d + 4 * g) = o[d];
    }
    if (g == 0) a.ml[at] = make_float2(m, l);
  }
}

// How a call runs: the kernel, and in how many splits a sequence's tiles.
struct AttnPlan {
  int rows;      // rows a workgroup: 16, 32 (attn_rows_kernel) or 128
  int64_t tiles; // row tiles of a key head, at most
  int S, least;  // splits of a row tile's key tiles, at most; tiles each, at least
};

AttnPlan plan_of(const srw_attention_t& a) {
  AttnPlan p{};
  const int64_t G = a.n_heads / a.kv.n_kv_heads, B = a.kv.B, T = a.kv.T, H = a.kv.n_kv_heads;
  const int64_t most = !a.kv.cu ? 1 : a.max_new > 0 ? a.max_new : T;
  int64_t keys = (a.kv.table_width * a.kv.page_size + kTile - 1) / kTile;  // key tiles of a row, at most
  if (a.window > 0) {
    const int64_t w = (a.window + most + kTile - 1) / kTile + 1 + (int64_t{a.sinks} + kTile - 1) / kTile;
    keys = w < keys ? w : keys;
  }
  // 32 rows a workgroup also where more would leave the GPU idle: 512 tokens of 6
  // heads in 9.8 us against 12.2 of the kernel for many rows, four times as many
  // in 13.5 against 13.0, 8 x 64 tokens over 2 000 positions in 40 against 25
  p.rows = most * G <= 16 ? 16 : most * G <= 32 || T * G * H * keys <= 65536 ? 32 : 128;
  p.tiles = !a.kv.cu ? B * ((G + p.rows - 1) / p.rows) : T * G / p.rows + B;
  const int64_t groups = p.tiles * H;
  // Splits where workgroups are too few for the GPU, of a few tiles at least: a
  // second launch joins them.  (Few rows: 2 x 100 000 positions of 8 heads in 85
  // us with about 1024 workgroups, 97 with 2048; one of 2 000 in 8.8 us with 4
  // tiles a split, 13.5 with 16; 64 x 512, 9 tiles, in 8.8 us whole, 10.2 in two.
  // Many rows: what the GPU holds at once, 512 workgroups, where a row tile gets
  // six splits or more of it; else more, since row tiles end early and sequences
  // differ: 512 tokens of 16 heads over 4 000 positions in 47.5 us with 448, 53
  // with 640; four ragged batches of 24 chunks over up to 2 000 in 47 with about
  // 1280, 50 with 768; a batch whose row tiles fill three quarters whole.)
  const bool many = p.rows == 128, once = groups * 6 <= 512;
  const int64_t want = !many ? 1024 : once ? 512 : 1280, least = many ? 8 : 4;
  const int64_t S = groups >= (many ? 384 : 512) || keys <= 12 ? 1 : want / groups;
  p.least = static_cast<int>(least);
  const int64_t most_splits = keys / least;
  p.S = static_cast<int>(S < most_splits ? S : most_splits > 1 ? most_splits : 1);
  return p;
}

template <int KIND, int DH>
hipError_t launch_attention(const srw_attention_t& a, const AttnPlan& pl, AttnArgs& g, hipStream_t s) {
  const dim3 grid(static_cast<unsigned>(pl.tiles), static_cast<unsigned>(g.kv.H), static_cast<unsigned>(g.S));
  if (pl.rows == 16)
    hipLaunchKernelGGL((attn_rows_kernel<KIND, DH, 1>), grid, dim3(256), 0, s, g);
  else if (pl.rows == 32)
    hipLaunchKernelGGL((attn_rows_kernel<KIND, DH, 2>), grid, dim3(256), 0, s, g);
  else
    hipLaunchKernelGGL((attn_tile_kernel<KIND, DH>), grid, dim3(512), 0, s, g);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || g.S == 1) return e;
  const int64_t rows = a.kv.T * a.n_heads;
  auto join = [&](auto w, auto th) {
    constexpr int W = decltype(w)::value, TH = decltype(th)::value, R = TH / (DH / 4) / W;
    hipLaunchKernelGGL((attn_join_kernel<DH, W, TH>), dim3(static_cast<unsigned>((rows + R - 1) / R)), dim3(TH), 0, s,
                       g.part, g.ml, g.out, rows, g.S);
  };
  using std::integral_constant;
  if (g.S <= 8)
    join(integral_constant<int, 1>{}, integral_constant<int, 256>{});
  else if (g.S <= 32 || rows > 256)
    join(integral_constant<int, 4>{}, integral_constant<int, 256>{});
  else
    join(integral_constant<int, 4096 / DH>{}, integral_constant<int, 1024>{});
  return hipGetLastError();
}

size_t align256(size_t b) { return (b + 255) & ~static_cast<size_t>(255); }

}  // namespace

size_t attention_workspace_bytes(const srw_attention_t& a) {
  const AttnPlan p = plan_of(a);
  if (p.S == 1) return 0;
  const size_t rows = static_cast<size_t>(a.kv.T) * a.n_heads * p.S;
  return align256(rows * sizeof(float2)) + align256(rows * a.kv.head_dim * sizeof(float));
}

void attention_plan(const srw_attention_t& a, int32_t* rows, int32_t* splits) {
  const AttnPlan p = plan_of(a);
  *rows = p.rows;
  *splits = p.S;
}

hipError_t attention(const srw_attention_t& a, char* ws, hipStream_t s) {
  const AttnPlan p = plan_of(a);
  AttnArgs g{};
  g.kv = kv_view(a.kv);
  g.q = static_cast<const uint16_t*>(a.q);
  g.out = static_cast<uint16_t*>(a.out);
  g.q_token = a.q_token_stride;
  g.q_head = a.q_head_stride;
  g.Hq = a.n_heads;
  g.G = a.n_heads / a.kv.n_kv_heads;
  g.window = a.window;
  g.sinks = a.sinks;
  g.sc = a.scale * 1.4426950408889634f;
  g.S = p.S;
  g.least = p.least;
  if (p.S > 1) {
    g.ml = reinterpret_cast<float2*>(ws);
    g.part = reinterpret_cast<float*>(ws + align256(static_cast<size_t>(a.kv.T) * a.n_heads * p.S * sizeof(float2)));
  }
  auto by = [&](auto kind) {
    constexpr int K = decltype(kind)::value;
    return a.kv.head_dim == 64 ? launch_attention<K, 64>(a, p, g, s) : launch_attention<K, 128>(a, p, g, s);
  };
  switch (a.kv.kind) {
    case SRW_KV_BF16: return by(std::integral_constant<int, SRW_KV_BF16>{});
    case SRW_KV_INT8: return by(std::integral_constant<int, SRW_KV_INT8>{});
    default: return by(std::integral_constant<int, SRW_KV_FP8>{});
  }
}

}  // namespace srw

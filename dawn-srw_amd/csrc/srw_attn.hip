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
// so that m follows the weights that the second product reads.  (l would lose
// keys only where value scales of one row differ by more than 2^100.)
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
// of a tile sees are cleared before the product, since 0 x NaN is NaN.  Where
// the tokens of a tile see different keys, bf16 values that are not finite are
// kept out of the product too and added to the tokens that see them
// (8-bit values are finite; their scales, which may not be, multiply weights,
// which are a token's own).  A token that sees nothing gets zeros.

#include <math.h>

#include "srw_kv.hpp"

namespace srw {
namespace {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kTile = 64;
constexpr float kLazy = 8.f;       // log2 of the largest weight before m is raised
constexpr float kLowest = -1e30f;  // m of a row that has seen nothing

struct AttnArgs {
  KvView kv;
  const uint16_t* q;
  uint16_t* out;
  float* part;    // [S][T Hq][DH]: unnormalised partial outputs
  float2* ml;     // [S][T Hq]: (m, l)
  int64_t q_token, q_head;
  int Hq, G, window, sinks;
  float sc;       // scale log2 e
  int S, per;     // splits of a sequence's tiles, tiles each
};

// The tiles that rows at positions [p_lo, p_hi] see: those of the first
// tokens, then those of the window.
struct Span {
  int lo, hi, sink_tiles, skip, tiles;  // window positions [lo, hi)
  __device__ int key0(int i) const { return (i < sink_tiles ? i : i + skip) * kTile; }
};
__device__ inline Span span_of(const AttnArgs& a, int p_lo, int p_hi) {
  Span s;
  s.hi = p_hi + 1 < a.kv.cap ? p_hi + 1 : a.kv.cap;
  if (s.hi < 0) s.hi = 0;
  s.lo = a.window > 0 && p_lo - a.window + 1 > 0 ? p_lo - a.window + 1 : 0;
  const int sinks = a.sinks < s.lo ? a.sinks : s.lo;
  const int t1 = (s.hi + kTile - 1) / kTile;
  s.sink_tiles = (sinks + kTile - 1) / kTile;
  if (s.sink_tiles > t1) s.sink_tiles = t1;
  const int t0 = s.lo / kTile > s.sink_tiles ? s.lo / kTile : s.sink_tiles;
  s.skip = t0 - s.sink_tiles;
  s.tiles = s.sink_tiles + (t1 > t0 ? t1 - t0 : 0);
  return s;
}

__device__ inline f32x4_t mfma16(u32x4_t a, u32x4_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0,
                                                 0, 0);
}
// c + the sum of two bf16 numbers
__device__ inline float add_bf16x2(uint32_t two, float c) {
  const bf16x2_t ones = {static_cast<__bf16>(1.0f), static_cast<__bf16>(1.0f)};
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, two), ones, c, false);
}
// The low n bits.
__device__ inline uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }
// The tile's keys (bit k: position key0 + k) that a token at position pos sees.
__device__ inline uint64_t seen_of(int pos, int key0, int window, int sinks) {
  const int rel = pos - key0;
  uint64_t see = low_bits(rel + 1);
  if (window > 0) see &= ~low_bits(rel - window + 1) | low_bits(sinks - key0);
  return see;
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
__device__ inline void settled(f32x16_t& a, f32x16_t& b) { asm volatile("s_nop 15\n\ts_nop 3" : "+v"(a), "+v"(b)); }
// A value's scale in the exponent: its log2 and its inverse.  A scale of zero
// stands for values of zero and takes 2^-100; NaN stays.
__device__ inline void in_exponent(float vs, float& lv, float& rv) {
  const float x = vs <= 7.888609052210118e-31f ? 7.888609052210118e-31f : vs;
  lv = __builtin_amdgcn_logf(x);
  rv = __builtin_amdgcn_rcpf(x);
}
// m after a tile whose largest exponent over m (over 0 at first) is mt.
__device__ inline float raised(float m, float mt) {
  if (m == kLowest) return mt == -INFINITY ? kLowest : mt;
  return mt > 0.f ? m + mt : m;
}
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
// Adds to o the values that are not finite of the tile's positions for which
// see(k) holds; value(d) gives the dim of o[d].  Rare: one load each.
template <int N, class See, class Dim, class Acc>
__device__ inline void add_not_finite(const KvView& kv, int64_t b, int h, int head_dim, int key0, See see, Dim dim,
                                      Acc add) {
  for (int k = 0; k < kTile; ++k) {
    const int pg = kv_page(kv, b, key0 + k);
    if (pg < 0 || !see(k)) continue;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(kv.v) +
                          (static_cast<int64_t>(pg) * kv.H + h) * head_dim * kv.P + ((key0 + k) & (kv.P - 1));
#pragma unroll
    for (int i = 0; i < N; ++i) {
      // one address and one load after the other: their registers are the kernel's
      int at = dim(i);
      asm volatile("" : "+v"(at) : : "memory");
      const float x = bf16_to_f32(src[static_cast<int64_t>(at) * kv.P]);
      if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) add(i, x);
    }
  }
}

template <class F, int... J>
__device__ inline void each16(F f, std::integer_sequence<int, J...>) {
  (f(std::integral_constant<int, J>{}), ...);
}
template <class F>
__device__ inline void for16(F f) {
  each16(f, std::make_integer_sequence<int, 16>{});
}

// -- few rows: single tokens, short chunks -----------------------------------
//
// A workgroup takes up to 16 NQ rows (token, head of the group) of one
// sequence and key head; its four waves take every fourth tile of its split,
// each with its own m, l and O, and join in LDS at the end.  Bound by the
// pages' bytes: a wave loads both operands' fragments straight into
// registers, 16 bytes a lane, no barrier in the loop.
template <int KIND, int DH, int NQ>
__global__ __launch_bounds__(256) void attn_rows_kernel(AttnArgs a) {
  constexpr int ES = kv_bytes<KIND>();
  constexpr int NPC = DH * ES / 64;  // 16-byte pieces of a key a lane
  constexpr int NS = DH / 32;        // k-steps of the first product
  constexpr int ND = DH / 16;
  __shared__ float sm[4][16 * NQ], sl[4][16 * NQ];
  __shared__ float so[4][16 * NQ][DH + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane & 15, g = lane >> 4;
  const int split = blockIdx.z, h = blockIdx.y;
  const int64_t b = blockIdx.x;
  const KvSeq sq = kv_seq(a.kv, b);
  const int rows = sq.n * a.G;
  const int P = a.kv.P;
  for (int r0 = 0; r0 < rows; r0 += 16 * NQ) {
    const int r1 = r0 + 16 * NQ < rows ? r0 + 16 * NQ : rows;
    const int p_lo = sq.len - sq.n + r0 / a.G, p_hi = sq.len - sq.n + (r1 - 1) / a.G;
    const Span sp = span_of(a, p_lo, p_hi);
    const int i0 = split * a.per;
    const int i1 = i0 + a.per < sp.tiles ? i0 + a.per : sp.tiles;

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
          mine = have ? static_cast<uint32_t>(seen_of(pos[x], key0, a.window, a.sinks) >> (16 * g)) & 0xffffu : 0u;
          seen |= mine;
        }
        // exponents of the weights, over m (0 while the row has seen nothing)
        float t[16];
        const float mu = m[x] == kLowest ? 0.f : m[x];
        for16([&](auto jt) {
          constexpr int j = decltype(jt)::value;
          const float s = acc[x][j >> 2][j & 3];
          t[j] = KIND == SRW_KV_BF16 ? fmaf(s, a.sc, -mu) : s * row_lane<j>(ksl) + (row_lane<j>(lvl) - mu);
        });
        if (!whole) {
          for16([&](auto jt) {
            constexpr int j = decltype(jt)::value;
            t[j] = only<j>(mine, t[j]);
          });
        }
        float mt = t[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) mt = fmaxf(mt, t[j]);
        if (__any(mt > (m[x] == kLowest ? -INFINITY : kLazy))) {
          auto mx = [](float u, float w) { return fmaxf(u, w); };
          mt = join32(join16(mt, mx), mx);
          const float mn = raised(m[x], mt), back = (mn == kLowest ? 0.f : mn) - mu;
          const float w = __builtin_amdgcn_exp2f(m[x] - mn);
          m[x] = mn;
          l[x] *= w;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int v = 0; v < 4; ++v) o[x][d][v] *= w;
#pragma unroll
          for (int j = 0; j < 16; ++j) t[j] -= back;
        }
#pragma unroll
        for (int j = 0; j < 16; ++j) t[j] = __builtin_amdgcn_exp2f(t[j]);
        if constexpr (KIND != SRW_KV_BF16) {
          if (whole) {
            for16([&](auto jt) {
              constexpr int j = decltype(jt)::value;
              l[x] += t[j] * row_lane<j>(rvl);
            });
          } else {  // the scale of a key that is not seen may be anything
            for16([&](auto jt) {
              constexpr int j = decltype(jt)::value;
              l[x] += __uint_as_float(__float_as_uint(t[j] * row_lane<j>(rvl)) & bit_mask<j>(mine));
            });
          }
        }
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const float p0 = t[8 * st + 2 * u], p1 = t[8 * st + 2 * u + 1];
            const uint32_t hi = pack_bf16(p0, p1);
            pf[x][st][u] = hi;
            pl[x][st][u] = pack_bf16(p0 - lo_f32(hi), p1 - hi_f32(hi));
            if constexpr (KIND == SRW_KV_BF16) l[x] += p0 + p1;
          }
      }
      bool odd = false;  // a value is not finite
      if (!whole && KIND != SRW_KV_INT8) {
        for (int w = 1; w < 16; w <<= 1) seen |= __shfl_xor(seen, w);  // over the columns: keys that some row sees
        u16x2_t most = {0, 0};
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
        if (KIND == SRW_KV_BF16 && p_lo != p_hi) {
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int j = 0; j < ES; ++j) most = most16(most, vf[d][j]);
          odd = __any(not_finite(most));
          if (odd) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
              for (int j = 0; j < ES; ++j) vf[d][j] = finite16(vf[d][j]);
          }
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
      if (KIND == SRW_KV_BF16 && odd) {
#pragma unroll
        for (int x = 0; x < NQ; ++x)
          add_not_finite<4 * ND>(
              a.kv, b, h, DH, key0,
              [&](int k) { return seen_of(pos[x], key0, a.window, a.sinks) >> k & 1; },
              [&](int i) { return 16 * (i / 4) + 4 * g + i % 4; }, [&](int i, float v) { o[x][i / 4][i % 4] += v; });
      }
    }

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
          const float e = sm[w][r] == mm ? 1.f : __builtin_amdgcn_exp2f(sm[w][r] - mm);
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
    __syncthreads();
  }
}

// Joins the splits: a workgroup a row, in groups of DH / 4 lanes that take the
// splits in turn, each with all its loads in flight, and join in LDS.
template <int DH>
__global__ __launch_bounds__(256) void attn_join_kernel(const float* part, const float2* ml, uint16_t* out,
                                                        int64_t rows, int S) {
  constexpr int L = DH / 4, N = 256 / L;  // lanes a group, groups
  __shared__ float sm[N], sl[N];
  __shared__ f32x4_t so[N][L];
  const int grp = threadIdx.x / L, c = threadIdx.x % L;
  const int64_t row = blockIdx.x;
  float m = kLowest, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  constexpr int U = 4;
  for (int s0 = grp; s0 < S; s0 += N * U) {
    float2 x[U];
    f32x4_t v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int s = s0 + N * u < S ? s0 + N * u : s0;
      x[u] = ml[s * rows + row];
      v[u] = *reinterpret_cast<const f32x4_t*>(part + (s * rows + row) * DH + 4 * c);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // a split without visible keys wrote no output
      if (s0 + N * u >= S || x[u].y == 0.f) continue;
      const float mn = fmaxf(m, x[u].x);
      const float e0 = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      const float e1 = x[u].x == mn ? 1.f : __builtin_amdgcn_exp2f(x[u].x - mn);
      m = mn;
      l = l * e0 + x[u].y * e1;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = o[k] * e0 + v[u][k] * e1;
    }
  }
  if (c == 0) {
    sm[grp] = m;
    sl[grp] = l;
  }
  so[grp][c] = o;
  __syncthreads();
  if (grp != 0) return;
  float mm = sm[0], ll = 0.f;
#pragma unroll
  for (int g = 1; g < N; ++g) mm = fmaxf(mm, sm[g]);
  o = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < N; ++g) {
    const float e = sm[g] == mm ? 1.f : __builtin_amdgcn_exp2f(sm[g] - mm);
    ll += sl[g] * e;
#pragma unroll
    for (int k = 0; k < 4; ++k) o[k] += so[g][c][k] * e;
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  *reinterpret_cast<uint2*>(out + row * DH + 4 * c) =
      make_uint2(pack_bf16(o[0] * inv, o[1] * inv), pack_bf16(o[2] * inv, o[3] * inv));
}

// -- many rows: chunks of prompts ---------------------------------------------
//
// 128 rows a workgroup, 32 a wave; a tile's keys and values go through LDS
// once for the four waves, two stages deep.  bf16 pages are copied there
// directly (global_load_lds), 8-bit ones are widened on the way.  16-byte
// pieces of a row are XOR-swizzled by the row so that 16 lanes' fragment
// reads cover all banks.
template <int DH> __device__ inline int k_swz(int row) { return DH == 64 ? (row >> 1) & 7 : row & 15; }
__device__ inline int v_swz(int row) { return (row >> 1) & 7; }

template <int KIND, int DH>
__global__ __launch_bounds__(256, 2) void attn_tile_kernel(AttnArgs a) {
  constexpr int ES = kv_bytes<KIND>();
  constexpr int NS = DH / 16, ND = DH / 32;
  constexpr int NP = DH / 8;                     // pieces of a key row
  constexpr int kStage = kTile * DH * 2;         // bytes of a tile's keys (or values) in LDS
  constexpr int NI = kStage / 4096;              // 16-byte pieces a thread of either
  constexpr bool Q8 = KIND != SRW_KV_BF16;
  __shared__ __align__(16) char kl[2][kStage];
  __shared__ __align__(16) char vl[2][kStage];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane & 31, hf = lane >> 5;
  const int h = blockIdx.y, split = blockIdx.z;
  const int P = a.kv.P;

  // sequence and row tile; the last tiles, which see most, come first
  int64_t b = 0;
  int rt = blockIdx.x;
  if (a.kv.cu) {
    auto start = [&](int64_t i) { return (static_cast<int64_t>(a.kv.cu[i]) * a.G >> 7) + i; };
    b = kv_find(a.kv.B, blockIdx.x, start);
    rt = static_cast<int>(blockIdx.x - start(b));
  } else {
    const int per = (a.G + 127) / 128;
    b = blockIdx.x / per;
    rt = blockIdx.x % per;
  }
  b = __builtin_amdgcn_readfirstlane(static_cast<int>(b));
  const KvSeq sq = kv_seq(a.kv, b);
  const int rows = sq.n * a.G;
  const int rts = (rows + 127) / 128;
  if (rt < 0 || rt >= rts) return;
  rt = rts - 1 - rt;
  const int r0 = rt * 128, r1 = r0 + 128 < rows ? r0 + 128 : rows;
  const Span sp = span_of(a, sq.len - sq.n + r0 / a.G, sq.len - sq.n + (r1 - 1) / a.G);
  const int i0 = split * a.per;
  const int i1 = i0 + a.per < sp.tiles ? i0 + a.per : sp.tiles;

  // this wave's rows
  const int w0 = r0 + 32 * wave, w1 = w0 + 32 < r1 ? w0 + 32 : r1;
  const bool active = w0 < r1;
  const int p_lo = sq.len - sq.n + w0 / a.G, p_hi = sq.len - sq.n + (w1 - 1) / a.G;
  const int fr = w0 + col;
  const bool in = fr < r1;
  const int tok = in ? fr / a.G : 0;
  const int head = h * a.G + (in ? fr - tok * a.G : 0);
  const int pos = in ? sq.len - sq.n + tok : -1;
  u32x4_t q[NS];
  {
    const uint16_t* src = a.q + (sq.row0 + tok) * a.q_token + head * a.q_head + 8 * hf;
#pragma unroll
    for (int s = 0; s < NS; ++s) q[s] = in ? ld16(src + 16 * s) : u32x4_t{0, 0, 0, 0};
  }
  float m = kLowest, l = 0.f;
  f32x16_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.f;

  // A tile's position in its pages: slot of its first key (pages of 64 and more
  // hold whole tiles; smaller ones start with one), then the slot of key k.
  const int64_t page_bytes = static_cast<int64_t>(a.kv.H) * P * DH * ES, head_at = static_cast<int64_t>(h) * P * DH * ES;
  const char* kbase = a.kv.k + head_at;
  const char* vbase = a.kv.v + head_at;
  // pages of tile i: lane c holds that of positions key0 + 16 (c & 3)
  auto pages_of = [&](int i) {
    const int at = sp.key0(i) + 16 * (lane & 3);
    return at < sp.hi ? kv_page(a.kv, b, at) : -1;
  };
  u32x4_t rk[Q8 ? NI / 2 : 1], rv[Q8 ? NI / 2 : 1];  // 8-bit tiles on their way
  auto fetch = [&](int i, int ids, int stage) {
    const int slot0 = sp.key0(i) & (P - 1);
    const int safe = ids < 0 ? 0 : ids;
    if constexpr (!Q8) {
      // pieces n of a lane: keys of one group of 16 for the whole wave
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int first = (wave * NI + n) * 64;      // piece of lane 0
        const int row = (first + lane) / NP, pc = ((first + lane) % NP) ^ k_swz<DH>(row);
        const int64_t pg = __builtin_amdgcn_readlane(safe, (first / NP) >> 4);
        g2lds16(kbase + pg * page_bytes + slot0 * (DH * ES) + ((row & (P - 1)) * DH + 8 * pc) * ES, kl[stage] + 16 * first);
      }
      // values: positions 8 pc .. of a dim, pc = (lane & 7) ^ (lane >> 4) ^ 4 (n & 1)
      const int pe = (lane & 7) ^ (lane >> 4);
      const int64_t pg[2] = {__shfl(safe, pe >> 1), __shfl(safe, (pe ^ 4) >> 1)};
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int first = (wave * NI + n) * 64;
        const int row = (first + lane) / 8, pc = pe ^ (4 * (n & 1));
        g2lds16(vbase + pg[n & 1] * page_bytes + (row * P + slot0 + ((8 * pc) & (P - 1))) * ES, vl[stage] + 16 * first);
      }
    } else {
      // a thread's 16 codes: of keys, 16 dims of a position (the wave's
      // positions in one group of 16); of values, 16 positions of a dim
#pragma unroll
      for (int n = 0; n < NI / 2; ++n) {
        const int at = n * 256 + threadIdx.x;
        const int row = at / (NP / 2), pc = at % (NP / 2);
        const int64_t pg = __builtin_amdgcn_readlane(safe, (n * 256 + wave * 64) / (NP / 2) >> 4);
        rk[n] = ld16(kbase + pg * page_bytes + slot0 * DH + ((row & (P - 1)) * DH + 16 * pc));
      }
      const char* vsrc = vbase + safe * page_bytes + slot0 + ((16 * (lane & 3)) & (P - 1));
#pragma unroll
      for (int n = 0; n < NI / 2; ++n) rv[n] = ld16(vsrc + (n * 64 + (threadIdx.x >> 2)) * P);
    }
  };
  auto settle = [&](int stage) {  // 8 bits: widen into LDS
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < NI / 2; ++n) {
        const int at = n * 256 + threadIdx.x;
        const int row = at / (NP / 2), pc = at % (NP / 2);
        const int vrow = at / 4, vpc = at % 4;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          *reinterpret_cast<u32x4_t*>(kl[stage] + row * (DH * 2) + 16 * ((2 * pc + u) ^ k_swz<DH>(row))) =
              widen8<KIND>(rk[n][2 * u], rk[n][2 * u + 1]);
          *reinterpret_cast<u32x4_t*>(vl[stage] + vrow * 128 + 16 * ((2 * vpc + u) ^ v_swz(vrow))) =
              widen8<KIND>(rv[n][2 * u], rv[n][2 * u + 1]);
        }
      }
    }
  };
  // scales of the lane's keys: of its 32 score registers (kb, v), register
  // kb of lane v of a row of 16 holds that of key 32 kb + 16 (v / 8) + 8 hf + v % 8
  float ksl[2], lvl[2], rvl[2], ksn[2], vsn[2];
  auto scales = [&](int i, int ids) {
    if constexpr (Q8) {
      const int slot0 = sp.key0(i) & (P - 1);
      const int safe = ids < 0 ? 0 : ids;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int k = 32 * kb + 16 * (lane >> 3 & 1) + 8 * hf + (lane & 7);
        const int64_t pg = lane & 8 ? __builtin_amdgcn_readlane(safe, 2 * kb + 1) : __builtin_amdgcn_readlane(safe, 2 * kb);
        const int64_t at = (pg * a.kv.H + h) * P + slot0 + (k & (P - 1));
        ksn[kb] = a.kv.ks[at];
        vsn[kb] = a.kv.vs[at];
      }
    }
  };

  int ids = i0 < i1 ? pages_of(i0) : -1, idn = -1;
  if (i0 < i1) {
    fetch(i0, ids, 0);
    scales(i0, ids);
    if (i0 + 1 < i1) idn = pages_of(i0 + 1);
  }
  for (int i = i0; i < i1; ++i) {
    const int stage = (i - i0) & 1;
    settle(stage);
    wait_vm0();
    __syncthreads();
    const int cur = ids;
    if constexpr (Q8) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        ksl[kb] = ksn[kb] * a.sc;
        in_exponent(vsn[kb], lvl[kb], rvl[kb]);
      }
    }
    if (i + 1 < i1) {
      fetch(i + 1, idn, stage ^ 1);
      scales(i + 1, idn);
      ids = idn;
      if (i + 2 < i1) idn = pages_of(i + 2);
    }
    const int key0 = sp.key0(i);
    if (!active || key0 > p_hi) continue;

    f32x16_t acc[2];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
      for (int v = 0; v < 16; ++v) acc[kb][v] = 0.f;
      // row m = 16 j + 8 u + 4 w + x of the product holds key 16 j + 8 w + 4 u + x
      const int row = 32 * kb + (col & 19) + ((col & 4) << 1) + ((col & 8) >> 1);
      const char* src = kl[stage] + row * (DH * 2);
#pragma unroll
      for (int s = 0; s < NS; ++s) acc[kb] = mfma(ld16(src + 16 * ((2 * s + hf) ^ k_swz<DH>(row))), q[s], acc[kb]);
    }
    // positions of the tile that some row of the workgroup sees
    uint64_t keys = low_bits(sp.hi - key0);
    {
      const uint64_t have = __ballot(cur >= 0) & 15;
      if (have != 15) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
          if (!(have >> u & 1)) keys &= ~(0xffffull << (16 * u));
      }
      if (key0 < sp.lo) keys &= ~low_bits(sp.lo - key0) | low_bits(a.sinks - key0);
    }
    const bool whole = keys == ~0ull && key0 + kTile - 1 <= p_lo &&
                       (a.window == 0 || key0 > p_hi - a.window || key0 + kTile <= a.sinks);
    // bits 32 kb + 16 (v / 8) + v % 8: the lane's row sees the key of its register (kb, v)
    uint32_t mine[2] = {~0u, ~0u};
    if (!whole) {
      const uint64_t see = (seen_of(pos, key0, a.window, a.sinks) & keys) >> (8 * hf);
      mine[0] = static_cast<uint32_t>(see);
      mine[1] = static_cast<uint32_t>(see >> 32);
    }
    // exponents of the weights, over m (0 while the row has seen nothing)
    float t[2][16];
    const float mu = m == kLowest ? 0.f : m;
    if constexpr (Q8) {
      settled(acc[0], acc[1]);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        float s[16];
        for16([&](auto vt) {
          constexpr int v = decltype(vt)::value;
          s[v] = acc[kb][v];
          t[kb][v] = row_lane<v>(lvl[kb]) - mu;
        });
        fma_lanes8<0>(t[kb], ksl[kb], s);
        fma_lanes8<8>(t[kb] + 8, ksl[kb], s + 8);
      }
    } else {
#pragma unroll
      for (int v = 0; v < 32; ++v) t[v >> 4][v & 15] = fmaf(acc[v >> 4][v & 15], a.sc, -mu);
    }
    if (!whole) {
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
        for16([&](auto vt) {
          constexpr int v = decltype(vt)::value;
          t[kb][v] = only<16 * (v / 8) + v % 8>(mine[kb], t[kb][v]);
        });
    }
    float mt = t[0][0];
#pragma unroll
    for (int v = 1; v < 32; ++v) mt = fmaxf(mt, t[v >> 4][v & 15]);
    if (__any(mt > (m == kLowest ? -INFINITY : kLazy))) {
      mt = join32(mt, [](float u, float w) { return fmaxf(u, w); });
      const float mn = raised(m, mt), back = (mn == kLowest ? 0.f : mn) - mu;
      const float w = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= w;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= w;
#pragma unroll
      for (int v = 0; v < 32; ++v) t[v >> 4][v & 15] -= back;
    }
    u32x4_t pf[4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      for16([&](auto vt) {
        constexpr int v = decltype(vt)::value;
        t[kb][v] = __builtin_amdgcn_exp2f(t[kb][v]);
      });
      if constexpr (Q8) {
        if (whole) {
          sum_lanes16(l, rvl[kb], t[kb]);
        } else {  // the scale of a key that is not seen may be anything
          for16([&](auto vt) {
            constexpr int v = decltype(vt)::value;
            l += __uint_as_float(__float_as_uint(row_lane<v>(rvl[kb]) * t[kb][v]) &
                                 bit_mask<16 * (v / 8) + v % 8>(mine[kb]));
          });
        }
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float p0 = t[kb][8 * j + 2 * u], p1 = t[kb][8 * j + 2 * u + 1];
          pf[2 * kb + j][u] = pack_bf16(p0, p1);
          if constexpr (!Q8) l = add_bf16x2(pf[2 * kb + j][u], l);
        }
    }
    bool odd = false;  // a value is not finite
    if (KIND == SRW_KV_BF16 && !whole) {
      u16x2_t most = {0, 0};
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int row = 32 * d + col;
          most = most16(most, ld16(vl[stage] + row * 128 + 16 * ((2 * j + hf) ^ v_swz(row))));
        }
      odd = __any(not_finite(most));
    }
#pragma unroll
    for (int d = 0; d < ND; ++d) {
      const int row = 32 * d + col;
      const char* src = vl[stage] + row * 128;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        u32x4_t vb = ld16(src + 16 * ((2 * j + hf) ^ v_swz(row)));
        if (KIND != SRW_KV_INT8 && keys != ~0ull) {
          const uint32_t bits = static_cast<uint32_t>(keys >> (16 * j + 8 * hf)) & 0xffu;
#pragma unroll
          for (int u = 0; u < 4; ++u)
            vb[u] &= (bits >> (2 * u) & 1 ? 0x0000ffffu : 0u) | (bits >> (2 * u + 1) & 1 ? 0xffff0000u : 0u);
        }
        if (KIND == SRW_KV_BF16 && odd) vb = finite16(vb);
        o[d] = mfma(vb, pf[j], o[d]);
      }
    }
    if (KIND == SRW_KV_BF16 && odd)
      add_not_finite<16 * ND>(
          a.kv, b, h, DH, key0,
          [&](int k) { return seen_of(pos, key0, a.window, a.sinks) >> k & 1; },
          [&](int i) { return 32 * (i / 16) + 8 * (i % 16 / 4) + 4 * hf + i % 4; },
          [&](int i, float v) { o[i / 16][i % 16] += v; });
  }
  if (!active) return;
  l = join32(l, [](float u, float w) { return u + w; });
  if (!in) return;
  const int64_t row = (sq.row0 + tok) * a.Hq + head;
  if (a.S == 1) {
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
      for (int v = 0; v < 16; v += 4)
        *reinterpret_cast<uint2*>(a.out + row * DH + 32 * d + 2 * v + 4 * hf) =
            make_uint2(pack_bf16(o[d][v] * inv, o[d][v + 1] * inv), pack_bf16(o[d][v + 2] * inv, o[d][v + 3] * inv));
  } else {
    const int64_t at = split * (a.kv.T * a.Hq) + row;
    if (l != 0.f) {
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; v += 4)
          *reinterpret_cast<f32x4_t*>(a.part + at * DH + 32 * d + 2 * v + 4 * hf) =
              f32x4_t{o[d][v], o[d][v + 1], o[d][v + 2], o[d][v + 3]};
    }
    if (hf == 0) a.ml[at] = make_float2(m, l);
  }
}

// How a call runs: the kernel, and in how many splits a sequence's tiles.
struct AttnPlan {
  int rows;       // rows a workgroup: 16, 32 (attn_rows_kernel) or 128
  int64_t groups; // workgroups of one split
  int S, per;
};

AttnPlan plan_of(const srw_attention_t& a) {
  AttnPlan p{};
  const int64_t G = a.n_heads / a.kv.n_kv_heads, B = a.kv.B, T = a.kv.T, H = a.kv.n_kv_heads;
  const int64_t most = !a.kv.cu ? 1 : a.max_new > 0 ? a.max_new : T;
  p.rows = most * G <= 16 ? 16 : most * G <= 32 ? 32 : 128;
  int64_t tiles = a.kv.table_width * a.kv.page_size / kTile + 1;  // of a row, at most
  if (a.window > 0) {
    const int64_t w = (a.window + most + kTile - 1) / kTile + 1 + (a.sinks + kTile - 1) / kTile;
    tiles = w < tiles ? w : tiles;
  }
  if (p.rows < 128) {
    p.groups = B * H;
    // about 2048 workgroups in all, of four tiles (one a wave) at least
    int64_t per = (tiles * p.groups + 2047) / 2048;
    per = per < 16 ? 16 : (per + 3) / 4 * 4;
    p.per = static_cast<int>(per < tiles ? per : tiles);
  } else {
    p.groups = (!a.kv.cu ? B * ((G + 127) / 128) : T * G / 128 + B) * H;
    int64_t per = (tiles * p.groups + 511) / 512;
    per = per < 8 ? 8 : per;
    p.per = static_cast<int>(per < tiles ? per : tiles);
  }
  if (p.per < 1) p.per = 1;
  p.S = static_cast<int>((tiles + p.per - 1) / p.per);
  return p;
}

template <int KIND, int DH>
hipError_t launch_attention(const srw_attention_t& a, const AttnPlan& pl, AttnArgs& g, hipStream_t s) {
  if (pl.rows < 128) {
    const dim3 grid(static_cast<unsigned>(a.kv.B), static_cast<unsigned>(g.kv.H), static_cast<unsigned>(g.S));
    if (pl.rows == 16)
      hipLaunchKernelGGL((attn_rows_kernel<KIND, DH, 1>), grid, dim3(256), 0, s, g);
    else
      hipLaunchKernelGGL((attn_rows_kernel<KIND, DH, 2>), grid, dim3(256), 0, s, g);
  } else {
    const dim3 grid(static_cast<unsigned>(pl.groups / g.kv.H), static_cast<unsigned>(g.kv.H),
                    static_cast<unsigned>(g.S));
    hipLaunchKernelGGL((attn_tile_kernel<KIND, DH>), grid, dim3(256), 0, s, g);
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || g.S == 1) return e;
  const int64_t rows = a.kv.T * a.n_heads;
  hipLaunchKernelGGL(attn_join_kernel<DH>, dim3(static_cast<unsigned>(rows)), dim3(256), 0, s, g.part, g.ml, g.out, rows,
                     g.S);
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
  g.per = p.per;
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

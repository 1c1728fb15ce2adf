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
// 8-bit pages: codes are bf16 numbers exactly, so the products run on the
// codes; a key's scale multiplies its score and a value's its weight, both in
// float32.  Weights are rounded to bf16 once (after their scale; the sum l
// takes them unrounded), as the matrix cores read them; everything else is
// float32.
//
// m is raised only when a score passes it by more than 2^8: weights then stay
// under 2^8 and their sum far inside float32, and the accumulators are
// rescaled a few times a row instead of once a tile.
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
constexpr float kLazy = 8.f;  // log2 of the largest weight before m is raised

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
      const float x = bf16_to_f32(src[static_cast<int64_t>(dim(i)) * kv.P]);
      if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) add(i, x);
    }
  }
}

// v times the value of lane J of v2's row of 16, for J = 0 .. 15 in turn.
template <int J>
__device__ inline float by_lane(float v, float of) {
  return v * row_lane<J>(of);
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
      m[x] = -INFINITY;
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
      float ksl = a.sc, vsl = 1.f;
      if constexpr (KIND != SRW_KV_BF16) {
        ksl = a.kv.ks[hv * P + (kv & (P - 1)) + col] * a.sc;
        vsl = a.kv.vs[hv * P + (kv & (P - 1)) + col];
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
      uint32_t seen = 0xffffu;  // bit 4 t + v: some row of the tile sees the lane's key
      if (!whole) seen = 0;
      u32x4_t pf[NQ][2];
#pragma unroll
      for (int x = 0; x < NQ; ++x) {
        float s[16];
        for16([&](auto jt) {
          constexpr int j = decltype(jt)::value;
          s[j] = KIND == SRW_KV_BF16 ? acc[x][j >> 2][j & 3] * a.sc : by_lane<j>(acc[x][j >> 2][j & 3], ksl);
        });
        if (!whole) {
          const int rel = pos[x] - kv;  // key kv + j: j <= rel, j > rel - window or j < sinks - kv
          const int below = a.window > 0 ? rel - a.window : -kTile - 1, first = a.sinks - kv;
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const bool see = have && j <= rel && (j > below || j < first);
            s[j] = see ? s[j] : -INFINITY;
            seen |= see ? 1u << j : 0u;
          }
        }
        float mt = s[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) mt = fmaxf(mt, s[j]);
        if (__any(mt > m[x] + kLazy)) {
          auto mx = [](float u, float w) { return fmaxf(u, w); };
          mt = join32(join16(mt, mx), mx);
          const float mn = fmaxf(m[x], mt);
          const float w = m[x] == mn ? 1.f : __builtin_amdgcn_exp2f(m[x] - mn);
          m[x] = mn;
          l[x] *= w;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int v = 0; v < 4; ++v) o[x][d][v] *= w;
        }
        const float ms = m[x] == -INFINITY ? 0.f : m[x];
        float p[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          p[j] = __builtin_amdgcn_exp2f(s[j] - ms);
          l[x] += p[j];
        }
        if constexpr (KIND != SRW_KV_BF16) {
          for16([&](auto jt) {
            constexpr int j = decltype(jt)::value;
            const float w = by_lane<j>(p[j], vsl);
            p[j] = whole || s[j] != -INFINITY ? w : 0.f;
          });
        }
#pragma unroll
        for (int st = 0; st < 2; ++st)
#pragma unroll
          for (int u = 0; u < 4; ++u) pf[x][st][u] = pack_bf16(p[8 * st + 2 * u], p[8 * st + 2 * u + 1]);
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
          for (int x = 0; x < NQ; ++x) o[x][d] = mfma16(vb, pf[x][st], o[x][d]);
        }
      }
      if (KIND == SRW_KV_BF16 && odd) {
#pragma unroll
        for (int x = 0; x < NQ; ++x)
          add_not_finite<4 * ND>(
              a.kv, b, h, DH, key0,
              [&](int k) {
                return key0 + k <= pos[x] &&
                       (a.window == 0 || key0 + k > pos[x] - a.window || key0 + k < a.sinks);
              },
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
          // a wave without visible keys has m = -inf and l = 0
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

// Joins the splits: one wave a row, DH / 64 dims a lane.
template <int DH>
__global__ __launch_bounds__(256) void attn_join_kernel(const float* part, const float2* ml, uint16_t* out,
                                                        int64_t rows, int S) {
  constexpr int N = DH / 64;
  const int lane = threadIdx.x & 63;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
  float mm = -INFINITY;
  for (int s = lane; s < S; s += 64) mm = fmaxf(mm, ml[s * rows + row].x);
  mm = wave_max(mm);
  float ll = 0.f, o[N] = {};
  for (int s = 0; s < S; ++s) {
    const float2 x = ml[s * rows + row];
    if (x.y == 0.f) continue;  // no visible keys there, and no output written
    const float e = x.x == mm ? 1.f : __builtin_amdgcn_exp2f(x.x - mm);
    ll += x.y * e;
#pragma unroll
    for (int d = 0; d < N; ++d) o[d] += part[(s * rows + row) * DH + lane * N + d] * e;
  }
  const float inv = ll == 0.f ? 0.f : 1.f / ll;
  if constexpr (N == 2)
    *reinterpret_cast<uint32_t*>(out + row * DH + 2 * lane) = pack_bf16(o[0] * inv, o[1] * inv);
  else
    out[row * DH + lane] = f32_to_bf16_bits(o[0] * inv);
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
  float m = -INFINITY, l = 0.f;
  f32x16_t o[ND];
#pragma unroll
  for (int d = 0; d < ND; ++d)
#pragma unroll
    for (int v = 0; v < 16; ++v) o[d][v] = 0.f;

  // pages of tile i: lane c holds that of positions key0 + 16 (c & 3)
  auto pages_of = [&](int i) {
    const int at = sp.key0(i) + 16 * (lane & 3);
    return at < sp.hi ? kv_page(a.kv, b, at) : -1;
  };
  u32x4_t rk[Q8 ? NI / 2 : 1], rv[Q8 ? NI / 2 : 1];  // 8-bit tiles on their way
  auto fetch = [&](int i, int ids, int stage) {
    const int key0 = sp.key0(i);
    const int safe = ids < 0 ? 0 : ids;
    if constexpr (!Q8) {
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int first = (wave * NI + n) * 64;      // piece of lane 0
        const int row = (first + lane) / NP, pc = ((first + lane) % NP) ^ k_swz<DH>(row);
        const int64_t pg = __builtin_amdgcn_readlane(safe, (first / NP) >> 4);
        g2lds16(a.kv.k + (((pg * a.kv.H + h) * P + ((key0 + row) & (P - 1))) * DH + 8 * pc) * ES, kl[stage] + 16 * first);
      }
#pragma unroll
      for (int n = 0; n < NI; ++n) {
        const int first = (wave * NI + n) * 64;
        const int row = (first + lane) / 8, pc = ((first + lane) % 8) ^ v_swz(row);
        const int64_t pg = __shfl(safe, pc >> 1);
        g2lds16(a.kv.v + (((pg * a.kv.H + h) * DH + row) * P + ((key0 + 8 * pc) & (P - 1))) * ES, vl[stage] + 16 * first);
      }
    } else {
      // a thread's 16 codes: of keys, 16 dims of a position; of values, 16
      // positions of a dim
#pragma unroll
      for (int n = 0; n < NI / 2; ++n) {
        const int at = n * 256 + threadIdx.x;
        const int row = at / (NP / 2), pc = at % (NP / 2);
        const int64_t pg = __shfl(safe, row >> 4);
        rk[n] = ld16(a.kv.k + ((pg * a.kv.H + h) * P + ((key0 + row) & (P - 1))) * DH + 16 * pc);
        const int vrow = at / 4, vpc = at % 4;
        const int64_t vg = __shfl(safe, vpc);
        rv[n] = ld16(a.kv.v + ((vg * a.kv.H + h) * DH + vrow) * P + ((key0 + 16 * vpc) & (P - 1)));
      }
    }
  };
  auto settle = [&](int stage) {  // 8 bits: widen into LDS
    if constexpr (Q8) {
#pragma unroll
      for (int n = 0; n < NI / 2; ++n) {
        const int at = n * 256 + threadIdx.x;
        const int row = at / (NP / 2), pc = at % (NP / 2);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          *reinterpret_cast<u32x4_t*>(kl[stage] + row * (DH * 2) + 16 * ((2 * pc + u) ^ k_swz<DH>(row))) =
              widen8<KIND>(rk[n][2 * u], rk[n][2 * u + 1]);
          const int vrow = at / 4, vpc = at % 4;
          *reinterpret_cast<u32x4_t*>(vl[stage] + vrow * 128 + 16 * ((2 * vpc + u) ^ v_swz(vrow))) =
              widen8<KIND>(rv[n][2 * u], rv[n][2 * u + 1]);
        }
      }
    }
  };
  // scales of the lane's keys: of its 32 score registers (kb, v), register
  // kb of lane v of a row of 16 holds that of key 32 kb + 16 (v / 8) + 8 hf + v % 8
  float ksl[2], vsl[2], ksn[2], vsn[2];
  auto scales = [&](int i, int ids) {
    if constexpr (Q8) {
      const int key0 = sp.key0(i);
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
        const int k = 32 * kb + 8 * (lane & 8 ? 2 : 0) + 8 * hf + (lane & 7);
        const int64_t pg = __shfl(ids < 0 ? 0 : ids, k >> 4);
        const int64_t at = (pg * a.kv.H + h) * P + ((key0 + k) & (P - 1));
        ksn[kb] = a.kv.ks[at] * a.sc;
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
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      ksl[kb] = ksn[kb];
      vsl[kb] = vsn[kb];
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
    // positions of the tile that some row of the workgroup can see
    uint64_t keys = ~0ull;
    {
      const uint64_t have = __ballot(cur >= 0);
      if ((have & 15) != 15) {
        keys = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) keys |= (have >> u & 1) ? 0xffffull << (16 * u) : 0ull;
      }
      if (sp.hi - key0 < kTile) keys &= (1ull << (sp.hi - key0)) - 1;  // hi > key0
      if (key0 < sp.lo) {
        const int below = sp.lo - key0, first = a.sinks - key0;
        uint64_t drop = below >= kTile ? ~0ull : (1ull << below) - 1;
        if (first > 0) drop &= first >= kTile ? 0ull : ~((1ull << first) - 1);
        keys &= ~drop;
      }
    }
    const bool whole = keys == ~0ull && key0 + kTile - 1 <= p_lo &&
                       (a.window == 0 || key0 > p_hi - a.window || key0 + kTile <= a.sinks);
    float s[2][16];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb)
      for16([&](auto vt) {
        constexpr int v = decltype(vt)::value;
        s[kb][v] = Q8 ? by_lane<v>(acc[kb][v], ksl[kb]) : acc[kb][v] * a.sc;
      });
    if (!whole) {
      const uint64_t mine = keys >> (8 * hf);
      const int rel = pos - key0 - 8 * hf, below = a.window > 0 ? rel - a.window : -2 * kTile,
                first = a.sinks - key0 - 8 * hf;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int v = 0; v < 16; ++v) {
          const int k = 32 * kb + 16 * (v / 8) + v % 8;
          const bool see = (mine >> k & 1) && k <= rel && (k > below || k < first);
          s[kb][v] = see ? s[kb][v] : -INFINITY;
        }
    }
    float mt = s[0][0];
#pragma unroll
    for (int v = 1; v < 32; ++v) mt = fmaxf(mt, s[v >> 4][v & 15]);
    if (__any(mt > m + kLazy)) {
      mt = join32(mt, [](float u, float w) { return fmaxf(u, w); });
      const float mn = fmaxf(m, mt);
      const float w = m == mn ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= w;
#pragma unroll
      for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int v = 0; v < 16; ++v) o[d][v] *= w;
    }
    const float ms = m == -INFINITY ? 0.f : m;
    u32x4_t pf[4];
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      float p[16];
#pragma unroll
      for (int v = 0; v < 16; ++v) {
        p[v] = __builtin_amdgcn_exp2f(s[kb][v] - ms);
        l += p[v];
      }
      if constexpr (Q8) {
        for16([&](auto vt) {
          constexpr int v = decltype(vt)::value;
          const float w = by_lane<v>(p[v], vsl[kb]);
          p[v] = whole || s[kb][v] != -INFINITY ? w : 0.f;
        });
      }
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int u = 0; u < 4; ++u) pf[2 * kb + j][u] = pack_bf16(p[8 * j + 2 * u], p[8 * j + 2 * u + 1]);
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
          [&](int k) {
            return key0 + k <= pos && (a.window == 0 || key0 + k > pos - a.window || key0 + k < a.sinks);
          },
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
  hipLaunchKernelGGL(attn_join_kernel<DH>, dim3(static_cast<unsigned>((rows + 3) / 4)), dim3(256), 0, s, g.part, g.ml,
                     g.out, rows, g.S);
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

// srw_kv.hpp -- the paged key/value cache as its kernels see it (srw_kv.hip,
// srw_attn.hip).
//
// Pages hold page_size positions of every key/value head.  Keys lie position
// by position (k[page][head][slot][dim]), values dimension by dimension
// (v[page][head][dim][slot]): a lane of either of the attention's matrix
// products then reads its operand -- eight dims of one key, eight keys of one
// value dim -- from consecutive bytes, and nothing is transposed on the way.
// Groups of 16 consecutive positions are aligned and never cross a page.
#pragma once

#include "srw_internal.hpp"
#include "srw_mfma_util.hpp"

namespace srw {

constexpr int kKvGroup = 16;  // positions that share a page whatever its size

template <int KIND> constexpr int kv_bytes() { return KIND == SRW_KV_BF16 ? 2 : 1; }

struct KvView {
  char* k;
  char* v;
  float* ks;
  float* vs;
  const int32_t* table;
  const int32_t* lens;
  const int32_t* cu;
  int64_t B, T, n_pages, tstride;
  int32_t cap;      // positions a table row can name
  int32_t H, P, logP;
};

inline KvView kv_view(const srw_kv_t& c) {
  KvView p{};
  p.k = static_cast<char*>(c.k);
  p.v = static_cast<char*>(c.v);
  p.ks = c.k_scale;
  p.vs = c.v_scale;
  p.table = c.table;
  p.lens = c.lens;
  p.cu = c.cu;
  p.B = c.B;
  p.T = c.T;
  p.n_pages = c.n_pages;
  p.tstride = c.table_stride;
  p.H = c.n_kv_heads;
  p.P = c.page_size;
  p.cap = c.n_pages > 0 ? static_cast<int32_t>(c.table_width * c.page_size) : 0;
  while ((1 << p.logP) < p.P) ++p.logP;
  return p;
}

// A sequence's new tokens: packed rows [row0, row0 + n) at positions
// [len - n, len).  Whatever the device arrays hold, the rows lie in [0, T);
// positions outside [0, cap) are left out by the kernels.
struct KvSeq {
  int64_t row0;
  int n, len;
};
__device__ inline KvSeq kv_seq(const KvView& p, int64_t b) {
  int64_t r0 = b, r1 = b + 1;
  if (p.cu) {
    r0 = p.cu[b];
    r1 = p.cu[b + 1];
  }
  r0 = r0 < 0 ? 0 : (r0 > p.T ? p.T : r0);
  r1 = r1 < r0 ? r0 : (r1 > p.T ? p.T : r1);
  int len = p.lens[b];
  // (positions stay below 2^31 - 2^16 so that tiles past the end do not wrap)
  len = len < 0 ? 0 : (len > 0x7fff0000 ? 0x7fff0000 : len);
  return KvSeq{r0, static_cast<int>(r1 - r0), len};
}

// The positions base + [first, last) of an aligned run of kKvGroup that are new tokens
// of a sequence, at packed rows row + [first, last): those of the at-th run from its
// first new token's on; false where there are none, as for a sequence without new
// tokens, which owns no row that could be read.
struct KvRun {
  int64_t row;
  int base, first, last;
};
__host__ __device__ inline bool kv_run(const KvSeq& s, int64_t at, KvRun& k) {
  const int64_t from = static_cast<int64_t>(s.len) - s.n;   // may lie before position 0
  const int64_t base = ((from >> 4) + at) * kKvGroup;
  if (s.n <= 0 || at < 0 || base >= s.len) return false;
  k.base = static_cast<int>(base);
  k.first = from > base ? static_cast<int>(from - base) : 0;
  k.last = s.len - base < kKvGroup ? static_cast<int>(s.len - base) : kKvGroup;
  k.row = s.row0 + (base - from);
  return true;
}
// i, or the nearest that is in the run.
__host__ __device__ inline int kv_in_run(const KvRun& k, int i) {
  return i < k.first ? k.first : i >= k.last ? k.last - 1 : i;
}

constexpr int kTile = 64;  // positions that the attention takes at a time

// The low n bits.
__host__ __device__ inline uint64_t low_bits(int n) { return n >= 64 ? ~0ull : n <= 0 ? 0ull : (1ull << n) - 1; }

// The tiles that rows at positions [p_lo, p_hi] see of cap positions: those of the
// first tokens, then those of the window.
struct KvSpan {
  int lo, hi, sink_tiles, skip, tiles;  // window positions [lo, hi)
  __host__ __device__ int key0(int i) const { return (i < sink_tiles ? i : i + skip) * kTile; }
};
__host__ __device__ inline KvSpan kv_span(int cap, int window, int first, int p_lo, int p_hi) {
  KvSpan s;
  s.hi = p_hi < cap ? p_hi + 1 : cap;
  if (s.hi < 0) s.hi = 0;
  // (p_lo may be far below 0, and window 2^31 - 1)
  s.lo = window > 0 && p_lo >= window ? p_lo - window + 1 : 0;
  const int sinks = first < s.lo ? first : s.lo;
  const int t1 = (s.hi + kTile - 1) / kTile;
  s.sink_tiles = (sinks + kTile - 1) / kTile;
  if (s.sink_tiles > t1) s.sink_tiles = t1;
  const int t0 = s.lo / kTile > s.sink_tiles ? s.lo / kTile : s.sink_tiles;
  s.skip = t0 - s.sink_tiles;
  s.tiles = s.sink_tiles + (t1 > t0 ? t1 - t0 : 0);
  return s;
}
// The tile's keys (bit k: position key0 + k) that a token at position pos sees.
__host__ __device__ inline uint64_t kv_seen(int pos, int key0, int window, int sinks) {
  if (pos < key0) return 0;
  const int rel = pos - key0;
  uint64_t see = low_bits(rel + 1);
  if (window > 0) see &= ~low_bits(rel - window + 1) | low_bits(sinks - key0);
  return see;
}

// A tensor's layers: n blocks of bytes, stride (at least as many) apart.
struct KvBlocks {
  uintptr_t at;
  int64_t bytes, stride, n;
};
// Whether some block of a and some block of b hold a byte in common.  (Layers of several
// tensors may lie between each other.)
inline bool kv_meet(const KvBlocks& a, const KvBlocks& b) {
  auto end = [](const KvBlocks& t) { return t.at + static_cast<uintptr_t>((t.n - 1) * t.stride + t.bytes); };
  if (a.n < 1 || b.n < 1 || a.bytes < 1 || b.bytes < 1 || !(a.at < end(b) && b.at < end(a))) return false;
  for (int64_t i = 0, j = 0; i < a.n && j < b.n;) {
    const uintptr_t x = a.at + static_cast<uintptr_t>(i * a.stride), y = b.at + static_cast<uintptr_t>(j * b.stride);
    if (x < y + static_cast<uintptr_t>(b.bytes) && y < x + static_cast<uintptr_t>(a.bytes)) return true;
    ++(x < y ? i : j);  // (that block ends before the other begins)
  }
  return false;
}

// The page of position pos of sequence b, or -1: past the table, or an entry
// that names no page.
__device__ inline int kv_page(const KvView& p, int64_t b, int pos) {
  if (pos < 0 || pos >= p.cap) return -1;
  const int id = p.table[b * p.tstride + (pos >> p.logP)];
  return id >= 0 && id < p.n_pages ? id : -1;
}

// The last b in [0, B) with start(b) <= at, for non-decreasing starts from
// start(0) <= at on: 64 probes a round, by the whole wave.
template <class F>
__device__ inline int64_t kv_find(int64_t B, int64_t at, F start) {
  const int lane = threadIdx.x & 63;
  int64_t lo = 0, n = B;
  while (n > 1) {
    const int64_t step = (n + 63) / 64, i = lane * step;
    const uint64_t le = __ballot(i < n && start(lo + i) <= at);
    const int c = __popcll(le);
    const int64_t skip = c > 0 ? (c - 1) * step : 0;
    lo += skip;
    n = n - skip < step ? n - skip : step;
  }
  return lo;
}

// Eight 8-bit codes (two dwords) as eight bf16 numbers, exactly: both formats'
// values fit bf16's eight significant bits.
template <int KIND>
__device__ inline u32x4_t widen8(uint32_t a, uint32_t b) {
  u32x4_t r;
  if constexpr (KIND == SRW_KV_FP8) {
    typedef __bf16 v2 __attribute__((ext_vector_type(2)));
    const v2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false);
    const v2 x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
    const v2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false);
    const v2 x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    r[0] = __builtin_bit_cast(uint32_t, x0);
    r[1] = __builtin_bit_cast(uint32_t, x1);
    r[2] = __builtin_bit_cast(uint32_t, x2);
    r[3] = __builtin_bit_cast(uint32_t, x3);
  } else {
    // the high halves of the floats hold all of an integer of eight bits
    auto two = [](uint32_t w, int i) {
      const float lo = static_cast<float>(static_cast<int8_t>(w >> (16 * i)));
      const float hi = static_cast<float>(static_cast<int8_t>(w >> (16 * i + 8)));
      return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
    };
    r[0] = two(a, 0);
    r[1] = two(a, 1);
    r[2] = two(b, 0);
    r[3] = two(b, 1);
  }
  return r;
}

// v of lane J of the lane's row of 16.
template <int J>
__device__ inline float row_lane(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x150 + J, 0xF, 0xF, true));
}

// Reductions over lanes (l ^ 16) and (l ^ 32): every lane gets the result.
template <class Op>
__device__ inline float join16(float v, Op op) {
  const auto r = __builtin_amdgcn_permlane16_swap(as_i(v), as_i(v), false, false);
  return op(as_f(r[0]), as_f(r[1]));
}
template <class Op>
__device__ inline float join32(float v, Op op) {
  const auto r = __builtin_amdgcn_permlane32_swap(as_i(v), as_i(v), false, false);
  return op(as_f(r[0]), as_f(r[1]));
}

// Host launches (arguments checked).
struct KvRows {
  const void* k;  // kv_write: sources; kv_read: destinations
  const void* v;
  int64_t k_token, k_head, v_token, v_head;  // strides in elements
};
hipError_t kv_write(const srw_kv_t& c, const KvRows& r, bool f32, hipStream_t s);
hipError_t kv_read(const srw_kv_t& c, const KvRows& r, bool f32, hipStream_t s);
srw_status_t check_kv(const srw_kv_t* c);
size_t attention_workspace_bytes(const srw_attention_t& a);
void attention_plan(const srw_attention_t& a, int32_t* rows, int32_t* splits);
hipError_t attention(const srw_attention_t& a, char* ws, hipStream_t s);
size_t attention_kept_workspace_bytes(const srw_attention_t& a, int64_t n_keep);
hipError_t attention_kept(const srw_attention_t& a, const int32_t* keep, int64_t n_keep, char* ws, hipStream_t s);

}  // namespace srw

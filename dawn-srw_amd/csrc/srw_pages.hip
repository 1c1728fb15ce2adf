// srw_pages.hip -- the paged cache's pages: copies of them, an index of what their
// keys are about, and the choice of pages by it.

#include <math.h>

#include <algorithm>
#include <vector>

#include "srw_kv.hpp"

namespace srw {
namespace {

bool aligned(const void* q, size_t a) { return q && !(reinterpret_cast<uintptr_t>(q) & (a - 1)); }

// -- copies -------------------------------------------------------------------------
//
// A workgroup copies up to kPiece bytes of one page of one layer of one tensor, every
// lane four 16-byte loads in flight, past the caches (what is copied is not read again
// here).  The pairs travel as kernel arguments, so a call copies nothing to the device
// first and waits for nothing.  Bound by the memory: 200 pages of 24 layers, 1.30 GB read
// and written, 236 us, 5.5 TB/s (a copy of one large tensor: 5.15); three pages of 12
// layers 3.5 us, the launch.
constexpr int kPiece = 16384, kPairs = 256, kCopyThreads = 256;

struct CopyArgs {
  const char* src[SRW_KV_COPY_TENSORS];
  char* dst[SRW_KV_COPY_TENSORS];
  int64_t page[SRW_KV_COPY_TENSORS];                                // bytes
  int64_t src_layer[SRW_KV_COPY_TENSORS], dst_layer[SRW_KV_COPY_TENSORS];
  int32_t begin[SRW_KV_COPY_TENSORS + 1];                           // of each tensor's pieces
  int32_t n, wide;                                                  // tensors; bit i: tensor i in units of 16 bytes
  int32_t from[kPairs], to[kPairs];
};

template <typename U>
__device__ inline void copy_piece(const char* src, char* dst, int bytes) {
  constexpr int K = kPiece / kCopyThreads / sizeof(U), N = K < 4 ? K : 4;
  const U* s = reinterpret_cast<const U*>(src);
  U* d = reinterpret_cast<U*>(dst);
  const int n = bytes / static_cast<int>(sizeof(U));
  for (int i = threadIdx.x; i < n; i += N * kCopyThreads) {
    U x[N];
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k * kCopyThreads < n) x[k] = __builtin_nontemporal_load(s + i + k * kCopyThreads);
#pragma unroll
    for (int k = 0; k < N; ++k)
      if (i + k * kCopyThreads < n) __builtin_nontemporal_store(x[k], d + i + k * kCopyThreads);
  }
}

__global__ __launch_bounds__(kCopyThreads) void kv_copy_kernel(CopyArgs a) {
  int t = 0;
  const int at = blockIdx.x;
  while (t + 1 < a.n && at >= a.begin[t + 1]) ++t;
  const int64_t page = a.page[t], off = static_cast<int64_t>(at - a.begin[t]) * kPiece;
  const char* src = a.src[t] + blockIdx.z * a.src_layer[t] + a.from[blockIdx.y] * page + off;
  char* dst = a.dst[t] + blockIdx.z * a.dst_layer[t] + a.to[blockIdx.y] * page + off;
  const int bytes = static_cast<int>(page - off < kPiece ? page - off : kPiece);
  if (a.wide >> t & 1)
    copy_piece<u32x4_t>(src, dst, bytes);
  else
    copy_piece<uint32_t>(src, dst, bytes);
}

srw_status_t check_copy(const srw_kv_copy_t* c) {
  if (!c || c->n_tensors < 0 || c->n_tensors > SRW_KV_COPY_TENSORS) return SRW_EINVAL;
  if (c->n_layers < 0 || c->n_src_pages < 0 || c->n_dst_pages < 0 || c->n_pairs < 0) return SRW_EINVAL;
  if (c->n_layers > 65535 || c->n_src_pages > 0x7fffffff || c->n_dst_pages > 0x7fffffff) return SRW_EUNSUPPORTED;
  if (c->n_pairs > c->n_dst_pages) return SRW_EINVAL;  // (some page is written twice)
  if (c->n_pairs == 0 || c->n_layers == 0 || c->n_tensors == 0) return SRW_OK;
  if (!aligned(c->src_page, 4) || !aligned(c->dst_page, 4)) return SRW_EINVAL;
  KvBlocks src[SRW_KV_COPY_TENSORS], dst[SRW_KV_COPY_TENSORS];
  bool inside = false;  // tensors copied within themselves
  for (int i = 0; i < c->n_tensors; ++i) {
    if (c->page_bytes[i] < 1 || c->page_bytes[i] % 4) return SRW_EINVAL;
    if (c->page_bytes[i] > (int64_t{1} << 30)) return SRW_EUNSUPPORTED;
    if (!aligned(c->src[i], 4) || !aligned(c->dst[i], 4)) return SRW_EINVAL;
    auto blocks = [&](const void* at, int64_t stride, int64_t pages, KvBlocks* b) {
      *b = {reinterpret_cast<uintptr_t>(at), pages * c->page_bytes[i], c->n_layers > 1 ? stride : 0, c->n_layers};  // below 2^61
      return c->n_layers == 1 || (stride >= b->bytes && stride % 4 == 0 && stride <= (int64_t{1} << 46));
    };
    if (!blocks(c->src[i], c->src_layer_stride[i], c->n_src_pages, &src[i]) ||
        !blocks(c->dst[i], c->dst_layer_stride[i], c->n_dst_pages, &dst[i]))
      return SRW_EINVAL;
  }
  for (int i = 0; i < c->n_tensors; ++i)
    for (int j = 0; j < c->n_tensors; ++j) {
      if (i < j && kv_meet(dst[i], dst[j])) return SRW_EINVAL;
      if (i == j && src[i].at == dst[i].at && src[i].bytes == dst[i].bytes && src[i].stride == dst[i].stride)
        inside = true;
      else if (kv_meet(src[i], dst[j]))
        return SRW_EINVAL;
    }
  for (int64_t j = 0; j < c->n_pairs; ++j)
    if (c->src_page[j] < 0 || c->src_page[j] >= c->n_src_pages || c->dst_page[j] < 0 || c->dst_page[j] >= c->n_dst_pages)
      return SRW_EINVAL;
  if (c->n_pairs <= 16) {
    for (int64_t j = 0; j < c->n_pairs; ++j)
      for (int64_t k = 0; k < c->n_pairs; ++k)
        if ((k != j && c->dst_page[j] == c->dst_page[k]) || (inside && c->src_page[j] == c->dst_page[k])) return SRW_EINVAL;
    return SRW_OK;
  }
  try {
    std::vector<uint64_t> written(static_cast<size_t>(c->n_dst_pages / 64 + 1));
    for (int64_t j = 0; j < c->n_pairs; ++j) {
      uint64_t& w = written[c->dst_page[j] >> 6];
      const uint64_t bit = uint64_t{1} << (c->dst_page[j] & 63);
      if (w & bit) return SRW_EINVAL;
      w |= bit;
    }
    if (inside)
      for (int64_t j = 0; j < c->n_pairs; ++j)
        if (written[c->src_page[j] >> 6] >> (c->src_page[j] & 63) & 1) return SRW_EINVAL;
  } catch (...) {  // no memory for the bits
    return SRW_EHIP;
  }
  return SRW_OK;
}

hipError_t kv_copy(const srw_kv_copy_t& c, hipStream_t s) {
  CopyArgs a{};
  a.n = c.n_tensors;
  for (int i = 0; i < c.n_tensors; ++i) {
    a.src[i] = static_cast<const char*>(c.src[i]);
    a.dst[i] = static_cast<char*>(c.dst[i]);
    a.page[i] = c.page_bytes[i];
    a.src_layer[i] = c.n_layers > 1 ? c.src_layer_stride[i] : 0;
    a.dst_layer[i] = c.n_layers > 1 ? c.dst_layer_stride[i] : 0;
    a.begin[i + 1] = a.begin[i] + static_cast<int32_t>((c.page_bytes[i] + kPiece - 1) / kPiece);
    if (aligned(c.src[i], 16) && aligned(c.dst[i], 16) && (a.page[i] | a.src_layer[i] | a.dst_layer[i]) % 16 == 0)
      a.wide |= 1 << i;
  }
  for (int64_t at = 0; at < c.n_pairs; at += kPairs) {
    const int n = static_cast<int>(c.n_pairs - at < kPairs ? c.n_pairs - at : kPairs);
    for (int j = 0; j < n; ++j) {
      a.from[j] = c.src_page[at + j];
      a.to[j] = c.dst_page[at + j];
    }
    hipLaunchKernelGGL(kv_copy_kernel,
                       dim3(static_cast<unsigned>(a.begin[a.n]), static_cast<unsigned>(n), static_cast<unsigned>(c.n_layers)),
                       dim3(kCopyThreads), 0, s, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// -- the index ------------------------------------------------------------------------

constexpr float kTiny = 7.888609052210118e-31f;  // 2^-100

// Codes of numbers whose largest magnitude has the bits `most`: x * inv to the nearest;
// inv 0 for zeros and where a number is not finite.
__device__ inline bool not_finite(uint32_t most) { return most >= 0x7f800000u; }
__device__ inline float code_factor(uint32_t most) {
  const float m = __uint_as_float(most);
  return not_finite(most) || m <= kTiny ? 0.f : 127.f / m;
}
__device__ inline uint32_t code_of(float x, float inv) {
  return static_cast<uint32_t>(static_cast<int>(rintf(inv == 0.f ? 0.f : x * inv))) & 0xffu;
}

// a's sum over the two halves (W 32; 16: over each half's two rows) in the lower one, b's
// in the upper one.
template <int W>
__device__ inline double traded(double a, double b) {
  const uint64_t x = __builtin_bit_cast(uint64_t, a), y = __builtin_bit_cast(uint64_t, b);
  auto trade = [](uint32_t u, uint32_t v) {
    if constexpr (W == 32)
      return __builtin_amdgcn_permlane32_swap(u, v, false, false);
    else
      return __builtin_amdgcn_permlane16_swap(u, v, false, false);
  };
  const auto lo = trade(static_cast<uint32_t>(x), static_cast<uint32_t>(y));
  const auto hi = trade(static_cast<uint32_t>(x >> 32), static_cast<uint32_t>(y >> 32));
  return __builtin_bit_cast(double, static_cast<uint64_t>(hi[0]) << 32 | lo[0]) +
         __builtin_bit_cast(double, static_cast<uint64_t>(hi[1]) << 32 | lo[1]);
}
// x of the lane W further on in the row of 16, around its end.
template <int W>
__device__ inline double turned(double x) {
  const uint64_t u = __builtin_bit_cast(uint64_t, x);
  auto turn = [](uint32_t v) {
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x120 | W, 0xf, 0xf, false));
  };
  const uint64_t hi = turn(static_cast<uint32_t>(u >> 32)), lo = turn(static_cast<uint32_t>(u));
  return __builtin_bit_cast(double, hi << 32 | lo);
}

// One wave: a page and head.  A lane holds 16 bytes' dims of every (64 / lanes a
// key)th key and sums them in 64 bits, where sums of up to 256 keys of any 8-bit or
// bf16 page are exact but for rare exponents far apart, so that the codes do not go by
// the order of adding.  The lanes' sums meet by trades of halves and rows, each lane
// going on with fewer dims (sums of all dims over all lanes took 5 us more).  Bound by the
// keys' bytes: 65 521 tokens of 8 heads of 128, int8, 17.2 us, 4.1 TB/s (13.6 at a copy's
// rate); 8 prompts of 512 bf16 4.5 us.
//
// `pages` > 0: a unit for every place of every table, which needs no search and goes by no
// number of tokens; 0: units by the tokens.
template <int KIND, int DH>
__global__ __launch_bounds__(256) void kv_index_kernel(KvView p, uint32_t pages, int8_t* codes, float* scale) {
  constexpr int ES = kv_bytes<KIND>(), N = 16 / ES;     // dims a lane
  constexpr int kLanes = DH / N, kKeys = 64 / kLanes;   // lanes a key, keys a step
  constexpr int U = 4;                                  // steps in flight
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, head = blockIdx.y;
  // units of a page of sequence b: start(b) = cu[b] / P + 2 b leaves room for both
  // partial ends
  int64_t b = unit, at = 0;
  if (pages > 0) {
    b = static_cast<uint32_t>(unit) / pages;
    if (b >= p.B) return;
    at = static_cast<uint32_t>(unit) % pages;
  } else if (p.cu) {
    auto start = [&](int64_t i) { return (static_cast<int64_t>(p.cu[i]) >> p.logP) + 2 * i; };
    b = kv_find(p.B, unit, start);
    at = unit - start(b);
  } else if (unit >= p.B) {
    return;
  }
  const KvSeq sq = kv_seq(p, b);
  if (sq.n <= 0 || at < 0) return;
  const int first = sq.len > sq.n ? (sq.len - sq.n) >> p.logP : 0;  // the first page with a new token
  if (pages > 0 && at < first) return;
  const int64_t base = (pages > 0 ? at : first + at) << p.logP;
  if (base >= sq.len) return;
  const int page = kv_page(p, b, static_cast<int>(base));
  if (page < 0) return;
  const int have = sq.len - base < p.P ? static_cast<int>(sq.len - base) : p.P;
  const int64_t ph = static_cast<int64_t>(page) * p.H + head;
  const char* src = p.k + ph * p.P * (DH * ES) + 16 * lane;
  double sum[N];
#pragma unroll
  for (int j = 0; j < N; ++j) sum[j] = 0.0;
  const int mine = lane / kLanes;
  for (int k0 = 0; k0 < have; k0 += kKeys * U) {
    u32x4_t w[U];
    float ks[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int key = k0 + u * kKeys + mine;
      w[u] = u32x4_t{0, 0, 0, 0};
      ks[u] = 0.f;
      if (key < have) {
        w[u] = *reinterpret_cast<const u32x4_t*>(src + static_cast<int64_t>(k0 + u * kKeys) * (DH * ES));
        if constexpr (KIND != SRW_KV_BF16) ks[u] = p.ks[ph * p.P + key];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if constexpr (KIND == SRW_KV_BF16) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          sum[2 * j] += static_cast<double>(lo_f32(w[u][j]));
          sum[2 * j + 1] += static_cast<double>(hi_f32(w[u][j]));
        }
      } else {
        const double s = ks[u];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float x[4];
          if constexpr (KIND == SRW_KV_FP8) {
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[u][j], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[u][j], true);
            x[0] = lo[0];
            x[1] = lo[1];
            x[2] = hi[0];
            x[3] = hi[1];
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w[u][j] >> (8 * i)));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[4 * j + i] = fma(static_cast<double>(x[i]), s, sum[4 * j + i]);
        }
      }
    }
  }
  // the keys' lanes join: halves, then rows of 16, trade half of their dims, so that a lane
  // ends with the sums of D of them; lanes of a row that hold the same dims add in turn
  constexpr int D = N / 4;
#pragma unroll
  for (int j = 0; j < N / 2; ++j) sum[j] = traded<32>(sum[j], sum[j + N / 2]);
#pragma unroll
  for (int j = 0; j < D; ++j) sum[j] = traded<16>(sum[j], sum[j + D]);
  float mean[D];
  uint32_t most = 0;
#pragma unroll
  for (int j = 0; j < D; ++j) {
    if constexpr (kLanes <= 8) sum[j] += turned<8>(sum[j]);
    if constexpr (kLanes <= 4) sum[j] += turned<4>(sum[j]);
    mean[j] = static_cast<float>(sum[j] / have);
    const uint32_t m = __float_as_uint(mean[j]) & 0x7fffffffu;
    most = m > most ? m : most;
  }
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) {
    if (w >= kLanes && w < 16) continue;
    const uint32_t o = __shfl_xor(most, w);
    most = o > most ? o : most;
  }
  if ((lane & 15) >= kLanes) return;
  const float inv = code_factor(most), m = __uint_as_float(most);
  uint32_t c = 0;
#pragma unroll
  for (int j = 0; j < D; ++j) c |= code_of(mean[j], inv) << 8 * j;
  char* dst = reinterpret_cast<char*>(codes) + ph * DH + (lane & 15) * N + (lane >> 5) * (N / 2) + (lane >> 4 & 1) * D;
  if constexpr (D == 4)
    *reinterpret_cast<uint32_t*>(dst) = c;
  else
    *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(c);
  if (lane == 0) scale[ph] = not_finite(most) ? __uint_as_float(0x7fc00000u) : inv == 0.f ? 0.f : m / 127.f;
}

// -- the choice of pages ----------------------------------------------------------------
//
// A workgroup takes R tokens of a sequence and one key head; the threads score pages
// (whole numbers by dot products of four codes, one page a thread and step), as keys
// that order like the scores, into LDS; NT / R threads then find each row's border and
// write the places that lie before it.  The border: a histogram of the scores between
// their smallest and largest, then, of the bin that it falls into, each key's number of
// larger ones.  Where that bin holds more than 64 keys (many equal scores), and for
// tables of more pages than LDS holds keys, which are scored again each time, the border
// comes by digits of the keys.
//
// Bound by the chain of loads (lengths, table, codes) and eight barriers: one row of 8
// heads over 64 pages 6.0 us, of which the border takes two; for few rows over many pages by
// what one CU reads (11 000 pages 34 us); 32 rows over 500 pages 8.4 us.

struct SelectArgs {
  KvView kv;
  const int8_t* codes;
  const float* scale;
  const uint16_t* q;
  int32_t* keep;
  int64_t q_token, q_head;
  int G, n, first, last, hold;  // hold: keys of a row in LDS, a multiple of 64
};

// A score's place among all; 0 is no page's.
constexpr uint32_t kAlways = 0xffffffffu;
__device__ inline uint32_t key_of(float score) {
  if (score != score) return kAlways - 1;
  const uint32_t b = __float_as_uint(score + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ inline float score_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key ^ 0x80000000u : ~key);
}

constexpr int kBinKeys = 64;
constexpr int64_t kKeys = 12288;  // of a workgroup in LDS: 48 KB

// x of the lane that C names within each four (quad_perm), all lanes active.
template <int C>
__device__ inline int dpp(int x) {
  return __builtin_amdgcn_mov_dpp(x, C, 0xf, 0xf, false);
}

template <int DH, int R, int NT>
__global__ __launch_bounds__(NT) void kv_select_kernel(SelectArgs a) {
  constexpr int kRow = NT / R;        // threads of a row
  constexpr int kWaves = kRow / 64;
  extern __shared__ uint32_t keys[];  // [R][hold]
  __shared__ __align__(16) uint32_t qc[R][DH / 4];
  __shared__ uint32_t hist[R][256], bin[R][kBinKeys], binned[R], ends[R][kWaves][2];
  const int tid = threadIdx.x, lane = tid & 63, head = blockIdx.y;
  const KvView& p = a.kv;
  int64_t b, at;
  if (p.cu) {
    auto start = [&](int64_t i) { return static_cast<int64_t>(p.cu[i]) / R + i; };
    b = kv_find(p.B, blockIdx.x, start);
    at = blockIdx.x - start(b);
  } else {
    b = blockIdx.x;
    at = 0;
  }
  b = __builtin_amdgcn_readfirstlane(static_cast<int>(b));
  const KvSeq sq = kv_seq(p, b);
  const int tok0 = static_cast<int>(at) * R;
  if (at < 0 || at * R >= sq.n) return;
  const int toks = sq.n - tok0 < R ? sq.n - tok0 : R;

  // pages that a row sees: [0, own]
  auto own_of = [&](int r) {
    const int pos = sq.len - sq.n + tok0 + r;
    const int most_pages = p.cap >> p.logP;
    if (r >= toks || pos < 0 || most_pages == 0) return -1;
    return pos >> p.logP < most_pages ? pos >> p.logP : most_pages - 1;
  };
  const int pages = own_of(toks - 1) + 1;

  auto id_of = [&](int j) { return j < pages ? kv_page(p, b, j << p.logP) : -1; };
  // the rows' codes: DH / 4 lanes a row, four dims a lane
  const int qr = tid / (DH / 4), qd = tid % (DH / 4);
  double x[4] = {0.0, 0.0, 0.0, 0.0};
  const bool reads = qr < toks && qr < R;
  const uint16_t* src =
      a.q + (sq.row0 + tok0 + (reads ? qr : 0)) * a.q_token + static_cast<int64_t>(head) * a.G * a.q_head + 4 * qd;
  constexpr int kHeads = 8;  // loads in flight
  uint2 w[kHeads];
#pragma unroll
  for (int g = 0; g < kHeads; ++g) w[g] = reads && g < a.G ? *reinterpret_cast<const uint2*>(src + g * a.q_head) : uint2{0, 0};
  int id = id_of(tid);
  if (tid < R) binned[tid] = 0;
  for (int i = tid; i < R * 256; i += NT) hist[0][i] = 0;
  for (int g0 = 0;;) {
#pragma unroll
    for (int g = 0; g < kHeads; ++g) {
      x[0] += static_cast<double>(lo_f32(w[g].x));
      x[1] += static_cast<double>(hi_f32(w[g].x));
      x[2] += static_cast<double>(lo_f32(w[g].y));
      x[3] += static_cast<double>(hi_f32(w[g].y));
    }
    g0 += kHeads;
    if (g0 >= a.G) break;
#pragma unroll
    for (int g = 0; g < kHeads; ++g)
      w[g] = reads && g0 + g < a.G ? *reinterpret_cast<const uint2*>(src + (g0 + g) * a.q_head) : uint2{0, 0};
  }
  if (qr < R) {
    uint32_t most = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t m = __float_as_uint(static_cast<float>(x[j])) & 0x7fffffffu;
      most = m > most ? m : most;
    }
#pragma unroll
    for (int o = 1; o < DH / 4; o <<= 1) {
      const uint32_t m = __shfl_xor(most, o);
      most = m > most ? m : most;
    }
    const float inv = code_factor(most);
    uint32_t c = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) c |= code_of(static_cast<float>(x[j]), inv) << 8 * j;
    qc[qr][qd] = c;
  }
  __syncthreads();

  // A wave scores 64 places, four lanes a page (a page a lane would touch each line of its
  // codes DH / 16 times): lane l of a quad loads 16 of every 64 dims of the quad's four
  // pages and ends up with the sum of the page of place l.
  constexpr int C = DH / 64;
  const int part = lane & 3;
  auto score = [&](int from) {  // keys of places [from, from + hold)
    const int to = pages - from < a.hold ? pages - from : a.hold;
    if (pages > a.hold) id = id_of(from + tid);
    for (int i = tid; i < ((to + 63) & ~63); i += NT) {
      const int j = from + i, next = i + NT < to ? id_of(j + NT) : -1;
      int dot[R][4];
      float scale = 0.f;
      if (p.n_pages > 0) {
        scale = a.scale[static_cast<int64_t>(id > 0 ? id : 0) * p.H + head];
        u32x4_t w[4][C];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int other = u == 0 ? dpp<0x00>(id) : u == 1 ? dpp<0x55>(id) : u == 2 ? dpp<0xaa>(id) : dpp<0xff>(id);
          const u32x4_t* src = reinterpret_cast<const u32x4_t*>(
              a.codes + (static_cast<int64_t>(other > 0 ? other : 0) * p.H + head) * DH);
#pragma unroll
          for (int c = 0; c < C; ++c) w[u][c] = src[4 * c + part];
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int u = 0; u < 4; ++u) dot[r][u] = 0;
#pragma unroll
          for (int c = 0; c < C; ++c) {
            const u32x4_t y = *reinterpret_cast<const u32x4_t*>(&qc[r][16 * c + 4 * part]);
#pragma unroll
            for (int u = 0; u < 4; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e)
                dot[r][u] = __builtin_amdgcn_sdot4(static_cast<int>(w[u][c][e]), static_cast<int>(y[e]), dot[r][u], false);
          }
        }
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const bool two = part & 2, one = part & 1;
        const int d0 = (two ? dot[r][2] : dot[r][0]) + dpp<0x4e>(two ? dot[r][0] : dot[r][2]);
        const int d1 = (two ? dot[r][3] : dot[r][1]) + dpp<0x4e>(two ? dot[r][1] : dot[r][3]);
        const int sum = (one ? d1 : d0) + dpp<0xb1>(one ? d0 : d1);
        const int own = own_of(r);
        uint32_t key = 0;
        if (id >= 0 && j <= own)
          key = j < a.first || j > own - a.last ? kAlways : key_of(static_cast<float>(sum) * scale);
        keys[r * a.hold + i] = key;
      }
      id = next;
    }
  };

  const int r = tid / kRow, t = tid % kRow;
  const uint32_t* row = keys + r * a.hold;
  // the bin of the 256, in order, in which `left` falls, with what lies before it and in
  // it; -1: all fall short of it
  auto find = [&](uint32_t left, uint32_t* before, uint32_t* count) {
    uint32_t c[4], s = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      c[k] = hist[r][4 * lane + k];
      s += c[k];
    }
    uint32_t run = s;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t v = __shfl_up(run, o);
      if (lane >= o) run += v;
    }
    const uint64_t past = __ballot(run >= left);
    if (!past) return -1;
    uint32_t at = run - s, n = c[0];
    int k = 0;
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (k == i && at + c[i] < left) {
        at += c[i];
        n = c[i + 1];
        k = i + 1;
      }
    const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(past));
    *before = __builtin_amdgcn_readlane(at, l);
    *count = __builtin_amdgcn_readlane(n, l);
    return 4 * l + __builtin_amdgcn_readlane(k, l);
  };
  // the border: keys above K, and as many equal to it as are left
  uint32_t K = 0, left = a.n;
  const bool held = pages <= a.hold;
  bool digits = !held;
  if (held) {
    score(0);
    __syncthreads();
  }
  if (pages <= a.n) {
    left = 0;
    digits = false;
  } else if (held) {
    uint32_t lo = kAlways, hi = 0;  // of finite scores
    for (int i = t; i < pages; i += kRow) {
      const uint32_t key = row[i];
      if (key > 0x007fffffu && key < 0xff800000u) {
        lo = key < lo ? key : lo;
        hi = key > hi ? key : hi;
      }
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t l = __shfl_xor(lo, o), h = __shfl_xor(hi, o);
      lo = l < lo ? l : lo;
      hi = h > hi ? h : hi;
    }
    if constexpr (kWaves > 1) {
      if (lane == 0) {
        ends[r][t >> 6][0] = lo;
        ends[r][t >> 6][1] = hi;
      }
      __syncthreads();
      lo = ends[r][lane % kWaves][0];
      hi = ends[r][lane % kWaves][1];
#pragma unroll
      for (int o = 1; o < kWaves; o <<= 1) {
        const uint32_t l = __shfl_xor(lo, o), h = __shfl_xor(hi, o);
        lo = l < lo ? l : lo;
        hi = h > hi ? h : hi;
      }
    }
    const float low = 0.5f * score_of(lo), wide = 0.5f * score_of(hi) - low;
    float to_bin = 253.f / wide;
    if (!(hi > lo) || !(to_bin < 1e38f)) to_bin = 0.f;
    // a larger key's bin is no later: each rounding keeps the order
    auto bin_of = [&](uint32_t key) {
      if (key >= kAlways - 1) return static_cast<int>(kAlways - key);
      const float y = (0.5f * score_of(key) - low) * to_bin;
      return 255 - (y >= 253.f ? 253 : y > 0.f ? static_cast<int>(y) : 0);
    };
    for (int i = t; i < pages; i += kRow) {
      const uint32_t key = row[i];
      if (key) atomicAdd(&hist[r][bin_of(key)], 1u);
    }
    __syncthreads();
    uint32_t before = 0, count = 0;
    const int border = find(left, &before, &count);
    if (border < 0) {
      left = 0;
    } else if (count > kBinKeys) {
      digits = true;
    } else {
      for (int i = t; i < pages; i += kRow) {
        const uint32_t key = row[i];
        if (key && bin_of(key) == border) bin[r][atomicAdd(&binned[r], 1u)] = key;
      }
    }
    digits = __syncthreads_or(digits);
    if (border >= 0 && count <= kBinKeys) {
      const uint32_t mine = lane < static_cast<int>(count) ? bin[r][lane] : 0;
      uint32_t more = before, same = 0;
      for (uint32_t i = 0; i < count; ++i) {
        const uint32_t o = __builtin_amdgcn_readlane(mine, i);
        more += o > mine;
        same += o == mine;
      }
      const int l = __builtin_amdgcn_readfirstlane(__builtin_ctzll(__ballot(mine && more < left && more + same >= left)));
      K = __builtin_amdgcn_readlane(mine, l);
      left -= __builtin_amdgcn_readlane(more, l);
    }
  }
  if (digits) {
    K = 0;
    left = a.n;
    for (int shift = 24; shift >= 0; shift -= 8) {
      __syncthreads();
      for (int i = t; i < 256; i += kRow) hist[r][i] = 0;
      __syncthreads();
      for (int from = 0; from < pages; from += a.hold) {
        if (!held) {
          score(from);
          __syncthreads();
        }
        const int to = pages - from < a.hold ? pages - from : a.hold;
        for (int i = t; i < to; i += kRow) {
          const uint32_t key = row[i];
          if (shift == 24 || key >> (shift + 8) == K >> (shift + 8)) atomicAdd(&hist[r][255 - (key >> shift & 255)], 1u);
        }
        __syncthreads();
      }
      // (places without a page count too: there are more pages than are kept)
      uint32_t before = 0, count = 0;
      const int digit = find(left, &before, &count);
      K |= static_cast<uint32_t>(255 - digit) << shift;
      left -= before;
    }
  }
  // write: a wave the places of a run of its own, in order
  const int tok = tok0 + r;
  const bool mine = r < toks;
  int32_t* out = a.keep + ((sq.row0 + (mine ? tok : 0)) * p.H + head) * a.n;
  uint32_t more = 0, same = 0;  // before the run
  for (int from = 0; from < pages; from += a.hold) {
    if (!held) {
      __syncthreads();
      score(from);
      __syncthreads();
    }
    const int to = pages - from < a.hold ? pages - from : a.hold;
    const int run = (to + kRow - 1) / kRow * 64, i0 = t / 64 * run, i1 = i0 + run < to ? i0 + run : to;
    uint32_t m = 0, e = 0;  // kept for sure, and equal to the border, in the run
    for (int i = i0; i < i1; i += 64) {
      const uint32_t key = i + lane < i1 ? row[i + lane] : 0;
      m += __popcll(__ballot(key > K));
      e += __popcll(__ballot(key != 0 && key == K));
    }
    uint32_t all_m = m, all_e = e;
    if constexpr (kWaves > 1) {
      if (lane == 0) {
        ends[r][t >> 6][0] = m;
        ends[r][t >> 6][1] = e;
      }
      __syncthreads();
      m = lane < kWaves ? ends[r][lane % kWaves][0] : 0;
      e = lane < kWaves ? ends[r][lane % kWaves][1] : 0;
      uint32_t sm = m, se = e;
#pragma unroll
      for (int o = 1; o < kWaves; o <<= 1) {
        const uint32_t vm = __shfl_up(sm, o), ve = __shfl_up(se, o);
        if (lane >= o) {
          sm += vm;
          se += ve;
        }
      }
      all_m = __shfl(sm, kWaves - 1);
      all_e = __shfl(se, kWaves - 1);
      m = __shfl(sm - m, t >> 6);
      e = __shfl(se - e, t >> 6);
      __syncthreads();
    } else {
      m = e = 0;
    }
    m += more;
    e += same;
    more += all_m;
    same += all_e;
    for (int i = i0; i < i1; i += 64) {
      const uint32_t key = i + lane < i1 ? row[i + lane] : 0;
      const uint64_t ab = __ballot(key > K), eq = __ballot(key != 0 && key == K), before = (1ull << lane) - 1;
      const uint32_t em = e + __popcll(eq & before);
      const uint32_t o = m + __popcll(ab & before) + (em < left ? em : left);
      if (mine && o < static_cast<uint32_t>(a.n) && ((ab >> lane & 1) || ((eq >> lane & 1) && em < left)))
        out[o] = from + i + lane;
      m += __popcll(ab);
      e += __popcll(eq);
    }
  }
  if (mine)
    for (int o = static_cast<int>(more + (same < left ? same : left)) + t; o < a.n; o += kRow) out[o] = -1;
}

template <int DH>
hipError_t launch_select(const srw_kv_select_t& c, hipStream_t s) {
  SelectArgs a{};
  a.kv = kv_view(c.kv);
  a.codes = c.index.codes;
  a.scale = c.index.scale;
  a.q = static_cast<const uint16_t*>(c.q);
  a.keep = c.keep;
  a.q_token = c.q_token_stride;
  a.q_head = c.q_head_stride;
  a.G = c.n_heads / c.kv.n_kv_heads;
  a.n = c.n;
  a.first = c.first;
  a.last = c.last;
  // Four rows share the codes' loads where LDS holds the keys of all four: 5 new tokens of
  // 32 sequences over 500 pages 18 us (one row a workgroup: five times the 8.1 of a single
  // token at most), but over 4000, scored anew for each digit, 391 us.
  const int R = c.kv.cu && c.kv.table_width <= kKeys / 4 ? 4 : 1;
  // 256 threads, or 512 where a thread would take more than two pages: one row of 8 heads
  // over 64 | 500 | 1563 | 11000 pages 6.0 | 7.7 | 13.2 | 57 us with 256, 6.2 | 7.3 | 10.8 |
  // 34 with 512 (1024: 8.3 | 9.0 | 11.6 | 31); 256 rows over 500 | 1000 31 | 72 and 37 | 74.
  const bool wide = c.kv.table_width > 512;
  const int64_t most = kKeys / R, width = (c.kv.table_width + 63) / 64 * 64;
  a.hold = static_cast<int>(width < 64 ? 64 : width < most ? width : most);
  const int64_t tiles = c.kv.cu ? c.kv.T / R + c.kv.B : c.kv.B;
  const dim3 grid(static_cast<unsigned>(tiles), static_cast<unsigned>(c.kv.n_kv_heads));
  const unsigned lds = static_cast<unsigned>(a.hold) * R * 4;
  if (R == 4)
    hipLaunchKernelGGL((kv_select_kernel<DH, 4, 256>), grid, dim3(256), lds, s, a);
  else if (wide)
    hipLaunchKernelGGL((kv_select_kernel<DH, 1, 512>), grid, dim3(512), lds, s, a);
  else
    hipLaunchKernelGGL((kv_select_kernel<DH, 1, 256>), grid, dim3(256), lds, s, a);
  return hipGetLastError();
}

srw_status_t check_index(const srw_kv_t& c, const srw_kv_index_t& i) {
  if (c.T > 0 && c.n_pages > 0 && (!aligned(i.codes, 16) || !aligned(i.scale, 4))) return SRW_EINVAL;
  return SRW_OK;
}

template <int KIND>
hipError_t launch_index(const srw_kv_t& c, const srw_kv_index_t& x, hipStream_t s) {
  const KvView p = kv_view(c);
  int64_t units = c.cu ? (c.T >> p.logP) + 2 * c.B : c.B;
  const bool by_table = c.cu && c.B * c.table_width <= units;
  if (by_table) units = c.B * c.table_width;
  if (units == 0) return hipSuccess;  // tables without places
  const uint32_t pages = by_table ? static_cast<uint32_t>(c.table_width) : 0;
  const dim3 grid(static_cast<unsigned>((units + 3) / 4), static_cast<unsigned>(c.n_kv_heads));
  if (c.head_dim == 64)
    hipLaunchKernelGGL((kv_index_kernel<KIND, 64>), grid, dim3(256), 0, s, p, pages, x.codes, x.scale);
  else
    hipLaunchKernelGGL((kv_index_kernel<KIND, 128>), grid, dim3(256), 0, s, p, pages, x.codes, x.scale);
  return hipGetLastError();
}

}  // namespace
}  // namespace srw

extern "C" {

srw_status_t srw_kv_copy(const srw_kv_copy_t* c, void* stream) {
  const srw_status_t st = srw::check_copy(c);
  if (st != SRW_OK) return st;
  if (c->n_pairs == 0 || c->n_layers == 0 || c->n_tensors == 0) return SRW_OK;
  (void)hipGetLastError();
  return srw::kv_copy(*c, static_cast<hipStream_t>(stream)) == hipSuccess ? SRW_OK : SRW_EHIP;
}

srw_status_t srw_kv_index(const srw_kv_t* cache, const srw_kv_index_t* index, void* stream) {
  srw_status_t st = srw::check_kv(cache);
  if (st != SRW_OK) return st;
  if (!index) return SRW_EINVAL;
  st = srw::check_index(*cache, *index);
  if (st != SRW_OK) return st;
  if (cache->T == 0 || cache->n_pages == 0) return SRW_OK;
  if (cache->T > (1 << 29)) return SRW_EUNSUPPORTED;  // (a launch has under 2^32 threads)
  (void)hipGetLastError();
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = cache->kind == SRW_KV_BF16   ? srw::launch_index<SRW_KV_BF16>(*cache, *index, s)
                       : cache->kind == SRW_KV_INT8 ? srw::launch_index<SRW_KV_INT8>(*cache, *index, s)
                                                    : srw::launch_index<SRW_KV_FP8>(*cache, *index, s);
  return e == hipSuccess ? SRW_OK : SRW_EHIP;
}

srw_status_t srw_kv_select(const srw_kv_select_t* c, void* stream) {
  if (!c) return SRW_EINVAL;
  srw_status_t st = srw::check_kv(&c->kv);
  if (st != SRW_OK) return st;
  st = srw::check_index(c->kv, c->index);
  if (st != SRW_OK) return st;
  if (c->n_heads < 1 || c->n_heads % c->kv.n_kv_heads || c->n < 1 || c->first < 0 || c->last < 1 ||
      static_cast<int64_t>(c->first) + c->last > c->n)
    return SRW_EINVAL;
  if (c->kv.T == 0) return SRW_OK;
  if (c->kv.T + c->kv.B > (1 << 22)) return SRW_EUNSUPPORTED;  // (a launch has under 2^32 threads)
  if (!srw::aligned(c->q, 8) || !srw::aligned(c->keep, 4) || c->q_token_stride < 0 || c->q_head_stride < 0 ||
      c->q_token_stride % 4 || c->q_head_stride % 4)
    return SRW_EINVAL;
  (void)hipGetLastError();
  const hipStream_t s = static_cast<hipStream_t>(stream);
  const hipError_t e = c->kv.head_dim == 64 ? srw::launch_select<64>(*c, s) : srw::launch_select<128>(*c, s);
  return e == hipSuccess ? SRW_OK : SRW_EHIP;
}

}  // extern "C"

// srw_kv.hip -- writing into and reading from the paged key/value cache, and
// the C entry points of the cache and of the attention over it.
//
// A key or value row x of one token and head is held in 8 bits as codes c and
// one float32 scale: m = max |x|, c = round(x * (top / m)) with the largest
// code top = 127 (int8, to the nearest, ties to even) or 448 (fp8 e4m3, its
// own nearest), scale = m / top; what is read back is c * scale.  The largest
// magnitude is a code of its own, so nothing saturates.  A row whose m is at
// most 2^-100 (where top / m would leave float32) is held as zeros with scale
// 0; one with an infinity or NaN reads back as NaN throughout (its scale).

#include <math.h>

#include "srw_kv.hpp"

namespace srw {
namespace {

constexpr float kKvTiny = 7.888609052210118e-31f;  // 2^-100

// One wave: 16 aligned positions of one head.  Lane (c, q) holds dims 4c..4c+3
// of KPL consecutive positions from q KPL on, a KPL x 4 block: rows of keys
// are stored along its one side, rows of values along the other, each in
// whole dwords, so neither tensor goes through LDS.  Bound by its bytes; a
// prompt's writes of 16-position runs of value rows meet in L2, where the
// workgroup's four waves (consecutive runs of one head) complete the lines.
// Measured, 65 521 positions of 8 heads of 128, int8 pages, float32 rows: written
// in 130 to 160 us, 4.2 to 5.2 TB/s, read back in 100 to 120, about 6 (part of the
// pages from cache); 64 sequences' single tokens of 6 heads of 64 in 5 us, a launch and one
// chain of dependent loads.
template <int DH>
struct Block : KvRun {
  static constexpr int kLanes = DH / 4;      // lanes a row
  static constexpr int kKeys = DH / 16;      // positions a lane
  int64_t b;                                 // sequence
  int head, c, key0;                         // the lane's dims / 4 and its first position
};

// Units of 16 positions of sequence b: start(b) = cu[b] / 16 + 2 b leaves room
// for both partial ends (n / 16 + 2 units).
template <int DH>
__device__ inline bool find_block(const KvView& p, Block<DH>& k) {
  const int64_t unit = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int lane = threadIdx.x & 63;
  int64_t at = 0;
  if (p.cu) {
    auto start = [&](int64_t b) { return (static_cast<int64_t>(p.cu[b]) >> 4) + 2 * b; };
    k.b = kv_find(p.B, unit, start);
    at = unit - start(k.b);
  } else {
    if (unit >= p.B) return false;
    k.b = unit;
  }
  if (!kv_run(kv_seq(p, k.b), at, k)) return false;
  k.head = blockIdx.y;
  k.c = lane % Block<DH>::kLanes;
  k.key0 = lane / Block<DH>::kLanes * Block<DH>::kKeys;
  return true;
}

// Rows of a call pass once, read by kv_write, written by kv_read: with ONCE, and in
// store4, they are marked so that they do not push the pages out of the caches
// (65 521 positions as above written and read back: 297 us, 356 unmarked).
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
template <bool ONCE, typename T>
__device__ inline void load4(const T* p, float (&x)[4]) {
  auto get = [](auto* at) {
    if constexpr (ONCE) return __builtin_nontemporal_load(at);
    else return *at;
  };
  if constexpr (sizeof(T) == 4) {
    const f32x4_t q = get(reinterpret_cast<const f32x4_t*>(p));
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = q[j];
  } else {
    const u32x2_t q = get(reinterpret_cast<const u32x2_t*>(p));
    x[0] = lo_f32(q[0]);
    x[1] = hi_f32(q[0]);
    x[2] = lo_f32(q[1]);
    x[3] = hi_f32(q[1]);
  }
}

// Four fp32 values as four codes.
template <int KIND>
__device__ inline uint32_t codes4(float a, float b, float c, float d) {
  if constexpr (KIND == SRW_KV_FP8) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
    return static_cast<uint32_t>(r);
  } else {
    auto u = [](float x) { return static_cast<uint32_t>(static_cast<int>(rintf(x))) & 0xffu; };
    return u(a) | u(b) << 8 | u(c) << 16 | u(d) << 24;
  }
}

template <int KIND, int DH, typename T>
__global__ __launch_bounds__(256) void kv_write_kernel(KvView p, KvRows r) {
  using B = Block<DH>;
  constexpr int ES = kv_bytes<KIND>(), KPL = B::kKeys;
  B k;
  if (!find_block(p, k)) return;
  const int page = kv_page(p, k.b, k.base);
  if (page < 0) return;
  const int64_t ph = static_cast<int64_t>(page) * p.H + k.head;
  const int slot = (k.base & (p.P - 1)) + k.key0;
  float xs[2][KPL][4];  // both tensors' rows are requested before either is used
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const T* src = static_cast<const T*>(which ? r.v : r.k) + k.head * (which ? r.v_head : r.k_head) + 4 * k.c;
    const int64_t ts = which ? r.v_token : r.k_token;
#pragma unroll
    for (int i = 0; i < KPL; ++i) {
      // (rows that are not in the call load one that is)
      load4<true>(src + (k.row + kv_in_run(k, k.key0 + i)) * ts, xs[which][i]);
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float(&x)[KPL][4] = xs[which];
    if constexpr (KIND != SRW_KV_BF16) {
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        // the bits of |x| order like the numbers, infinity and NaN above all
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t a = __float_as_uint(x[i][j]) & 0x7fffffffu;
          m = a > m ? a : m;
        }
        auto mx = [](float u, float w) {
          return __float_as_uint(u) > __float_as_uint(w) ? u : w;
        };
        float mf = __uint_as_float(m);
        const int lane = threadIdx.x & 63;
        mf = mx(mf, lane_xor<1>(mf, lane));
        mf = mx(mf, lane_xor<2>(mf, lane));
        mf = mx(mf, lane_xor<4>(mf, lane));
        mf = mx(mf, lane_xor<8>(mf, lane));
        if constexpr (B::kLanes == 32) mf = join16(mf, mx);
        constexpr float top = KIND == SRW_KV_INT8 ? 127.f : 448.f;
        const bool bad = __float_as_uint(mf) >= 0x7f800000u, zero = mf <= kKvTiny;
        const float inv = top / mf;
#pragma unroll
        for (int j = 0; j < 4; ++j) x[i][j] = bad || zero ? 0.f : x[i][j] * inv;
        if (k.c == 0 && k.key0 + i >= k.first && k.key0 + i < k.last)
          (which ? p.vs : p.ks)[ph * p.P + slot + i] = bad ? __uint_as_float(0x7fc00000u) : zero ? 0.f : mf / top;
      }
    }
    if (which == 0) {
      char* dst = p.k + (ph * p.P + slot) * (DH * ES) + 4 * k.c * ES;
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        if (k.key0 + i < k.first || k.key0 + i >= k.last) continue;
        if constexpr (KIND == SRW_KV_BF16)
          *reinterpret_cast<uint2*>(dst + i * (DH * ES)) =
              make_uint2(pack_bf16(x[i][0], x[i][1]), pack_bf16(x[i][2], x[i][3]));
        else
          *reinterpret_cast<uint32_t*>(dst + i * (DH * ES)) = codes4<KIND>(x[i][0], x[i][1], x[i][2], x[i][3]);
      }
    } else {
      char* dst = p.v + (ph * DH + 4 * k.c) * p.P * ES + slot * ES;
      const bool whole = k.key0 >= k.first && k.key0 + KPL <= k.last;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t w[KPL * ES / 4];
#pragma unroll
        for (int i = 0; i < KPL; i += 4 / ES) {
          if constexpr (KIND == SRW_KV_BF16)
            w[i / 2] = pack_bf16(x[i][j], x[i + 1][j]);
          else
            w[i / 4] = codes4<KIND>(x[i][j], x[i + 1][j], x[i + 2][j], x[i + 3][j]);
        }
        char* at = dst + static_cast<int64_t>(j) * p.P * ES;
        if (whole) {
          if constexpr (KPL * ES == 16)
            *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
          else if constexpr (KPL * ES == 8)
            *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
          else
            *reinterpret_cast<uint32_t*>(at) = w[0];
        } else {  // the other positions of the run hold other tokens
#pragma unroll
          for (int i = 0; i < KPL; ++i) {
            if (k.key0 + i < k.first || k.key0 + i >= k.last) continue;
            if constexpr (KIND == SRW_KV_BF16)
              reinterpret_cast<uint16_t*>(at)[i] = static_cast<uint16_t>(w[i / 2] >> (16 * (i & 1)));
            else
              reinterpret_cast<uint8_t*>(at)[i] = static_cast<uint8_t>(w[i / 4] >> (8 * (i & 3)));
          }
        }
      }
    }
  }
}

// Four codes as floats.
template <int KIND>
__device__ inline void values4(uint32_t w, float (&x)[4]) {
  if constexpr (KIND == SRW_KV_FP8) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = a[0];
    x[1] = a[1];
    x[2] = b[0];
    x[3] = b[1];
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) x[j] = static_cast<float>(static_cast<int8_t>(w >> (8 * j)));
  }
}

template <typename T>
__device__ inline void store4(T* p, const float (&x)[4]) {
  if constexpr (sizeof(T) == 4)
    __builtin_nontemporal_store(f32x4_t{x[0], x[1], x[2], x[3]}, reinterpret_cast<f32x4_t*>(p));
  else
    __builtin_nontemporal_store(u32x2_t{pack_bf16(x[0], x[1]), pack_bf16(x[2], x[3])}, reinterpret_cast<u32x2_t*>(p));
}

// The same blocks read back; positions without a page give zeros.
template <int KIND, int DH, typename T>
__global__ __launch_bounds__(256) void kv_read_kernel(KvView p, KvRows r) {
  using B = Block<DH>;
  constexpr int ES = kv_bytes<KIND>(), KPL = B::kKeys;
  B k;
  if (!find_block(p, k)) return;
  const int page = kv_page(p, k.b, k.base);
  const int64_t ph = static_cast<int64_t>(page < 0 ? 0 : page) * p.H + k.head;
  const int slot = (k.base & (p.P - 1)) + k.key0;
  T* out[2] = {static_cast<T*>(const_cast<void*>(r.k)) + k.head * r.k_head + 4 * k.c,
               static_cast<T*>(const_cast<void*>(r.v)) + k.head * r.v_head + 4 * k.c};
  float x[2][KPL][4] = {};
  if (page >= 0) {
    const char* src = p.k + (ph * p.P + slot) * (DH * ES) + 4 * k.c * ES;
    const char* vsrc = p.v + (ph * DH + 4 * k.c) * p.P * ES + slot * ES;
    if constexpr (KIND == SRW_KV_BF16) {
#pragma unroll
      for (int i = 0; i < KPL; ++i) load4<false>(reinterpret_cast<const uint16_t*>(src + i * (DH * ES)), x[0][i]);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < KPL; i += 4) {
          float t[4];
          load4<false>(reinterpret_cast<const uint16_t*>(vsrc + (static_cast<int64_t>(j) * p.P + i) * ES), t);
#pragma unroll
          for (int u = 0; u < 4; ++u) x[1][i + u][j] = t[u];
        }
    } else {
      uint32_t wk[KPL], wv[4][KPL / 4];
      float sc[2][KPL];
#pragma unroll
      for (int i = 0; i < KPL; ++i) wk[i] = *reinterpret_cast<const uint32_t*>(src + i * (DH * ES));
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < KPL / 4; ++i)
          wv[j][i] = *reinterpret_cast<const uint32_t*>(vsrc + static_cast<int64_t>(j) * p.P + 4 * i);
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        sc[0][i] = p.ks[ph * p.P + slot + i];
        sc[1][i] = p.vs[ph * p.P + slot + i];
      }
#pragma unroll
      for (int i = 0; i < KPL; ++i) {
        values4<KIND>(wk[i], x[0][i]);
#pragma unroll
        for (int j = 0; j < 4; ++j) x[0][i][j] *= sc[0][i];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int i = 0; i < KPL / 4; ++i) {
          float t[4];
          values4<KIND>(wv[j][i], t);
#pragma unroll
          for (int u = 0; u < 4; ++u) x[1][4 * i + u][j] = t[u] * sc[1][4 * i + u];
        }
    }
  }
#pragma unroll
  for (int i = 0; i < KPL; ++i) {
    if (k.key0 + i < k.first || k.key0 + i >= k.last) continue;
    store4(out[0] + (k.row + k.key0 + i) * r.k_token, x[0][i]);
    store4(out[1] + (k.row + k.key0 + i) * r.v_token, x[1][i]);
  }
}

template <bool WRITE, int KIND, int DH, typename T>
hipError_t launch_rows(const srw_kv_t& c, const KvRows& r, hipStream_t s) {
  const KvView p = kv_view(c);
  const int64_t units = c.cu ? (c.T >> 4) + 2 * c.B : c.B;
  const dim3 grid(static_cast<unsigned>((units + 3) / 4), static_cast<unsigned>(c.n_kv_heads));
  if constexpr (WRITE)
    hipLaunchKernelGGL((kv_write_kernel<KIND, DH, T>), grid, dim3(256), 0, s, p, r);
  else
    hipLaunchKernelGGL((kv_read_kernel<KIND, DH, T>), grid, dim3(256), 0, s, p, r);
  return hipGetLastError();
}

template <bool WRITE, typename T>
hipError_t rows_by_kind(const srw_kv_t& c, const KvRows& r, hipStream_t s) {
  auto by = [&](auto kind) {
    constexpr int K = decltype(kind)::value;
    return c.head_dim == 64 ? launch_rows<WRITE, K, 64, T>(c, r, s) : launch_rows<WRITE, K, 128, T>(c, r, s);
  };
  switch (c.kind) {
    case SRW_KV_BF16: return by(std::integral_constant<int, SRW_KV_BF16>{});
    case SRW_KV_INT8: return by(std::integral_constant<int, SRW_KV_INT8>{});
    default: return by(std::integral_constant<int, SRW_KV_FP8>{});
  }
}

bool aligned(const void* q, size_t a) { return q && !(reinterpret_cast<uintptr_t>(q) & (a - 1)); }

srw_status_t check_kv(const srw_kv_t* c) {
  if (!c) return SRW_EINVAL;
  if (c->B < 0 || c->T < 0 || c->n_pages < 0 || c->table_width < 0 || c->n_kv_heads < 1) return SRW_EINVAL;
  if (c->kind != SRW_KV_BF16 && c->kind != SRW_KV_INT8 && c->kind != SRW_KV_FP8) return SRW_EINVAL;
  if (c->head_dim < 1 || c->page_size < 1) return SRW_EINVAL;
  if (c->head_dim != 64 && c->head_dim != 128) return SRW_EUNSUPPORTED;
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1))) return SRW_EUNSUPPORTED;
  // grid dimensions and 32-bit positions
  if (c->n_kv_heads > 65535 || c->B > (1 << 24) || c->T > 0x7fffffff || c->n_pages > 0x7fffffff)
    return SRW_EUNSUPPORTED;
  if (c->table_width > 0x7fff0000 / c->page_size) return SRW_EUNSUPPORTED;
  if (!c->cu && c->T != c->B) return SRW_EINVAL;  // one token a sequence
  if (c->T == 0 || c->B == 0) return c->T == 0 ? SRW_OK : SRW_EINVAL;
  if (c->table_width > 0 && (!aligned(c->table, 4) || c->table_stride < c->table_width)) return SRW_EINVAL;
  if (!aligned(c->lens, 4) || (c->cu && !aligned(c->cu, 4))) return SRW_EINVAL;
  if (c->n_pages > 0) {
    if (!aligned(c->k, 16) || !aligned(c->v, 16)) return SRW_EINVAL;
    if (c->kind != SRW_KV_BF16 && (!aligned(c->k_scale, 16) || !aligned(c->v_scale, 16))) return SRW_EINVAL;
  }
  return SRW_OK;
}

// Rows of dtype at these strides, read or written four elements at a time.
srw_status_t check_rows(const srw_kv_t& c, const KvRows& r, int32_t dtype) {
  if (dtype != SRW_F32 && dtype != SRW_BF16) return SRW_EINVAL;
  if (c.T == 0) return SRW_OK;
  const size_t piece = dtype == SRW_F32 ? 16 : 8;
  if (!aligned(r.k, piece) || !aligned(r.v, piece)) return SRW_EINVAL;
  for (const int64_t st : {r.k_token, r.k_head, r.v_token, r.v_head})
    if (st < 0 || st % 4) return SRW_EINVAL;
  return SRW_OK;
}

srw_status_t check_attention(const srw_attention_t* a) {
  if (!a) return SRW_EINVAL;
  const srw_status_t st = check_kv(&a->kv);
  if (st != SRW_OK) return st;
  if (a->n_heads < 1 || a->n_heads % a->kv.n_kv_heads) return SRW_EINVAL;
  if (a->window < 0 || a->sinks < 0 || (a->sinks > 0 && a->window == 0) || a->max_new < 0) return SRW_EINVAL;
  if (!isfinite(a->scale)) return SRW_EINVAL;
  // rows of a call: tokens x heads
  if (a->kv.T > 0 && a->n_heads > 0x7fffffff / a->kv.T) return SRW_EUNSUPPORTED;
  return SRW_OK;
}

}  // namespace

hipError_t kv_write(const srw_kv_t& c, const KvRows& r, bool f32, hipStream_t s) {
  return f32 ? rows_by_kind<true, float>(c, r, s) : rows_by_kind<true, uint16_t>(c, r, s);
}
hipError_t kv_read(const srw_kv_t& c, const KvRows& r, bool f32, hipStream_t s) {
  return f32 ? rows_by_kind<false, float>(c, r, s) : rows_by_kind<false, uint16_t>(c, r, s);
}

}  // namespace srw

extern "C" {

srw_status_t srw_kv_write(const srw_kv_t* cache, const srw_kv_rows_t* rows, int32_t dtype, void* stream) {
  srw_status_t st = srw::check_kv(cache);
  if (st != SRW_OK) return st;
  if (!rows) return SRW_EINVAL;
  const srw::KvRows r{rows->k, rows->v, rows->k_token_stride, rows->k_head_stride, rows->v_token_stride,
                      rows->v_head_stride};
  st = srw::check_rows(*cache, r, dtype);
  if (st != SRW_OK) return st;
  if (cache->T == 0 || cache->n_pages == 0) return SRW_OK;
  (void)hipGetLastError();
  return srw::kv_write(*cache, r, dtype == SRW_F32, static_cast<hipStream_t>(stream)) == hipSuccess ? SRW_OK : SRW_EHIP;
}

srw_status_t srw_kv_read(const srw_kv_t* cache, const srw_kv_rows_t* rows, int32_t dtype, void* stream) {
  srw_status_t st = srw::check_kv(cache);
  if (st != SRW_OK) return st;
  if (!rows) return SRW_EINVAL;
  const srw::KvRows r{rows->k, rows->v, rows->k_token_stride, rows->k_head_stride, rows->v_token_stride,
                      rows->v_head_stride};
  st = srw::check_rows(*cache, r, dtype);
  if (st != SRW_OK) return st;
  if (cache->T == 0) return SRW_OK;
  (void)hipGetLastError();
  return srw::kv_read(*cache, r, dtype == SRW_F32, static_cast<hipStream_t>(stream)) == hipSuccess ? SRW_OK : SRW_EHIP;
}

srw_status_t srw_attention_workspace_size(const srw_attention_t* a, size_t* bytes) {
  const srw_status_t st = srw::check_attention(a);
  if (st != SRW_OK) return st;
  if (!bytes) return SRW_EINVAL;
  *bytes = a->kv.T == 0 ? 0 : srw::attention_workspace_bytes(*a);
  return SRW_OK;
}

srw_status_t srw_attention_plan(const srw_attention_t* a, int32_t* rows, int32_t* splits) {
  const srw_status_t st = srw::check_attention(a);
  if (st != SRW_OK) return st;
  if (!rows || !splits) return SRW_EINVAL;
  *rows = *splits = 0;
  if (a->kv.T > 0) srw::attention_plan(*a, rows, splits);
  return SRW_OK;
}

srw_status_t srw_attention(const srw_attention_t* a, void* workspace, size_t workspace_bytes, void* stream) {
  const srw_status_t st = srw::check_attention(a);
  if (st != SRW_OK) return st;
  if (a->kv.T == 0) return SRW_OK;
  // q rows are read 16 bytes at a time, out is written 8
  if (!srw::aligned(a->q, 16) || !srw::aligned(a->out, 16)) return SRW_EINVAL;
  if (a->q_token_stride < 0 || a->q_head_stride < 0 || a->q_token_stride % 8 || a->q_head_stride % 8) return SRW_EINVAL;
  const size_t need = srw::attention_workspace_bytes(*a);
  if (need > 0 && (!srw::aligned(workspace, 16) || workspace_bytes < need)) return SRW_EWORKSPACE;
  (void)hipGetLastError();
  return srw::attention(*a, static_cast<char*>(workspace), static_cast<hipStream_t>(stream)) == hipSuccess ? SRW_OK
                                                                                                         : SRW_EHIP;
}

}  // extern "C"

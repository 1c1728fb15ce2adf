/* CPU: the C entry points of page copies, the pages' index and choice, attention to
 * kept pages and sampling under AddressSanitizer and UndefinedBehaviorSanitizer: over
 * grids of calls up to the ends of their fields' ranges, sizes and the checks that
 * return before any launch.  No GPU work: every call here is refused on the host or
 * has nothing to do. */
#include <math.h>
#include <stdint.h>
#include <stdio.h>

#include "srw_amd.h"

static int failures = 0;
#define EXPECT(cond, ...)                                  \
  do {                                                     \
    if (!(cond)) {                                         \
      fprintf(stderr, "FAIL %s:%d: ", __FILE__, __LINE__); \
      fprintf(stderr, __VA_ARGS__);                        \
      fprintf(stderr, "\n");                               \
      ++failures;                                          \
    }                                                      \
  } while (0)
#define COUNT(a) (int)(sizeof(a) / sizeof((a)[0]))

static int32_t memory[64];
static const int64_t ends[] = {INT64_MIN, -1, 0, 1, 4, 1000, 0x7fffffff, (int64_t)1 << 40, INT64_MAX};
static const int32_t whole[] = {INT32_MIN, -1, 0, 1, 4, 1000, 0x7fffffff};
static long cases = 0;

static void copies(void) {
  static int32_t src[100], dst[100];
  for (int i = 0; i < 100; ++i) {
    src[i] = i;
    dst[i] = i; /* read and written: refused by the lists at the latest */
  }
  for (int l = 0; l < COUNT(ends); ++l)
    for (int p = 0; p < COUNT(ends); ++p)
      for (int b = 0; b < COUNT(ends); ++b)
        for (int s = 0; s < COUNT(ends); ++s)
          for (int n = 0; n < 2; ++n) {
            srw_kv_copy_t c = {{0}};
            for (int i = 0; i < 2; ++i) {
              c.src[i] = c.dst[i] = (char*)memory + 4 * i;
              c.page_bytes[i] = ends[b];
              c.src_layer_stride[i] = c.dst_layer_stride[i] = ends[s];
            }
            c.n_layers = ends[l];
            c.n_src_pages = c.n_dst_pages = ends[p];
            c.n_pairs = n ? 100 : 10;
            c.src_page = src;
            c.dst_page = dst;
            c.n_tensors = 1 + n;
            const srw_status_t st = srw_kv_copy(&c, NULL);
            EXPECT(st == SRW_EINVAL || st == SRW_EUNSUPPORTED || (st == SRW_OK && c.n_layers == 0), "status %d", st);
            ++cases;
          }
  for (int i = 0; i < COUNT(whole); ++i) {
    srw_kv_copy_t c = {{0}};
    c.n_tensors = whole[i];
    c.n_layers = c.n_src_pages = c.n_dst_pages = 1;
    c.n_pairs = 1;
    c.src_page = c.dst_page = src;
    EXPECT((srw_kv_copy(&c, NULL) == SRW_OK) == (whole[i] == 0), "%d tensors", whole[i]);
  }
}

static srw_kv_t pages(int kind, int64_t B, int64_t T, int64_t width, int P) {
  srw_kv_t c = {0};
  c.k = c.v = memory;
  c.k_scale = c.v_scale = (float*)memory;
  c.table = c.lens = c.cu = memory;
  c.B = B;
  c.T = T;
  c.n_pages = 100;
  c.table_width = c.table_stride = width;
  c.n_kv_heads = 2;
  c.head_dim = 64;
  c.page_size = P;
  c.kind = kind;
  return c;
}

static void kept(void) {
  for (int kind = 0; kind < 3; ++kind)
    for (int b = 0; b < COUNT(ends); ++b)
      for (int t = 0; t < COUNT(ends); ++t)
        for (int w = 0; w < COUNT(ends); ++w)
          for (int n = 0; n < COUNT(ends); ++n)
            for (int P = 16; P <= 256; P *= 16) {
              srw_attention_t a = {{0}};
              a.kv = pages(kind, ends[b], ends[t], ends[w], P);
              a.n_heads = 8;
              a.scale = 1.0f;
              size_t bytes = 12345;
              const srw_status_t st = srw_attention_kept_workspace_size(&a, ends[n], &bytes);
              EXPECT((st == SRW_OK) == (bytes != 12345), "status %d", st);
              if (st == SRW_OK && a.kv.T > 0)
                EXPECT(bytes <= (size_t)a.kv.T * 8 * 256 * (8 + 4 * 64) + 512, "%zu bytes", bytes);
              if (a.kv.T != 0) EXPECT(srw_attention_kept(&a, memory, ends[n], NULL, 0, NULL) != SRW_OK, "no q");
              srw_kv_select_t s = {{0}};
              s.kv = a.kv;
              s.index.codes = (int8_t*)memory;
              s.index.scale = (float*)memory;
              s.n_heads = 8;
              s.n = 4;
              s.last = 1;
              if (a.kv.T != 0) EXPECT(srw_kv_select(&s, NULL) != SRW_OK, "no q");
              const srw_kv_index_t none = {NULL, NULL};
              if (a.kv.T != 0) EXPECT(srw_kv_index(&a.kv, &none, NULL) != SRW_OK, "no index");
              ++cases;
            }
  for (int n = 0; n < COUNT(whole); ++n)
    for (int f = 0; f < COUNT(whole); ++f)
      for (int l = 0; l < COUNT(whole); ++l)
        for (int h = 0; h < COUNT(whole); ++h) {
          srw_kv_select_t s = {{0}};
          s.kv = pages(SRW_KV_INT8, 2, 0, 3, 16);
          s.n_heads = whole[h];
          s.n = whole[n];
          s.first = whole[f];
          s.last = whole[l];
          const int good = whole[h] > 0 && whole[h] % 2 == 0 && whole[f] >= 0 && whole[l] > 0 &&
                           (int64_t)whole[f] + whole[l] <= whole[n];
          EXPECT((srw_kv_select(&s, NULL) == SRW_OK) == good, "%d %d %d %d", whole[n], whole[f], whole[l], whole[h]);
          ++cases;
        }
}

static void samples(void) {
  const float numbers[] = {-1.0f, -0.0f, 0.0f, 1e-45f, 0.5f, 1.0f, 1.5f, INFINITY, NAN};
  for (int b = 0; b < COUNT(ends); ++b)
    for (int v = 0; v < COUNT(ends); ++v)
      for (int k = 0; k < COUNT(whole); ++k)
        for (int t = 0; t < COUNT(numbers); ++t)
          for (int p = 0; p < COUNT(numbers); ++p)
            for (int m = 0; m < COUNT(numbers); ++m) {
              srw_sample_t s = {0};
              s.logits = memory;
              s.u = (const float*)memory;
              s.token = (int64_t*)memory;
              s.B = ends[b];
              s.V = ends[v];
              s.temperature_all = numbers[t];
              s.top_k_all = whole[k];
              s.top_p_all = numbers[p];
              s.min_p_all = numbers[m];
              s.dtype = SRW_F32;
              size_t bytes = 12345;
              const srw_status_t st = srw_sample_workspace_size(&s, &bytes);
              EXPECT((st == SRW_OK) == (bytes != 12345), "status %d", st);
              if (st == SRW_OK && s.B > 0)
                EXPECT(s.top_k_all >= 0 && numbers[t] >= 0 && numbers[p] >= 0 && numbers[p] <= 1 && numbers[m] >= 0 &&
                           numbers[m] <= 1, "taken");
              s.u = NULL;
              EXPECT(srw_sample(&s, NULL, 0, NULL) != SRW_OK || s.B == 0, "no numbers");
              ++cases;
            }
}

int main(void) {
  copies();
  kept();
  samples();
  printf("%ld cases, %d failures\n", cases, failures);
  return failures != 0;
}

/* CPU: the paged cache's C entry points under AddressSanitizer and
 * UndefinedBehaviorSanitizer: descriptions, workspace sizes over a grid of calls up
 * to the ends of their fields' ranges, the checks that return before any launch.
 * No GPU work: every call here is refused on the host or has no tokens. */
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

static int32_t memory[64];

static srw_attention_t call(int kind, int dh, int P, int64_t width, int64_t B, int64_t T, int H, int G, int has_cu) {
  srw_attention_t a = {{0}};
  a.kv.k = a.kv.v = memory;
  if (kind != SRW_KV_BF16) a.kv.k_scale = a.kv.v_scale = (float*)memory;
  a.kv.table = a.kv.lens = memory;
  a.kv.cu = has_cu ? memory : NULL;
  a.kv.B = B;
  a.kv.T = T;
  a.kv.n_pages = 100;
  a.kv.table_width = a.kv.table_stride = width;
  a.kv.n_kv_heads = H;
  a.kv.head_dim = dh;
  a.kv.page_size = P;
  a.kv.kind = kind;
  a.n_heads = H * G;
  a.scale = 1.0f;
  return a;
}

static size_t size_of(const srw_attention_t* a) {
  size_t n = 12345;
  const srw_status_t st = srw_attention_workspace_size(a, &n);
  EXPECT(st == SRW_OK, "status %d", st);
  return n;
}

int main(void) {
  const int32_t most = 0x7fffffff;
  const int64_t widths[] = {0, 1, 9, 300, 8388000};
  const int64_t Bs[] = {1, 3, 64, 65536, 1 << 24};
  const int32_t windows[] = {0, 1, 64, 1000, most - 64, most};
  const int32_t sinks[] = {0, 1, 70, most - 63, most};
  const int32_t news[] = {0, 1, 40, most};
  long cases = 0;
  for (int kind = 0; kind < 3; ++kind)
    for (int dh = 64; dh <= 128; dh *= 2)
      for (int P = 16; P <= 256; P *= 2)
        for (int w = 0; w < 5; ++w)
          for (int b = 0; b < 5; ++b)
            for (int h = 1; h <= 64; h *= 8)
              for (int g = 1; g <= 16; g *= 4)
                for (int n = 0; n < 3; ++n) {
                  const int64_t T = n == 0 ? Bs[b] : n == 1 ? 300 : most / (h * g);
                  if (T * h * g > most) continue;
                  srw_attention_t a = call(kind, dh, P, widths[w], Bs[b], T, h, g, n > 0);
                  if (widths[w] > 0x7fff0000 / P) {
                    size_t bytes = 7;
                    EXPECT(srw_attention_workspace_size(&a, &bytes) == SRW_EUNSUPPORTED && bytes == 7, "width");
                    continue;
                  }
                  for (int x = 0; x < 6; ++x)
                    for (int s = 0; s < 5; ++s)
                      for (int m = 0; m < 4; ++m) {
                        if (sinks[s] && !windows[x]) continue;
                        a.window = windows[x];
                        a.sinks = sinks[s];
                        a.max_new = news[m];
                        const size_t bytes = size_of(&a);
                        /* a float2 and head_dim floats for each row of up to 1024 splits */
                        const double rows = (double)T * h * g;
                        EXPECT((double)bytes <= 1024 * rows * (8 + 4.0 * dh) + 512, "bytes %zu", bytes);
                        ++cases;
                        /* first tokens beyond what the table holds are all of them: the call of no window */
                        if (sinks[s] >= most - 63 && windows[x] >= most - 64) {
                          srw_attention_t all = a;
                          all.window = all.sinks = 0;
                          EXPECT(size_of(&all) == bytes, "sinks %d window %d: %zu, all: %zu", a.sinks, a.window, bytes,
                                 size_of(&all));
                        }
                      }
                  EXPECT(srw_attention(&a, NULL, 0, NULL) == SRW_EINVAL, "no q");
                }
  /* refusals, and calls with nothing to do */
  srw_attention_t a = call(SRW_KV_INT8, 64, 16, 3, 2, 0, 2, 2, 1);
  srw_kv_rows_t r = {memory, memory, 128, 64, 128, 64};
  EXPECT(srw_kv_write(&a.kv, &r, SRW_BF16, NULL) == SRW_OK, "nothing to write");
  EXPECT(srw_kv_read(&a.kv, &r, SRW_F32, NULL) == SRW_OK, "nothing to read");
  EXPECT(srw_attention(&a, NULL, 0, NULL) == SRW_OK, "nothing to attend");
  a.kv.T = 5;
  EXPECT(srw_kv_write(&a.kv, NULL, SRW_BF16, NULL) == SRW_EINVAL, "no rows");
  EXPECT(srw_kv_write(&a.kv, &r, 9, NULL) == SRW_EINVAL, "dtype");
  r.v_token_stride = -4;
  EXPECT(srw_kv_read(&a.kv, &r, SRW_BF16, NULL) == SRW_EINVAL, "stride");
  a.scale = NAN;
  EXPECT(srw_attention_workspace_size(&a, NULL) == SRW_EINVAL, "scale");
  printf("%ld sizes, %d failures\n", cases, failures);
  return failures != 0;
}

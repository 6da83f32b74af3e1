// The host-only side of the projections (kappa_amd/csrc/linear_host.cpp) driven on
// the CPU under -fsanitize=address,undefined (tests/test_linear_abi.py builds and
// runs it): overflow edges of the size checks, enum fields out of range, and the
// sizes over a sweep. Prints "linear checks: ok" and exits 0 when every check holds.
#include <stdio.h>
#include <string.h>

#include <initializer_list>

#include "linear.h"

using namespace kmoe_host;

static int g_fail = 0;

#define CHECK(cond)                                                            \
  do {                                                                         \
    if (!(cond)) {                                                             \
      ++g_fail;                                                                \
      fprintf(stderr, "%s:%d: check failed: %s\n", __FILE__, __LINE__, #cond); \
    }                                                                          \
  } while (0)

static void* const P = reinterpret_cast<void*>(0x1000);

static kmoe_linear_weight weight(int64_t in, int64_t out, int dtype = KMOE_DTYPE_I8) {
  kmoe_linear_weight w;
  memset(&w, 0, sizeof w);
  w.values = P;
  w.scale = reinterpret_cast<float*>(P);
  memcpy(&w.dtype, &dtype, sizeof dtype);
  w.in_features = in;
  w.out_features = out;
  return w;
}

static kmoe_lora adapters(int64_t L, int64_t R, int64_t in, int64_t out) {
  kmoe_lora l;
  memset(&l, 0, sizeof l);
  l.a = l.b = P;
  l.factor = reinterpret_cast<float*>(P);
  l.num_adapters = L;
  l.rank = R;
  l.in_features = in;
  l.out_features = out;
  return l;
}

int main() {
  const int64_t edge[] = {INT64_MIN, -1, 0, 1, 31, 32, 33, 127, 128, 129, 65536, 65537, (int64_t)1 << 20,
                          ((int64_t)1 << 20) + 1, INT64_MAX - 127, INT64_MAX};
  size_t a, b;
  for (int64_t in : edge)
    for (int64_t out : edge)
      for (int t : {(int)KMOE_DTYPE_F32, (int)KMOE_DTYPE_BF16, (int)KMOE_DTYPE_I8, -5, 77}) {
        const kmoe_linear_weight w = weight(in, out, t);
        const bool fits = in >= 1 && out >= 1 && in <= 65536 && out <= (1 << 20);
        const bool typed = t == KMOE_DTYPE_BF16 || t == KMOE_DTYPE_I8;
        const kmoe_status st = validate_linear_pack_bytes(&w, &a, &b);
        CHECK((st == KMOE_OK) == (fits && typed));
        if (st != KMOE_OK) continue;
        CHECK(a >= (size_t)in * out * (t == KMOE_DTYPE_I8 ? 1 : 2) && a % 4096 == 0 && b >= 4 * (size_t)out);
        size_t before = 0;
        for (int64_t T : {(int64_t)0, (int64_t)1, (int64_t)64, (int64_t)65, (int64_t)4096, (int64_t)1 << 20}) {
          const kmoe_lora l = adapters(3, 17, in, out);
          size_t n;
          CHECK(validate_linear_workspace_bytes(&w, T, KMOE_DTYPE_BF16, &l, &n) == KMOE_OK);
          CHECK(n >= before && n >= (size_t)T * (2 * in + 4 * 17));
          before = n;
        }
        for (int64_t T : {INT64_MIN, (int64_t)-1, ((int64_t)1 << 20) + 1, INT64_MAX})
          CHECK(validate_linear_workspace_bytes(&w, T, KMOE_DTYPE_BF16, nullptr, &a) != KMOE_OK);
        for (int64_t stride : edge) {
          LinearSpace sp;
          for (int64_t T : {(int64_t)0, (int64_t)1, (int64_t)2, (int64_t)1 << 20}) {
            const kmoe_status s = validate_linear(&w, T, P, KMOE_DTYPE_BF16, stride, nullptr, nullptr, nullptr, P, P,
                                                  (size_t)-1, &sp);
            // a span of 4 GiB or more, or rows that overlap, is refused
            if (T > 1) CHECK(s != KMOE_OK || (stride >= in && stride <= (((int64_t)1 << 32) / T) / 2));
          }
        }
      }
  for (int64_t L : edge)
    for (int64_t R : edge) {
      const kmoe_lora l = adapters(L, R, 200, 40);
      const bool ok = L >= 1 && L <= 1024 && R >= 1 && R <= 256;
      CHECK((validate_lora_pack_bytes(&l, &a, &b) == KMOE_OK) == ok);
      if (ok) CHECK(a >= (size_t)(2 * L * R * 200) && b >= (size_t)(2 * L * R * 40));
      for (int64_t first : edge)
        for (int64_t count : edge) {
          const kmoe_status s = validate_lora_pack(&l, first, count, R, P, P, reinterpret_cast<float*>(P));
          CHECK(s != KMOE_OK || (ok && first >= 0 && count >= 0 && first <= L && count <= L - first));
        }
    }
  for (int64_t T : edge)
    for (int64_t L : edge) {
      kmoe_lora_batch bt;
      memset(&bt, 0, sizeof bt);
      bt.adapter = bt.order = bt.sorted = bt.offsets = reinterpret_cast<int32_t*>(P);
      bt.tokens = T;
      bt.num_adapters = L;
      const bool ok = T >= 0 && T <= (1 << 20) && L >= 1 && L <= 1024;
      CHECK((validate_lora_sort_bytes(&bt, &a) == KMOE_OK) == ok);
      if (ok) CHECK(validate_lora_sort(bt.order, &bt, P, a) == KMOE_OK);
      if (ok && T > 0) CHECK(validate_lora_sort(bt.order, &bt, P, a - 1) == KMOE_ERR_WORKSPACE_TOO_SMALL);
    }
  if (g_fail) return 1;
  printf("linear checks: ok\n");
  return 0;
}

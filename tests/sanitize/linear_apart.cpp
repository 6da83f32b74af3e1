// validate_linear_apart (kappa_amd/csrc/linear_host.cpp) against every byte of small buffers:
// out, the workspace and x's rows at all offsets of one another. Prints "linear apart: ok"
// and exits 0 when the answers agree (tests/test_linear_buffers.py builds and runs it).
#include <stdio.h>
#include <string.h>

#include <initializer_list>

#include "linear.h"

using namespace kmoe_host;

int main() {
  long n = 0;
  for (const kmoe_dtype t : {KMOE_DTYPE_BF16, KMOE_DTYPE_I8})
    for (int tokens = 1; tokens <= 3; ++tokens)
      for (int in : {1, 5})
        for (int extra : {0, 1, 9})
          for (int out = 1; out <= 3; out += 2)
            for (int total : {0, 4, 16})
              for (int o = 0; o < 64; ++o)
                for (int s = 0; s < 64; s += 3) {
                  const int size = (int)dtype_size(t), stride = in + extra;
                  const int x = 24;  // out and the workspace start before, inside and behind the rows
                  bool xs[256] = {}, os[256] = {}, ss[256] = {};
                  for (int r = 0; r < tokens; ++r)
                    for (int i = 0; i < in * size; ++i) xs[x + r * stride * size + i] = true;
                  for (int i = 0; i < 2 * tokens * out; ++i) os[o + i] = true;
                  for (int i = 0; i < total; ++i) ss[s + i] = true;
                  bool meet = false;
                  for (int i = 0; i < 256; ++i) meet |= (xs[i] && os[i]) || (os[i] && ss[i]) || (ss[i] && xs[i]);
                  kmoe_linear_weight w;
                  memset(&w, 0, sizeof w);
                  w.in_features = in;
                  w.out_features = out;
                  auto at = [](int v) { return reinterpret_cast<void*>((uintptr_t)4096 + v); };
                  const kmoe_status st = validate_linear_apart(w, tokens, at(x), t, stride, at(o), total ? at(s) : nullptr,
                                                               LinearSpace{0, 0, (size_t)total});
                  if ((st != KMOE_OK) != meet) {
                    fprintf(stderr, "tokens %d in %d stride %d out %d at %d, workspace %d at %d: status %d\n", tokens, in,
                            stride, out, o, total, s, (int)st);
                    return 1;
                  }
                  ++n;
                }
  printf("linear apart: ok (%ld)\n", n);
  return 0;
}

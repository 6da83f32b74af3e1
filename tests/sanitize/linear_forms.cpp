// Which kernels a projection's call runs (the host-side choice in
// kappa_amd/csrc/linear_host.cpp): reads lines "T K N x_is_i8 w_is_i8 L R" (L = 0: no
// adapters) and prints a line for each. tests/test_linear_forms.py builds and runs it.
#include <stdio.h>
#include <string.h>

#include "linear.h"

using namespace kmoe_host;

int main() {
  long long T, K, N, L, R;
  int xi, wi;
  while (scanf("%lld %lld %lld %d %d %lld %lld", &T, &K, &N, &xi, &wi, &L, &R) == 7) {
    kmoe_linear_weight w;
    memset(&w, 0, sizeof w);
    w.dtype = wi ? KMOE_DTYPE_I8 : KMOE_DTYPE_BF16;
    w.in_features = K;
    w.out_features = N;
    const kmoe_dtype x = xi ? KMOE_DTYPE_I8 : KMOE_DTYPE_BF16;
    const char* const lora = L ? " lora" : "";
    const long long rows = (T + 15) / 16, cgs = padded_out(N) / 16, chunks = (K + 63) / 64;
    const long long steps = xi ? (chunks + 1) / 2 : chunks;
    switch (linear_form(w, T, x, L > 0)) {
      case LinearForm::kOne:
        printf("one %lldx%d%s\n", rows, decode_groups(cgs), chunks > 32 ? " deep" : "");
        break;
      case LinearForm::kSplit:
        printf("split %lld%s%s\n", rows, lora, steps > kmoe::kSplitSteps ? " deep" : "");
        break;
      case LinearForm::kTiles: {
        const char* name[] = {"32x64", "64x64", "64x128", "128x128", "256x256"};
        const LinearTile t = linear_tile(T, cgs, !xi && wi, L > 0);
        const LinearRounds r = linear_rounds(((T + 255) / 256) * ((cgs + 15) / 16));
        const bool quarters = t == LinearTile::k256x256 && r.blocks > r.whole;
        printf("%s%s%s%s", name[(int)t], quarters ? " quarters" : "", lora, steps > 8 ? " deep" : "");
        if (L) {
          const LoraShrink s = lora_shrink(T, R, L);
          printf(", shrink %d%s", s.groups, chunks > 16 * (s.groups == 1 ? 4 : 2) ? " again" : "");
        }
        printf("\n");
      }
    }
  }
  return 0;
}

// Plays the bins of csrc/gv_shares.h through on the host: whether values further down are in the same bins or in later ones, the largest in the first.
#include <math.h>
#include <stdio.h>

#include <initializer_list>

#include "../gevva_b200/csrc/gv_shares.h"

int main() {
  bool ascending = true, first = true, last = true, wide = true;
  for (int count : {128, 256, 1024})
    for (float high : {0.0f, 1e-37f, 2e-45f, 1.0f, -30.0f, 1e30f})
      for (int e = -150; e < 127; ++e) {
        const float low = static_cast<float>(high - ldexp(1.0, e)), extent = high - low;
        if (!(extent > 0.0f) || !isfinite(extent)) continue;
        const float per = gv::bins_for_one(count, extent);
        int at = 0;
        for (int i = 0; i <= 500; ++i) {
          const float x = fminf(fmaxf(static_cast<float>(high - i / 500.0 * (static_cast<double>(high) - low)), low), high);
          const int bin = gv::bin_at(high - x, per, count);
          first &= i > 0 || bin == 0;
          ascending &= bin >= at;
          at = bin;
        }
        last &= at <= count - 1;
        wide &= extent < 1e-30f || at == count - 1;
      }
  printf("%d %d %d %d\n", ascending, first, last, wide);
  return 0;
}

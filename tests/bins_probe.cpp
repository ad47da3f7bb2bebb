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
  // the same by halves, from one end of the numbers to the other and with infinite values among them
  const float most = 3.402823466e38f;
  for (float high : {most, 1e38f, 1.0f, 0.0f, 2e-45f, -1e30f})
    for (float low : {-most, -1e36f, -3e31f, -1.0f, -1e-45f, 0.5f}) {
      if (!(low < high)) continue;
      const float per = gv::bins_for_one(1024, gv::half_distance(high, low));
      first &= gv::bin_at(gv::half_distance(high, INFINITY), per, 1024) == 0 && gv::bin_at(gv::half_distance(high, high), per, 1024) == 0;
      int at = 0;
      for (int i = 0; i <= 500; ++i) {
        const float x = fmaxf(static_cast<float>(high - i / 500.0 * (static_cast<double>(high) - low)), low);
        const int bin = gv::bin_at(gv::half_distance(high, x), per, 1024);
        ascending &= bin >= at;
        at = bin;
      }
      wide &= static_cast<double>(high) - low < 1e-30 || at == 1023;
    }
  printf("%d %d %d %d\n", ascending, first, last, wide);
  return 0;
}

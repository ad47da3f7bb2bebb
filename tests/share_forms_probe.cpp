// Plays the choice of the plain form of shares (csrc/gv_shares.h) through on the host, from very low temperatures to high ones.  Prints the largest
// relative error of a share of up to kShareOctaves as a power of two, the largest share of what is below, and whether ordinary rows have the form.
#include <math.h>
#include <stdio.h>

#include <initializer_list>

#include "../gevva_b200/csrc/gv_shares.h"

int main() {
  static const double table[] = GV_EXP2_TABLE_INIT;
  long double worst = 0, most_below = 0;
  bool ordinary = true, in_range = true;
  int fitting = 0;
  for (float largest : {0.0f, 1e-30f, 0.1f, 1.0f, 10.0f, 17.3f, 20.0f, 88.0f, 1e4f, 3e29f, -0.3f, -10.0f, -1e6f, -9e29f})
    for (double exponent = -30; exponent < 30; exponent += 0.0625) {
      const float temperature = static_cast<float>(pow(10.0, exponent));
      if (!(temperature > 1e-30f && temperature < 1e30f)) continue;
      const double degrees = temperature, scale = 1.4426950408889634074 * gv::kExp2Entries / degrees;
      const gv::PlainRange range = gv::plain_range(largest, degrees);
      if (fabsf(largest) <= 100.0f && temperature >= 1e-6f && temperature <= 1e6f) ordinary &= range.fits;
      if (!range.fits) continue;
      ++fitting;
      // the floats next to the largest and next to the cut, and some between and below
      float near = largest, low = range.cut;
      for (int i = 0; i < 240; ++i) {
        float x;
        if (i < 80) x = near, near = nextafterf(near, -INFINITY);
        else if (i < 120) x = low, low = nextafterf(low, INFINITY);
        else x = static_cast<float>(largest - (i - 119) / 100.0 * (static_cast<double>(largest) - range.cut));
        const float clamped = fmaxf(x, range.cut);
        if (clamped > largest) continue;
        const uint32_t n = gv::share_whole(clamped - largest, static_cast<float>(scale));
        const double share = gv::share_with(static_cast<double>(clamped) - largest, scale, n, table, 1);
        const long double octaves = (static_cast<long double>(clamped) - largest) / degrees * 1.442695040888963407359924681001892137L;
        in_range &= share >= 0.0 && share <= 1.0;
        if (octaves > -static_cast<long double>(gv::kShareOctaves)) worst = fmaxl(worst, fabsl(share / exp2l(octaves) - 1));
        else most_below = fmaxl(most_below, share);
      }
    }
  printf("%.2f %.2f %d %d %d\n", static_cast<double>(log2l(worst)), static_cast<double>(log2l(most_below)), ordinary, in_range, fitting);
  return 0;
}

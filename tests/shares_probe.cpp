// Plays csrc/gv_shares.h through on the host against long double: prints the largest relative errors as powers of two.
#include <math.h>
#include <stdio.h>
#include <stdlib.h>

#include <initializer_list>

#include "../gevva_b200/csrc/gv_shares.h"

int main() {
  static const double table[] = GV_EXP2_TABLE_INIT;
  long double worst_table = 0, worst_rest = 0, worst_finely = 0, worst_with = 0, worst_of = 0;
  for (int j = 0; j < gv::kExp2Entries; ++j) worst_table = fmaxl(worst_table, fabsl(table[j] / exp2l(j / 32.0L) - 1));
  for (int i = -505000; i <= 505000; ++i) {
    const double f = i * 1e-6;
    const long double want = exp2l(static_cast<long double>(f) / 32);
    worst_rest = fmaxl(worst_rest, fabsl(gv::exp2_rest(f) / want - 1));
    worst_finely = fmaxl(worst_finely, fabsl(gv::exp2_rest_finely(f) / want - 1));
  }
  srand48(7);
  for (int i = 0; i < 2000000; ++i) {
    const float x = static_cast<float>(drand48() * 40 - 20), top = static_cast<float>(x + drand48() * 90);
    const double scale = 1.4426950408889634074 * gv::kExp2Entries / (0.7 + drand48()), distance = static_cast<double>(x) - top;
    const uint32_t n = gv::share_whole(x - top, static_cast<float>(scale));
    const long double want = exp2l(static_cast<long double>(distance) * scale / 32);
    worst_with = fmaxl(worst_with, fabsl(gv::share_with(distance, scale, n, table, 1) / want - 1));
    worst_of = fmaxl(worst_of, fabsl(gv::share_of(distance, scale, table, 1) / want - 1));
  }
  // exactly one for the largest, whatever the scale; zero far below
  bool ends = true;
  for (double scale : {1e-30, 0.3, 46.0, 1e6, 1e45}) {
    ends &= gv::share_of(0.0, scale, table, 1) == 1.0;
    if (scale < 1e30) ends &= gv::share_with(0.0, scale, gv::share_whole(0.0f, static_cast<float>(scale)), table, 1) == 1.0;
  }
  ends &= gv::share_of(-1e6, 46.0, table, 1) == 0.0 && gv::share_of(-INFINITY, 46.0, table, 1) == 0.0;
  // floats as doubles
  bool wide = true;
  for (uint32_t bits = 0x00800000u; bits < 0x7f800000u; bits += 9973u) {
    float x;
    memcpy(&x, &bits, 4);
    wide &= gv::wide_of(x) == static_cast<double>(x) && gv::wide_of(-x) == -static_cast<double>(x);
  }
  wide &= fabs(gv::wide_of(0.0f)) < 1e-38 && fabs(gv::wide_of(-0.0f)) < 1e-38 && fabs(gv::wide_of(1e-45f)) < 2e-38;
  wide &= gv::wide_of(3.402823466e38f) == static_cast<double>(3.402823466e38f);
  // the order of floats
  const float values[] = {-INFINITY, -3.402823466e38f, -1.0f, -1e-45f, 0.0f, 1e-45f, 1.0f, 3.402823466e38f, INFINITY};
  bool order = gv::order_of(-INFINITY) == gv::kNothing && gv::order_of(-0.0f) == gv::order_of(0.0f);
  for (int i = 0; i < 9; ++i) {
    order &= gv::value_of(gv::order_of(values[i])) == values[i];
    if (i) order &= gv::order_of(values[i]) > gv::order_of(values[i - 1]);
  }
  printf("%.2f %.2f %.2f %.2f %.2f %d %d %d\n", static_cast<double>(log2l(worst_table)), static_cast<double>(log2l(worst_rest)),
         static_cast<double>(log2l(worst_finely)), static_cast<double>(log2l(worst_with)), static_cast<double>(log2l(worst_of)), ends, wide, order);
  return 0;
}

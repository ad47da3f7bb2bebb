// Arithmetic of the shares that tokens have, for host and device (tests/shares_probe.cpp plays it through on the host).
//
// A token is taken where a running sum over the vocabulary passes a random number's share of the whole.  Among 2^18 nearly equal shares a
// border lies within 2^-18 / 2 of the number on average, and 2^18 terms that are each off by e in the same direction move it by up to
// e: terms in 32 bits (e = 2^-24) would give another token once in about a hundred flat rows.  Shares and their sums
// are in 64 bits therefore.
#pragma once

#include <math.h>
#include <stdint.h>
#include <string.h>

#ifdef __CUDACC__
#define GV_SHARES_HD __host__ __device__ __forceinline__
#else
#define GV_SHARES_HD inline
#endif

namespace gv {

// 2^(j / 32), correctly rounded.
#define GV_EXP2_TABLE_INIT                                                                                                    \
  {                                                                                                                           \
    0x1.0000000000000p+0, 0x1.059b0d3158574p+0, 0x1.0b5586cf9890fp+0, 0x1.11301d0125b51p+0, 0x1.172b83c7d517bp+0,             \
    0x1.1d4873168b9aap+0, 0x1.2387a6e756238p+0, 0x1.29e9df51fdee1p+0, 0x1.306fe0a31b715p+0, 0x1.371a7373aa9cbp+0,             \
    0x1.3dea64c123422p+0, 0x1.44e086061892dp+0, 0x1.4bfdad5362a27p+0, 0x1.5342b569d4f82p+0, 0x1.5ab07dd485429p+0,             \
    0x1.6247eb03a5585p+0, 0x1.6a09e667f3bcdp+0, 0x1.71f75e8ec5f74p+0, 0x1.7a11473eb0187p+0, 0x1.82589994cce13p+0,             \
    0x1.8ace5422aa0dbp+0, 0x1.93737b0cdc5e5p+0, 0x1.9c49182a3f090p+0, 0x1.a5503b23e255dp+0, 0x1.ae89f995ad3adp+0,             \
    0x1.b7f76f2fb5e47p+0, 0x1.c199bdd85529cp+0, 0x1.cb720dcef9069p+0, 0x1.d5818dcfba487p+0, 0x1.dfc97337b9b5fp+0,             \
    0x1.ea4afa2a490dap+0, 0x1.f50765b6e4540p+0                                                                                \
  }
constexpr int kExp2Entries = 32;

// 2^f / 32nd for a remainder of at most a little over half a 32nd: four terms of the exponential's series, of which the first and the third take
// over what the best polynomial of their degree has for the fifth, x^5 / 120 ~ (5/4 a^2 x^3 - 5/16 a^4 x) / 120 for |x| <= a = ln 2 / 64;
// off by a^5 / 1920 = 2^-43.5 of itself.  One for a remainder of zero.
GV_SHARES_HD double exp2_rest(double f) {
  double p = 0x1.3b2ab6fba4e77p-27;
  p = p * f + 0x1.c6b167e549176p-20;
  p = p * f + 0x1.ebfbdff82c58fp-13;
  p = p * f + 0x1.62e42fef6d01bp-6;
  return p * f + 1.0;
}
// The same with a term more (the sixth's taken over in the same way, x^6 / 720 ~ (3/2 a^2 x^4 - 9/16 a^4 x^2 + a^6 / 32) / 720, its last part
// left out): off by a^6 / 11520 = 2^-52.7.
GV_SHARES_HD double exp2_rest_finely(double f) {
  double p = 0x1.5d87fe78a6731p-35;
  p = p * f + 0x1.3b2b301f0c04ap-27;
  p = p * f + 0x1.c6b08d704a0c0p-20;
  p = p * f + 0x1.ebfbdff7feebap-13;
  p = p * f + 0x1.62e42fefa39efp-6;
  return p * f + 1.0;
}
// value * 2^floor(n / 32), for n by its low bits (any multiple of 2^17 more is the same), where that is a normal number.
GV_SHARES_HD double scaled_by(double value, uint32_t n) {
  const uint32_t exponent = (n >> 5) * (1u << 20);
#ifdef __CUDA_ARCH__
  return __hiloint2double(__double2hiint(value) + static_cast<int>(exponent), __double2loint(value));
#else
  uint64_t bits;
  memcpy(&bits, &value, 8);
  bits += static_cast<uint64_t>(exponent) << 32;
  memcpy(&value, &bits, 8);
  return value;
#endif
}

// Shares below 2^-200 of the largest are none: a sum in 64 bits does not notice them.
constexpr float kShareOctaves = 200.0f;

// distance * scale in whole 32nds of an octave, from 32 bits: the number stands in the low bits, kShareWhole more.  |distance * scale| <= 2^21.
constexpr uint32_t kShareWhole = 0x4b400000u;
GV_SHARES_HD uint32_t share_whole(float distance, float scale) {
#ifdef __CUDA_ARCH__
  return __float_as_uint(__fmaf_rn(distance, scale, 12582912.0f));
#else
  const float t = __builtin_fmaf(distance, scale, 12582912.0f);
  uint32_t bits;
  memcpy(&bits, &t, 4);
  return bits;
#endif
}
// 2^(distance * scale / 32) with its whole part as given; `table` has entry j at [j * stride].  The whole part may be off by a little (it comes from
// 32 bits): the rest is what it leaves.
template <bool kFinely = false>
GV_SHARES_HD double share_with(double distance, double scale, uint32_t n, const double* table, int stride) {
  // 2^52 and the bits, as a number of 64 bits, without a conversion
#ifdef __CUDA_ARCH__
  const double whole = __hiloint2double(0x43300000, static_cast<int>(n)) - (0x1p52 + kShareWhole);
  const double rest = __fma_rn(distance, scale, -whole);
#else
  const double whole = static_cast<double>(n) - static_cast<double>(kShareWhole);
  const double rest = __builtin_fma(distance, scale, -whole);
#endif
  return scaled_by((kFinely ? exp2_rest_finely(rest) : exp2_rest(rest)) * table[(n & (kExp2Entries - 1)) * stride], n);
}

// The same for any finite scale, zero below 2^-1020.
GV_SHARES_HD double share_of(double distance, double scale, const double* table, int stride) {
  constexpr double kWhole = 0x1.8p52;  // a sum with it is rounded to a whole number, which stands in its low bits
  if (!(distance * scale > -1020.0 * kExp2Entries)) return 0.0;
#ifdef __CUDA_ARCH__
  const double near = __fma_rn(distance, scale, kWhole), whole = near - kWhole, rest = __fma_rn(distance, scale, -whole);
  const uint32_t n = static_cast<uint32_t>(__double2loint(near));
#else
  const double near = __builtin_fma(distance, scale, kWhole), whole = near - kWhole, rest = __builtin_fma(distance, scale, -whole);
  const uint32_t n = static_cast<uint32_t>(static_cast<int>(whole));
#endif
  return scaled_by(exp2_rest(rest) * table[(n & (kExp2Entries - 1)) * stride], n);
}

// From which value on the plain form works shares out of uncapped values: values below `cut` count as `cut`, kShareOctaves below the largest, rounded
// down to 32 bits.  Where a step of 32 bits at the largest is many temperatures, that is thousands of octaves down, which an exponent's bits do not
// hold, or the largest itself: the plain form fits between kShareOctaves (less one, for rounding) and twice as many.
struct PlainRange {
  float cut;
  bool fits;
};
GV_SHARES_HD PlainRange plain_range(float largest, double degrees) {
  const double bound = static_cast<double>(largest) - kShareOctaves * 0.69314718055994530942 * degrees;
#ifdef __CUDA_ARCH__
  const float down = __double2float_rd(bound);
#else
  float down = static_cast<float>(bound);
  if (down > bound) down = nextafterf(down, -INFINITY);
#endif
  const float cut = fmaxf(down, -3.402823466e38f);
  const double octaves = (static_cast<double>(largest) - cut) / degrees * 1.4426950408889634074;
  return {cut, fabsf(largest) < 1e30f && cut > -1e30f && octaves >= kShareOctaves - 1.0f && octaves <= 2.0f * kShareOctaves};
}

// A float as a double by three whole-number operations, which leave the pipe of conversions free.  Exact for normal numbers; zero and what is next
// to it come out as about 2^-127, which no sum with a number of ordinary size notices.  Finite ones only.
GV_SHARES_HD double wide_of(float x) {
#ifdef __CUDA_ARCH__
  const int bits = __float_as_int(x);
  return __hiloint2double(((bits >> 3) & static_cast<int>(0x8fffffffu)) + (896 << 20), bits << 29);
#else
  int32_t bits;
  memcpy(&bits, &x, 4);
  const uint32_t high = (static_cast<uint32_t>(bits >> 3) & 0x8fffffffu) + (896u << 20);
  const uint64_t both = static_cast<uint64_t>(high) << 32 | static_cast<uint32_t>(bits) << 29;
  double y;
  memcpy(&y, &both, 8);
  return y;
#endif
}

// Order of floats as whole numbers; zeros of both signs are one number.  Everything that may be taken, infinity among it, is above
// kNothing (minus infinity's).
constexpr uint32_t kNothing = 0x007fffffu;
GV_SHARES_HD uint32_t order_of(float x) {
  x += 0.0f;
  uint32_t bits;
#ifdef __CUDA_ARCH__
  bits = __float_as_uint(x);
#else
  memcpy(&bits, &x, 4);
#endif
  return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
GV_SHARES_HD float value_of(uint32_t order) {
  const uint32_t bits = order & 0x80000000u ? order & 0x7fffffffu : ~order;
#ifdef __CUDA_ARCH__
  return __uint_as_float(bits);
#else
  float x;
  memcpy(&x, &bits, 4);
  return x;
#endif
}

// Half of what `x` is below `high`.
GV_SHARES_HD float half_distance(float high, float x) {
#ifdef __CUDA_ARCH__
  return __fmaf_rn(x, -0.5f, 0.5f * high);
#else
  return __builtin_fmaf(x, -0.5f, 0.5f * high);
#endif
}
// How many of `count` bins of equal width one has, for bins that reach over `extent`.  A number of 32 bits: of an extent so small that they
// would be more, fewer bins are in use.  (With infinitely many the largest, at a distance of zero, would be none of them.)
GV_SHARES_HD float bins_for_one(int count, float extent) { return fminf(static_cast<float>(count - 1) / extent, 3.402823466e38f); }
// Which one a distance is in, its count a power of two; of no number, or one beyond the bins, any.
GV_SHARES_HD int bin_at(float distance, float per, int count) { return static_cast<int>(share_whole(distance, per) & static_cast<uint32_t>(count - 1)); }
static_assert(kShareWhole % 4096 == 0, "the bits behind a whole number");

}  // namespace gv

// Numbers of sampling.hip that every compiler has: also a host's, whose checks of arithmetic know
// what the GPU does without a word (a conversion that overflows, a NaN that becomes 0).
#pragma once

namespace mzk {

constexpr int kBins = 1024, kRest = kBins - 1;  // bins of a histogram; the last takes what is too small to count, 2^-51
constexpr double kPerOctave = 20.0;
constexpr double kLog2eD = 1.4426950408889634074, kLn2D = 0.69314718055994530942;

// 2^t for t <= 1000, to 2^-51 of itself: the power series of exp(f ln 2) for |f| <= 1/2, whose first term left out
// is (ln 2 / 2)^13 / 13! = 1.7e-16.  Of NaN and of t below -1100 0.
__device__ __forceinline__ double exp2_of(double t) {
  t = __builtin_fmax(t, -1100.0);
  const double n = __builtin_rint(t);
  const double x = (t - n) * kLn2D;
  double e = 1.0 / 479001600.0;
  e = __builtin_fma(e, x, 1.0 / 39916800.0);
  e = __builtin_fma(e, x, 1.0 / 3628800.0);
  e = __builtin_fma(e, x, 1.0 / 362880.0);
  e = __builtin_fma(e, x, 1.0 / 40320.0);
  e = __builtin_fma(e, x, 1.0 / 5040.0);
  e = __builtin_fma(e, x, 1.0 / 720.0);
  e = __builtin_fma(e, x, 1.0 / 120.0);
  e = __builtin_fma(e, x, 1.0 / 24.0);
  e = __builtin_fma(e, x, 1.0 / 6.0);
  e = __builtin_fma(e, x, 0.5);
  e = __builtin_fma(e, x, 1.0);
  e = __builtin_fma(e, x, 1.0);
  return __builtin_ldexp(e, static_cast<int>(n));
}

// The weight of a logit in units of 2^-scale of the largest one's, at s bins a logit.  Values above a row's largest, of which it has no
// tokens, are weighed too: as that, so that 0 of them are 0 (at a small temperature they are any number of octaves above it).
__device__ __forceinline__ double weight_of(float l, float largest, double s, int scale) {
  const double bins = (static_cast<double>(__builtin_fminf(l, largest)) - static_cast<double>(largest)) * s;
  return exp2_of(bins / kPerOctave) * __builtin_ldexp(1.0, scale);  // (a NaN, of -inf at an infinite temperature, is 0)
}

constexpr int kNoTop = -0x7fffffff;  // the largest bin of no token

// The bin above which a survey's bins are kept whose largest is `top`.
__device__ __forceinline__ double bottom_of(int top) { return static_cast<double>(top) - kRest; }

constexpr int kCopies = 2;  // of each bin, side by side, by the lane

// The offset in bytes of the place of bin n, n mod kBins; n, however far, in the low bits of n + 3 2^51.
__device__ __forceinline__ int place_of(double sum) {
  return static_cast<int>(static_cast<unsigned>(__builtin_bit_cast(unsigned long long, sum)) * (8u * kCopies) & 8u * kCopies * kRest);
}

}  // namespace mzk

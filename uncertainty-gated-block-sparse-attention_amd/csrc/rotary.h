// Rotary positions: pair j < pairs of a head's dims turns by the angle pos * f_j,
//
//   y_a = m (x_a cos - x_b sin),   y_b = m (x_b cos + x_a sin),
//
// (a, b) = (j, j + pairs) or, interleaved, (2 j, 2 j + 1); dims from 2 pairs on
// pass.  The table holds f_j / 2 pi in 64 bits: a position of 2^20 turns the first
// pair 1.7e5 times, and 32 bits would leave 2^-7 of a turn of it; after the whole turns
// are taken off 32 bits are enough.
#pragma once

#include "common.h"
#include "launch.h"

namespace ugbsa {

// cos and sin (times m) of pos * turns turns: whole quarters are taken off in 64
// bits, then x in [-pi/4, pi/4] goes through the Taylor series, whose first terms left
// out are x^11 / 11! < 2^-29 and x^12 / 12! < 2^-33.  Off by less than 2^-22 from what
// is done in 32 bits, mostly the angle's two roundings, and from those in 64 bits by
// 2.4 |pos| f 2^-53: the product's (2^-53 of it), the table's f / 2 pi (as much) and its 2 pi's
// (2^-54.5).  That is 2^-26 at 2^26 radians, and passes 2^-22 at 2^30.
__device__ __forceinline__ void turn_cos_sin(double pos, double turns, float m, float& cs, float& sn) {
  const double u = pos * turns * 4.0;
  const double n = __builtin_rint(u);
  const float x = static_cast<float>(u - n) * 1.57079632679489661923f;
  const int quarter = static_cast<int>(n - 4.0 * __builtin_floor(n * 0.25));
  const float z = x * x;
  float s = __builtin_fmaf(z, 1.f / 362880.f, -1.f / 5040.f);
  s = __builtin_fmaf(z, s, 1.f / 120.f);
  s = __builtin_fmaf(z, s, -1.f / 6.f);
  s = __builtin_fmaf(z * x, s, x);
  float c = __builtin_fmaf(z, -1.f / 3628800.f, 1.f / 40320.f);
  c = __builtin_fmaf(z, c, -1.f / 720.f);
  c = __builtin_fmaf(z, c, 1.f / 24.f);
  c = __builtin_fmaf(z, c, -0.5f);
  c = __builtin_fmaf(z, c, 1.f);
  cs = (quarter & 1) ? s : c;
  sn = (quarter & 1) ? c : s;
  cs *= (quarter == 1 || quarter == 2) ? -m : m;
  sn *= quarter >= 2 ? -m : m;
}

// The two values of a pair, turned, as fp32 values that no instruction has rounded to 16 bits
// in the same step: the caller's rounding is the same whatever is compiled around it, so
// that keys turned as they are written have the bits of keys turned before.
__device__ __forceinline__ void turn_pair(float a, float b, float cs, float sn, float& ya, float& yb) {
  ya = __builtin_fmaf(a, cs, -(b * sn));
  yb = __builtin_fmaf(b, cs, a * sn);
  asm("" : "+v"(ya), "+v"(yb));
}

}  // namespace ugbsa

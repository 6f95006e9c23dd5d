// The quotient that an e4m3 code is the rounding of, without a division for each element.

#pragma once

#include <cmath>

#ifdef __HIPCC__
#define ROOST_BOTH_SIDES __host__ __device__ __forceinline__
#else
#define ROOST_BOTH_SIDES inline
#endif

namespace roost {

// Scales between these, and their reciprocals and remainders, stay clear of f32's smallest and largest numbers: a remainder is
// a multiple of 2^-46 of quotient times scale, so exact for every quotient that is not far below e4m3's smallest code.
constexpr float kQuotientLow = 0x1p-90f, kQuotientHigh = 0x1p126f;

// y / scale to f32, given inverse = 1 / scale rounded to nearest and a scale within those bounds: the product is off by up to
// two units in the last place, the remainder's share brings it back. Wherever the quotient lies next to a midpoint of two e4m3
// values the result is the correctly rounded one (tests/quotient_codes.cpp goes through all of them), so the codes are
// those of a division.
ROOST_BOTH_SIDES float Quotient(float y, float scale, float inverse) {
  const float q = y * inverse;
  return fmaf(fmaf(-q, scale, y), inverse, q);
}

}  // namespace roost

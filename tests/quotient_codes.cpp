// Holds roost_amd/csrc/quotient.h against f32 division next to every midpoint of two e4m3 values: all mantissas of the scale,
// all mantissas that a midpoint has, the six values around their product. Powers of two change nothing within the bounds that
// the header gives, which the scales at both ends of them show.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <cstring>

#include "quotient.h"

static float Near(float v, int steps) {
  uint32_t b;
  std::memcpy(&b, &v, 4);
  b += steps;
  std::memcpy(&v, &b, 4);
  return v;
}

int main(int argc, char** argv) {
  const uint32_t stride = argc > 1 ? std::atoi(argv[1]) : 1;
  // Normal codes have 3 bits behind the first, so their midpoints 4; half steps of subnormal codes are odd numbers up to 15.
  const float mids[] = {17 / 16.f, 19 / 16.f, 21 / 16.f, 23 / 16.f, 25 / 16.f, 27 / 16.f, 29 / 16.f, 31 / 16.f,
                        1.f,       3 / 2.f,   5 / 4.f,   7 / 4.f,   9 / 8.f,   11 / 8.f,  13 / 8.f,  15 / 8.f};
  // The largest midpoint is 432 (27 * 16), the smallest 2^-10.
  struct End { float scale, top; } ends[] = {{1.f, 1.f}, {roost::kQuotientLow, 0x1p-10f}, {roost::kQuotientHigh / 2, 1.f},
                                             {0x1p-60f, 0x1p8f}};
  unsigned long wrong = 0, tried = 0;
  for (const End& end : ends)
    for (uint32_t m = 0; m < 1u << 23; m += &end == ends ? stride : 97 * stride) {
      const float scale = std::ldexp(1.0f + m * 0x1p-23f, std::ilogb(end.scale)), inverse = 1.0f / scale;
      for (const float mid : mids) {
        const float want = mid * end.top, y0 = want * scale;
        if (!std::isfinite(y0)) continue;
        for (int k = -3; k <= 3; ++k) {
          const float y = Near(y0, k), exact = y / scale, got = roost::Quotient(y, scale, inverse);
          ++tried;
          // Below, at or above the midpoint alike.
          const bool same = (got < want) == (exact < want) && (got > want) == (exact > want);
          if (!same && wrong++ < 8) std::printf("%a / %a: %a, not %a\n", y, scale, got, exact);
        }
      }
    }
  std::printf("%lu quotients, %lu on the wrong side of a midpoint\n", tried, wrong);
  return wrong != 0;
}

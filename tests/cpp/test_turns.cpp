// csrc/turns.h on the host: cosines and sines of positions' angles against 80-bit
// ones, at every place in a turn and at the borders of its integers. Built with
// -fsanitize=undefined.
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <initializer_list>
#include <limits>

#include "turns.h"

namespace {

int failures = 0;

void check(int pos, double inv_freq, double most) {
  float c, s;
  inl::turn_of(pos, inl::turn_step(inv_freq), c, s);
  const long double a = static_cast<long double>(pos) * inv_freq;
  const double dc = std::fabs(static_cast<double>(c - cosl(a))), ds = std::fabs(static_cast<double>(s - sinl(a)));
  if (!(dc <= most && ds <= most)) {
    std::printf("pos %d inv_freq %.17g: cos off by %.3g, sin by %.3g\n", pos, inv_freq, dc, ds);
    ++failures;
  }
}

}  // namespace

int main() {
  // the reduced angle and the functions: 3 * 2^-24; inv_freq / (2 pi) is rounded to 53 bits, times the position
  const double u = std::ldexp(1.0, -24), two_pi = 6.283185307179586476925287;
  auto most = [&](int pos, double f) { return 3 * u + 4 * std::fabs(static_cast<double>(pos) * f) * std::ldexp(1.0, -53); };
  const int far[] = {0, 1, -1, 2, 31, 4096, 131071, 1000003, -1000003, 1 << 30, std::numeric_limits<int>::max(),
                     std::numeric_limits<int>::min()};
  for (int i = 0; i < 64; ++i)
    for (int pos : far) check(pos, std::pow(1e6, -i / 64.0), most(pos, std::pow(1e6, -i / 64.0)));
  // one position, all around the turn: eighths (quarters' borders) and half a turn's neighbours among them
  for (int i = -4096; i <= 4096; ++i)
    for (double d : {0.0, 1e-9, -1e-9, 2.3283064365386963e-10, -2.3283064365386963e-10}) {
      const double f = two_pi * (i / 4096.0 + d);
      check(1, f, most(1, f));
      check(-1, f, most(1, f));
    }
  // no turn at all, from either side of zero
  for (double f : {0.0, -0.0, 1e-300, -1e-300, 1e-25, -1e-25, std::numeric_limits<double>::denorm_min()})
    for (int pos : far) check(pos, f, most(pos, f));
  // not finite: no angle is meant, but nothing undefined happens
  float c, s;
  for (double f : {std::numeric_limits<double>::infinity(), -std::numeric_limits<double>::infinity(),
                   std::numeric_limits<double>::quiet_NaN(), 1e300, -1e300})
    inl::turn_of(7, inl::turn_step(f), c, s);
  if (failures == 0) std::printf("all passed\n");
  return failures != 0;
}

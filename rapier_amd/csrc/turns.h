// turns.h - cos and sin of an angle in turns, in fp64.  Nothing but arithmetic, so that the host can compile it for its test.
#pragma once

namespace rmi {

// cos and sin of 2 pi t: the quarter turn next to t is taken off, the rest (at most an eighth of a turn, |x| <= pi / 4) goes into
// Taylor's series up to x^16 / 16! and x^15 / 15!, whose first terms left out are below 3e-18 and 5e-17: with the roundings of x and
// of the last sums, within 2^-51
__host__ __device__ __forceinline__ void cos_sin_turns(double t, double* c, double* s) {
    const double k = __builtin_rint(4.0 * t), x = (t - 0.25 * k) * 6.28318530717958647692, y = x * x;
    double sn = -1.0 / 1307674368000.0, cs = 1.0 / 20922789888000.0;   // x^15, x^16
    cs = cs * y - 1.0 / 87178291200.0;
    sn = sn * y + 1.0 / 6227020800.0;
    cs = cs * y + 1.0 / 479001600.0;
    sn = sn * y - 1.0 / 39916800.0;
    cs = cs * y - 1.0 / 3628800.0;
    sn = sn * y + 1.0 / 362880.0;
    cs = cs * y + 1.0 / 40320.0;
    sn = sn * y - 1.0 / 5040.0;
    cs = cs * y - 1.0 / 720.0;
    sn = sn * y + 1.0 / 120.0;
    cs = cs * y + 1.0 / 24.0;
    sn = sn * y - 1.0 / 6.0;
    cs = cs * y - 0.5;
    sn = x + x * y * sn;
    cs = 1.0 + y * cs;
    const int q = static_cast<int>(k) & 3;
    const double a = q & 1 ? sn : cs, b = q & 1 ? cs : sn;
    *c = q == 1 || q == 2 ? -a : a;
    *s = q >= 2 ? -b : b;
}

}  // namespace rmi

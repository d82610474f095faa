// Powers of two and logarithms in 64 bits, in few instructions and constants.
#pragma once
#include "common.h"

namespace ixa {

// 2^t for t in [-1022, 1000]: the nearest integer by adding 1.5 * 2^52, whose low bits then are the exponent, and the polynomial of
// degree 9 through 2^r at Chebyshev's points of [-1/2, 1/2], its constant set to 1 (2^0 is 1): off by 3.8e-14 of the value at most (at
// the ends, worked out with 50 digits).
__device__ __forceinline__ double power_of_two(double t)
{
    constexpr double kRound = 6755399441055744.0;
    const double u = t + kRound, r = t - (u - kRound);
    double v = 1.0205905413765595e-07;
    v = fma(v, r, 1.325964524488711e-06);
    v = fma(v, r, 1.5252672924850737e-05);
    v = fma(v, r, 0.0001540343375125101);
    v = fma(v, r, 0.0013333558200794592);
    v = fma(v, r, 0.009618129193934313);
    v = fma(v, r, 0.05550410866465167);
    v = fma(v, r, 0.2402265069564034);
    v = fma(v, r, 0.6931471805599462);
    v = fma(v, r, 1.0);
    int2 bits = __builtin_bit_cast(int2, v);
    bits.y += __builtin_bit_cast(int2, u).x << 20;
    return __builtin_bit_cast(double, bits);
}

// The same for every t; no number stays none.
__device__ __forceinline__ double any_power_of_two(double t)
{
    const double v = power_of_two(fmin(fmax(t, -1021.0), 1000.0));
    return t > -1021.0 ? v : t <= -1021.0 ? 0.0 : t;
}

// The logarithm of x in (2^-120, 2^120): the instruction's in 32 bits and the series of what it leaves, as right as the power of two by
// which that is found: to within 2^-44.
__device__ __forceinline__ double log2_of(double x)
{
    const double first = (double)__builtin_amdgcn_logf((float)x), e = x * power_of_two(-first) - 1.0;
    return first + 1.44269504088896340736 * e * (1.0 - e * (0.5 - e * (1.0 / 3.0)));
}

}  // namespace ixa

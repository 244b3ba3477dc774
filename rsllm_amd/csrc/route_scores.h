// What the routing kernels share: 64-bit score arithmetic and the order of places.
#pragma once

#include "kernels.h"

namespace rsllm_hip {

// exp(x) to some 2^-52: x = n log 2 + r, |r| < 0.35, and the power series of exp(r)
// up to r^12 / 12!, after Cody and Waite's reduction. (Short, where the library's
// is long: most calls of these kernels pay for fetching their code.)
__device__ __forceinline__ double route_exp64(double x) {
    x = fmin(fmax(x, -1000.0), 1000.0);
    const double n = rint(x * 0x1.71547652b82fep+0);  // log2 e
    // log 2 in two parts, the first of few enough bits that n times it is exact
    const double r = fma(n, -0x1.7f7d1cf79abcap-20, fma(n, -0x1.62e4p-1, x));
    double p = 1.0 / 479001600.0;
    p = fma(p, r, 1.0 / 39916800.0);
    p = fma(p, r, 1.0 / 3628800.0);
    p = fma(p, r, 1.0 / 362880.0);
    p = fma(p, r, 1.0 / 40320.0);
    p = fma(p, r, 1.0 / 5040.0);
    p = fma(p, r, 1.0 / 720.0);
    p = fma(p, r, 1.0 / 120.0);
    p = fma(p, r, 1.0 / 24.0);
    p = fma(p, r, 1.0 / 6.0);
    p = fma(p, r, 0.5);
    p = fma(p, r, 1.0);
    p = fma(p, r, 1.0);
    return ldexp(p, (int)n);
}
// log(1 + e), 0 <= e <= 1: 2 atanh(z), z = e / (2 + e) <= 1/3, to z^33.
__device__ __forceinline__ double route_log1p(double e) {
    const double z = e / (2.0 + e), q = z * z;
    double p = 2.0 / 33.0;
    p = fma(p, q, 2.0 / 31.0);
    p = fma(p, q, 2.0 / 29.0);
    p = fma(p, q, 2.0 / 27.0);
    p = fma(p, q, 2.0 / 25.0);
    p = fma(p, q, 2.0 / 23.0);
    p = fma(p, q, 2.0 / 21.0);
    p = fma(p, q, 2.0 / 19.0);
    p = fma(p, q, 2.0 / 17.0);
    p = fma(p, q, 2.0 / 15.0);
    p = fma(p, q, 2.0 / 13.0);
    p = fma(p, q, 2.0 / 11.0);
    p = fma(p, q, 2.0 / 9.0);
    p = fma(p, q, 2.0 / 7.0);
    p = fma(p, q, 2.0 / 5.0);
    p = fma(p, q, 2.0 / 3.0);
    p = fma(p, q, 2.0);
    return p * z;
}

constexpr double kNever = -__builtin_inf();  // an expert that is not to be chosen

// (a, ia) comes before (b, ib): the larger, then the lower index.
__device__ __forceinline__ bool route_before(double a, int ia, double b, int ib) {
    return a > b || (a == b && ia < ib);
}

__device__ __forceinline__ void route_best(double &v, int &i, double v2, int i2) {
    if (route_before(v2, i2, v, i)) {
        v = v2;
        i = i2;
    }
}

}  // namespace rsllm_hip

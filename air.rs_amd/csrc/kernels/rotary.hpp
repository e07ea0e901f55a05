// Rotary positions: the angles, and the elements of a row that turn with them.
//
// A row's first rot elements are rot / 2 pairs (x, y); pair i of a row at position p turns
// by the angle p * inv_freq[i]:
//   (x, y) -> (x c - y s, x s + y c),   c = magnitude * cos(angle), s = magnitude * sin(angle)
// Pair i is (row[i], row[i + rot / 2]) in the half layout, (row[2i], row[2i + 1]) where pairs
// lie side by side.  Elements past rot stay.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace airkv {

// c and s, rounded to 32 bits once.  The angle is held in 64 bits: a position times an f32
// frequency is exact up to 2^29, and at position 10^6 f32 angles would be off by 0.06.  The
// multiple k of pi / 2 nearest to it is taken off in two steps: k times the f64 nearest to
// pi / 2 has no bits below 2^-52 and lies within 1 of the angle, so the first difference is
// exact, and the second takes what pi / 2 has beyond.  On [-pi / 4, pi / 4] the Taylor sums
// to r^17 and r^16 are within 2^-57 and 2^-58 of sine and cosine.
//
// rotary_scalar: a coefficient in scalar registers, which leaves the vector ones to rows on their way
// (as literals they took 34, held from loop to loop).
__device__ __forceinline__ double rotary_scalar(double x) {
    asm("" : "+s"(x));
    return x;
}
__device__ __forceinline__ float2 rotary_turn(int64_t position, float inv_freq, float magnitude) {
    constexpr double kSin[8] = {-1.0 / 6.0, 1.0 / 120.0, -1.0 / 5040.0, 1.0 / 362880.0, -1.0 / 39916800.0,
                                1.0 / 6227020800.0, -1.0 / 1307674368000.0, 1.0 / 355687428096000.0};
    constexpr double kCos[8] = {-0.5, 1.0 / 24.0, -1.0 / 720.0, 1.0 / 40320.0, -1.0 / 3628800.0,
                                1.0 / 479001600.0, -1.0 / 87178291200.0, 1.0 / 20922789888000.0};
    const double angle = (double)position * (double)inv_freq;
    const double k = __builtin_rint(angle * 0x1.45f306dc9c883p-1);
    double r = __builtin_fma(-k, 0x1.921fb54442d18p+0, angle);
    r = __builtin_fma(-k, 0x1.1a62633145c07p-54, r);
    const double z = r * r;
    double s = kSin[7], c = kCos[7];
#pragma unroll
    for (int i = 6; i >= 0; --i) {
        s = __builtin_fma(s, z, rotary_scalar(kSin[i]));
        c = __builtin_fma(c, z, rotary_scalar(kCos[i]));
    }
    s = __builtin_fma(s * z, r, r);
    c = __builtin_fma(c, z, 1.0);
    // k mod 4 (past 2^55 or so every k is a multiple of 4)
    const int quarter = (int)(k - 4.0 * __builtin_floor(k * 0.25));
    const double cq = quarter & 1 ? -s : c, sq = quarter & 1 ? c : s;
    const double m = quarter & 2 ? -(double)magnitude : (double)magnitude;
    return make_float2((float)(cq * m), (float)(sq * m));
}

// Where the partner of elements e .. e + 3 (e a multiple of 4, below rot) begins in the half
// layout, and their pairs' indices: rot is a multiple of 8, so that four neighbours are all
// first or all second elements.
__device__ __forceinline__ int rotary_partner(int e, int half) { return e < half ? e + half : e - half; }

// One pair.  Products and sums round one by one: what a 1-byte page's codes are made from is defined
// bit for bit.
__device__ __forceinline__ void rotary_pair(float &x, float &y, float2 cs) {
#pragma clang fp contract(off)
    const float xc = x * cs.x, ys = y * cs.y, xs = x * cs.y, yc = y * cs.x;
    x = xc - ys;
    y = xs + yc;
}
// Four elements x of a row from element e on, turned; y their partners (half layout), cs the
// pairs' (c, s).
__device__ __forceinline__ void rotary_half4(float (&x)[4], const float (&y)[4], const float2 *cs, int e, int half) {
#pragma clang fp contract(off)
    const bool second = e >= half;
    const float2 *p = cs + (second ? e - half : e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float a = x[j] * p[j].x, b = y[j] * p[j].y;
        x[j] = second ? b + a : a - b;
    }
}
__device__ __forceinline__ void rotary_pairs4(float (&x)[4], const float2 *cs, int e) {
#pragma unroll
    for (int j = 0; j < 4; j += 2) rotary_pair(x[j], x[j + 1], cs[(e + j) / 2]);
}

}  // namespace airkv

// Score modifications of the certified attention: what happens to a logit between t = RN32(alpha s) and
// the weight RN24(2^t), and which keys a row sees.
//
//   cap    t1 = RN32(c tanh(t / c)), in a fixed sequence of IEEE fp64 operations within 2^-39 of the
//          tanh, relative: RN32 of the exact value except within 2^-14 of a step of a midpoint
//   bias   t2 = RN32(t1 - m |n - p|), one fused multiply-add: m the query head's slope, n the key, p
//          the query's position, |n - p| converted to fp32
//   keys   begin <= n < kv_len, begin the larger of the token's kv_begin and kv_len - window, and the
//          tree keys as before
//
// Each step is a function of the fp32 number before it. So every tier that knows t exactly (all of
// them decide that before they weigh a key) gets the same t2, on the device and on the host alike, and
// the output's bits still depend on nothing but the definition. A t2 that is not finite is a domain
// error, as an overflow of t is.
//
// With a bias the weights of one row span any range of exponents (a slope of 1/2 over 10,000 keys: 2^-7000).
// Weights below 2^-800 of the row's largest are then dropped by the fp64 tiers instead of leaving the row to the
// 128-bit path: fewer than 2^31 of them add less than 2^-700 of Z, and of N times max |v|, which one
// more unit of u' in the error bounds covers (its 2^-53).
#pragma once
#include <math.h>
#include <stdint.h>
#include <string.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define EA_HD __host__ __device__ __forceinline__
#else
#define EA_HD inline
#endif

namespace ea {

// The cap's constants: c (0: none), 1 / c and 2 log2(e) / c, each rounded to fp64 on the host
struct ModCap {
    double c, ic, k2;
};
inline ModCap mod_cap_of(float c) {
    if (!(c > 0.0f)) return ModCap{0.0, 0.0, 0.0};
    return ModCap{(double)c, 1.0 / (double)c, 0x1.71547652b82fep+1 / (double)c};
}

EA_HD uint32_t mod_bits(float x) {
    uint32_t u;
    memcpy(&u, &x, 4);
    return u;
}
EA_HD float mod_float(uint32_t u) {
    float x;
    memcpy(&x, &u, 4);
    return x;
}

// RN32(c tanh(t / c)). tanh(x) = (1 - e) / (1 + e) with e = 2^-y, y = |t| 2 log2(e) / c (64 and above:
// e is below the rounding of 1 + e); e from the 2^(j/256) table (times 2^tsh) and a quartic in the rest,
// r < 2^-8 (truncation below 2^-49). 1 - e cancels for small x, whose error 2^-50 / (2 x) stays below
// 2^-39 down to x = 2^-11; below it x - x^3 / 3 (next term 2^-45 of x).
EA_HD float mod_cap(float t, const ModCap& C, const double* T1, int tsh) {
    const double a = fabs((double)t);
    const double y = fmin(a * C.k2, 64.0);
    const double N = ceil(y);
    const double f = (N - y) * 256.0;
    const double fj = floor(f);
    const double r = (f - fj) * 0x1p-8;
    double p = fma(r, 0x1.3b2ab6fba4e77p-7, 0x1.c6b08d704a0c0p-5);
    p = fma(r, p, 0x1.ebfbdff82c58fp-3);
    p = fma(r, p, 0x1.62e42fefa39efp-1);
    p = fma(r, p, 1.0);
    const double e = ldexp(T1[(int)fj & 255] * p, -(int)N - tsh);
    const double th = (1.0 - e) / (1.0 + e);
    const double x = a * C.ic;
    const double ts = x * fma(x * x, -0x1.5555555555555p-2, 1.0);
    return copysignf((float)(C.c * (x < 0x1p-11 ? ts : th)), t);
}

// RN32(t - m |dist|)
EA_HD float mod_bias(float t, float m, int32_t dist) {
    const uint32_t ad = dist < 0 ? 0u - (uint32_t)dist : (uint32_t)dist;
    return fmaf(-m, (float)ad, t);
}

// The modified logit of a pair whose unmodified one was decided exactly: st 0, *tb its fp32 bits; or st
// 1, |alpha s| <= 2^-25 without its value (0 when zero). Returns 0 and the bits in *tb, 2 for a domain
// error, 3 when t's value would be needed; other states pass through. A |t| up to 2^-25 gives the
// weight 1 whatever it is, so two ends that both do are taken as 0.
EA_HD int mod_logit(int st, bool zero, const ModCap& C, float m, int32_t dist, const double* T1, int tsh, uint32_t* tb) {
    if (st > 1) return st;
    if (st == 1 && !zero) {
        const float lo = mod_bias(-0x1p-25f, m, dist), hi = mod_bias(0x1p-25f, m, dist);
        if (!(fabsf(lo) < INFINITY) || !(fabsf(hi) < INFINITY)) return 2;
        if (lo == hi) *tb = mod_bits(lo);
        else if (fabsf(lo) <= 0x1p-25f && fabsf(hi) <= 0x1p-25f) *tb = 0;
        else return 3;
        return 0;
    }
    float t = st == 1 ? 0.0f : mod_float(*tb);
    if (C.c > 0.0) t = mod_cap(t, C, T1, tsh);
    t = mod_bias(t, m, dist);
    if (!(fabsf(t) < INFINITY)) return 2;
    *tb = mod_bits(t);
    return 0;
}

}  // namespace ea

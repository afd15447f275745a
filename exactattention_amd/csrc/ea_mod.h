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
// What it costs (d = 128, plain, ranges, bias, cap, both; us a step): 32 sequences of 4096 keys, one token, 32/8
// heads, on ea_mrow 121, 120, 122, 122, 123 (they wait for memory); 8 x 8 tokens, 8000 keys, 16/8 heads 140, 141, 149,
// 156, 160; 2500 causal tokens, 16/8 heads, on ea_pf_main 386, 403, 633, 475, 648 (a bias raises the bases in 9
// of 10 tile steps).
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
#define EA_MOD_HD __host__ __device__ __forceinline__
#else
#define EA_MOD_HD inline
#endif

namespace ea {

// The cap's constants: c (0: none) and 512 log2(e) / c, rounded to fp64 on the host
struct ModCap {
    double c, k256;
};
inline ModCap mod_cap_of(float c) {
    if (!(c > 0.0f)) return ModCap{0.0, 0.0};
    return ModCap{(double)c, 0x1.71547652b82fep+9 / (double)c};
}

EA_MOD_HD uint32_t mod_bits(float x) {
    uint32_t u;
    memcpy(&u, &x, 4);
    return u;
}
EA_MOD_HD float mod_float(uint32_t u) {
    float x;
    memcpy(&x, &u, 4);
    return x;
}

// n / d for d in [1, 2] and |n| <= 1, correctly rounded: on the device the steps of the IEEE division
// without its scaling, which numbers of this size do not need (11 instructions -> 8).
EA_MOD_HD double mod_div(double n, double d) {
#ifdef __HIP_DEVICE_COMPILE__
    double y = __builtin_amdgcn_rcp(d);
    y = fma(fma(-d, y, 1.0), y, y);
    y = fma(fma(-d, y, 1.0), y, y);
    const double q = n * y;
    return fma(fma(-d, q, n), y, q);
#else
    return n / d;
#endif
}

// RN32(c tanh(t / c)). tanh(x) = -g / (2 + g) with g = 2^-y - 1, y = |t| 2 log2(e) / c (64 and above: 2^-y
// is below the rounding of g). y = (i + r) / 256 with i whole: g = S P + (S - 1), S = 2^(-i/256) from the
// 2^(j/256) table (times 2^tsh), P = 2^(-r/256) - 1 a quartic in r (truncation 2^-41 of it). For i = 0
// S - 1 is 0 and g = P keeps its relative accuracy down to t = 0; for i > 0 S - 1 is exact and above 2^-9.
EA_MOD_HD float mod_cap(float t, const ModCap& C, const double* T1, int tsh) {
    const double y = fmin(fabs((double)t) * C.k256, 16384.0);
    const double fi = floor(y), r = y - fi;
    const int j = -(int)fi;
    double P = fma(r, 0x1.3b2ab6fba4e77p-39, -0x1.c6b08d704a0c0p-29);
    P = fma(r, P, 0x1.ebfbdff82c58fp-19);
    P = r * fma(r, P, -0x1.62e42fefa39efp-9);
    const double S = ldexp(T1[j & 255], (j >> 8) - tsh);
    const double g = fma(S, P, S - 1.0);
    return copysignf((float)(C.c * mod_div(-g, 2.0 + g)), t);
}

// RN32(t - m |dist|)
EA_MOD_HD float mod_bias(float t, float m, int32_t dist) {
    const uint32_t ad = dist < 0 ? 0u - (uint32_t)dist : (uint32_t)dist;
    return fmaf(-m, (float)ad, t);
}

// The modified logit of a pair whose unmodified one was decided exactly: st 0, *tb its fp32 bits; or st
// 1, |alpha s| <= 2^-25 without its value (0 when zero). Returns 0 and the bits in *tb, 2 for a domain
// error, 3 when t's value would be needed; other states pass through. A |t| up to 2^-25 gives the
// weight 1 whatever it is, so two ends that both do are taken as 0.
EA_MOD_HD int mod_logit(int st, bool zero, const ModCap& C, float m, int32_t dist, const double* T1, int tsh, uint32_t* tb) {
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

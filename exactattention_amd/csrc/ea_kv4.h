// Caches held in 4 bits: the microscaling format of 4-bit floats, 32 elements to a scale.
//
//   element  4 bits, sign, 2 of exponent and 1 of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives;
//            element 2 i of a row in the low half of byte i
//   scale    a byte b for 32 elements: 2^(b - 127), 255 NaN
//
// A value has 2 significant bits, so every one of them is a bf16 (b = 0: a subnormal one; beyond the largest bf16 an
// infinity, as its rounding is): attention over such a cache is attention over the bf16 cache of its values, to the bit,
// and the exact tiers only need these loaders. gfx950 converts two elements and their scale in one instruction, whose
// results were compared with the table above for every element and scale, subnormals, infinities and NaN among them.
//
// Geometry: strides count elements, as those of bf16 caches; an element's codes lie at half its offset and its scale at a
// 32nd, so strides are multiples of 32 and a row of d elements takes (d + 31) / 32 groups.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ea {

typedef float kv4_f2 __attribute__((ext_vector_type(2)));

// elements 2 SEL and 2 SEL + 1 of a dword of eight, times their scale
template <int SEL>
__device__ __forceinline__ kv4_f2 kv4_pair(uint32_t w, uint32_t scale) {
    return __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, __uint_as_float(scale << 23), SEL);
}
// the same as two bf16 (exact)
template <int SEL>
__device__ __forceinline__ uint32_t kv4_bf16x2(uint32_t w, uint32_t scale) {
    const kv4_f2 p = kv4_pair<SEL>(w, scale);
    return __builtin_amdgcn_perm(__float_as_uint(p.y), __float_as_uint(p.x), 0x07060302u);
}
// An upper bound of a group's magnitudes: 6 times its scale, or infinity where that has no fp32 value
__device__ __forceinline__ float kv4_bound(uint32_t scale) {
    return 6.0f * __uint_as_float(max(scale, 1u) << 23);
}

// 8 elements from element offset `off` (a multiple of 8) as bf16
__device__ __forceinline__ uint4 kv4_load8(const void* codes, const uint8_t* scales, int64_t off) {
    const uint32_t w = *(const uint32_t*)((const uint8_t*)codes + (off >> 1)), s = scales[off >> 5];
    return make_uint4(kv4_bf16x2<0>(w, s), kv4_bf16x2<1>(w, s), kv4_bf16x2<2>(w, s), kv4_bf16x2<3>(w, s));
}
// 2 elements from `off` (even), the first in the low half
__device__ __forceinline__ uint32_t kv4_load2(const void* codes, const uint8_t* scales, int64_t off) {
    return kv4_bf16x2<0>(((const uint8_t*)codes)[off >> 1], scales[off >> 5]);
}

// a whole group from `off` (a multiple of 32), zeros past the first `have` (a multiple of 8, or negative)
__device__ __forceinline__ void kv4_load32(const void* codes, const uint8_t* scales, int64_t off, int have, uint32_t (&raw)[16]) {
    const uint4 c = *(const uint4*)((const uint8_t*)codes + (off >> 1));
    const uint32_t s = scales[off >> 5], w[4] = {c.x, c.y, c.z, c.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = 8 * i < have;
        raw[4 * i] = in ? kv4_bf16x2<0>(w[i], s) : 0u;
        raw[4 * i + 1] = in ? kv4_bf16x2<1>(w[i], s) : 0u;
        raw[4 * i + 2] = in ? kv4_bf16x2<2>(w[i], s) : 0u;
        raw[4 * i + 3] = in ? kv4_bf16x2<3>(w[i], s) : 0u;
    }
}

}  // namespace ea

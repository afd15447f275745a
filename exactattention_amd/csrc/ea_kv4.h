// Caches held in 4 bits: the microscaling format of 4-bit floats, 32 elements to a scale.
//
//   element  4 bits, sign, 2 of exponent and 1 of mantissa: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives
//   scale    a byte b for 32 elements: 2^(b - 127), 255 NaN
//
// A value has 2 significant bits, so every one of them is a bf16 (b = 0: a subnormal one; beyond the largest bf16 an
// infinity, as its rounding is): attention over such a cache is attention over the bf16 cache of its values, to the bit,
// and the exact tiers only need these loaders. gfx950 converts two elements and their scale in one instruction, whose
// results were compared with the table above for every element and scale, subnormals, infinities and NaN among them.
//
// K: strides count elements, as those of bf16 caches; element 2 i of a row is the low half of byte i, an element's code lies at
// half its offset and its scale at a 32nd, so strides are multiples of 32 and a row of d elements takes (d + 31) / 32 groups.
// V: 16 slots are a tile, w / 2 pairs of channels by 16 slots, a byte for a pair (the even channel in its low half) and slot; their
// scales w / 32 groups by 16 slots (w: the channels in whole groups). So a lane of a matrix instruction, which wants 16 keys of a
// channel, has those of two in one 16-byte load. The code of channels c, c + 1 of a slot lies at kv4_v(..) + 16 (c / 2), their scale
// at kv4_vscale(that) + 16 (c / 32).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ea_params.h"

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

// 8 elements of K from element offset `off` (a multiple of 8) as bf16
__device__ __forceinline__ uint4 kv4_load8(const void* codes, const uint8_t* scales, int64_t off) {
    const uint32_t w = *(const uint32_t*)((const uint8_t*)codes + (off >> 1)), s = scales[off >> 5];
    return make_uint4(kv4_bf16x2<0>(w, s), kv4_bf16x2<1>(w, s), kv4_bf16x2<2>(w, s), kv4_bf16x2<3>(w, s));
}
// 2 elements of K from `off` (even), the first in the low half
__device__ __forceinline__ uint32_t kv4_load2(const void* codes, const uint8_t* scales, int64_t off) {
    return kv4_bf16x2<0>(((const uint8_t*)codes)[off >> 1], scales[off >> 5]);
}

// channels of V in whole groups
__host__ __device__ __forceinline__ int kv4_width(int dv) { return (dv + 31) & ~31; }
// the byte of channels 0 and 1 of slot `slot` of a page's head at element offset `at` (all its tiles are 16 slots of w channels)
__device__ __forceinline__ int64_t kv4_v_at(int64_t at, int64_t slot, int w) {
    return (at >> 1) + (slot >> 4) * (8 * w) + (slot & 15);
}
__device__ __forceinline__ int64_t kv4_vscale(int64_t code) { return (code >> 4) + (code & 15); }
// the same for key n of sequence b and head hk
__device__ __forceinline__ int64_t kv4_v(const Params& P, int64_t b, int64_t n, int hk) {
    int64_t page = b, slot = n;
    if (P.bt) {
        page = P.bt[(P.bt_off ? P.bt_off[b] : b * (int64_t)P.g.block_table_stride) + (n >> P.pshift)];
        slot = n & ((1 << P.pshift) - 1);
    }
    return kv4_v_at(page * P.g.v_page_stride + (int64_t)hk * P.g.v_head_stride, slot, kv4_width(P.g.head_dim_v));
}
// channels c (even) and c + 1 as bf16; `code` from kv4_v
__device__ __forceinline__ uint32_t kv4_vload2(const void* codes, const uint8_t* scales, int64_t code, int c) {
    return kv4_bf16x2<0>(((const uint8_t*)codes)[code + 16 * (c >> 1)], scales[kv4_vscale(code) + 16 * (c >> 5)]);
}

}  // namespace ea

// Rows of bf16 or fp32 elements as the rotation's kernels read and write them: V consecutive elements at a time,
// held as doubles in between and rounded once.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ea {

// RN of a double to bf16 bits, one rounding: the fp32 value decides except where it is itself the
// midpoint of two bf16 values and inexact; there the double's side of it does
__device__ __forceinline__ uint32_t f64_bf16(double x) {
    const float f = (float)x;
    uint32_t b = __float_as_uint(f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return (b >> 16) | 0x40u;
    if ((b & 0xFFFFu) == 0x8000u) {
        const double a = fabs(x), d = (double)fabsf(f);
        b += (a > d ? 1u : 0u) - (a < d ? 1u : 0u);
    }
    return (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
}
// The same of N values, two to a word. Rounded to fp32 first, which only a value next to a tie of bf16 can tell: where one looks like a tie
// (2^-16 of them do) all are rounded singly. 3 instructions a value; f64_bf16 takes two branches.
template <int N>
__device__ __forceinline__ void f64_bf16_all(const double (&x)[N], uint32_t* out) {
    typedef float two_f __attribute__((ext_vector_type(2)));
    typedef __bf16 two_b __attribute__((ext_vector_type(2)));
    typedef unsigned short two_h __attribute__((ext_vector_type(2)));
    two_h tie = {0xFFFF, 0xFFFF};
#pragma unroll
    for (int i = 0; i < N; i += 2) {
        const two_f f = {(float)x[i], (float)x[i + 1]};
        out[i / 2] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, two_b));
        const uint32_t low = __builtin_amdgcn_perm(__float_as_uint(f.y), __float_as_uint(f.x), 0x05040100u) ^ 0x80008000u;
        tie = __builtin_elementwise_min(tie, __builtin_bit_cast(two_h, low));
    }
    if (__builtin_expect(tie.x == 0 || tie.y == 0, 0)) {
#pragma unroll
        for (int i = 0; i < N; i += 2) out[i / 2] = f64_bf16(x[i]) | f64_bf16(x[i + 1]) << 16;
    }
}
__device__ __forceinline__ uint32_t f32_bf16(float f) {
    const uint32_t b = __float_as_uint(f);
    if ((b & 0x7FFFFFFFu) > 0x7F800000u) return (b >> 16) | 0x40u;
    return (b + 0x7FFFu + ((b >> 16) & 1u)) >> 16;
}

// V consecutive elements of type bf16 (FP32 = 0) or fp32, as doubles
template <int V, bool FP32>
struct Chunk {
    uint32_t r[FP32 ? V : (V + 1) / 2];
    __device__ __forceinline__ void load(const void* p, int64_t at) {
        if constexpr (V == 8) {
            const uint4* s = (const uint4*)((const char*)p + at * (FP32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < (FP32 ? 2 : 1); ++i) {
                const uint4 x = s[i];
                r[4 * i] = x.x;
                r[4 * i + 1] = x.y;
                r[4 * i + 2] = x.z;
                r[4 * i + 3] = x.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if constexpr (FP32) r[i] = ((const uint32_t*)p)[at + i];
                else if (i & 1) r[i >> 1] |= (uint32_t)((const uint16_t*)p)[at + i] << 16;
                else r[i >> 1] = ((const uint16_t*)p)[at + i];
            }
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (FP32) return __uint_as_float(r[i]);
        else return __uint_as_float(i & 1 ? r[i >> 1] & 0xFFFF0000u : r[i >> 1] << 16);
    }
    __device__ __forceinline__ void put(int i, double x) {
        if constexpr (FP32) r[i] = __float_as_uint((float)x);
        else if (i & 1) r[i >> 1] |= f64_bf16(x) << 16;
        else r[i >> 1] = f64_bf16(x);
    }
    __device__ __forceinline__ void put_all(const double (&x)[V]) {
        if constexpr (FP32 || V < 2) {
#pragma unroll
            for (int i = 0; i < V; ++i) put(i, x[i]);
        } else {
            f64_bf16_all<V>(x, r);
        }
    }
    __device__ __forceinline__ void store(void* p, int64_t at) const {
        if constexpr (V == 8) {
            uint4* s = (uint4*)((char*)p + at * (FP32 ? 4 : 2));
#pragma unroll
            for (int i = 0; i < (FP32 ? 2 : 1); ++i) s[i] = make_uint4(r[4 * i], r[4 * i + 1], r[4 * i + 2], r[4 * i + 3]);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                if constexpr (FP32) ((uint32_t*)p)[at + i] = r[i];
                else ((uint16_t*)p)[at + i] = (uint16_t)(i & 1 ? r[i >> 1] >> 16 : r[i >> 1]);
            }
        }
    }
};

// V elements to dst, of another type or the same
template <int V, bool IN32, bool OUT32>
__device__ __forceinline__ void store_as(const Chunk<V, IN32>& a, void* dst, int64_t at) {
    if constexpr (IN32 == OUT32) {
        a.store(dst, at);
    } else {
        Chunk<V, OUT32> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const uint32_t h = f32_bf16(a.get(i));  // fp32 to bf16 only
            if (i & 1) o.r[i >> 1] |= h << 16;
            else o.r[i >> 1] = h;
        }
        o.store(dst, at);
    }
}

}  // namespace ea

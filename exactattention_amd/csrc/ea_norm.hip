// Per-head norms of q and k with their rotary positions in one pass (gfx950), into bf16 or fp32 rows or a cache held in 4
// bits, and the gradient of both. No reference counterpart: the reference takes q and k as its demo's model
// leaves them (scripts/spec_decode_demo.py:57-73).
//
//   forward   y = R(pos) (x r w), r = 1 / sqrt(mean x^2 + eps)
//   gradient  g = R(pos)^T gy, xh = x r:  dx = r (g w - xh mean(g w xh)),  dw = sum over tokens and heads of g xh
//   4 bits    a scale for 32 elements: the smallest 2^e with max|y| < 7 2^e, elements to the nearest of 0, 0.5, 1,
//             1.5, 2, 3, 4, 6 times it
//
// All of it runs in fp64 and is rounded once, as the rotation by itself does. 16384 tokens of 32/8 heads of 128 bf16 into a 4-bit cache
// 116 us (353 MB, 68 us at the copy rate); 4096 tokens of 16/8 heads forward 20 (50 MB, 10), gradient 31 (75 MB, 15), which 232
// registers keep at 2 waves a SIMD. No one unit bounds it. In those three the VALU issues 64, 61 and 50% of the CUs' busy cycles (16 to
// 30 instructions an element) and conflicts on LDS banks take 38, 39 and 27%: the lanes of a head read turns 128 and weights 64 bytes
// apart. Waves wait for 61, 53 and 41% of their time.
// Layout: L lanes hold a head, 2 C elements each: the two halves of C rotated pairs, or two runs of C others. So a head's sums
// are log2 L shuffles, the rotation needs no other lane's elements, and with C = 8 every access has 16 bytes. C = 2 and 1
// take what is not aligned so, or whose halves are not whole runs.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/exactattn_hip.h"
#include "ea_chunk.h"
#include "ea_kv4.h"
#include "ea_params.h"

using namespace ea;

namespace {

int herr(hipError_t e) { return e == hipSuccess ? 0 : -100 - (int)e; }

constexpr int NR_THREADS = 256;
constexpr int NG_BLOCKS = 512;  // of the gradient: its partial sums of the weights' gradients are a row each

// What lane u of a head's L holds: C elements from e[0] and C from e[1] (-1: none); turn[0]: they are the two halves of C pairs
// (halves apart) or the first run holds adjacent pairs, turn[1]: the second run does
struct Held {
    int e[2];
    bool turn[2];
};
template <int C, bool ADJ>
__device__ __forceinline__ Held held_by(int u, int d, int R, bool isv) {
    Held x;
    const int h = R / 2;
    const int pu = isv || ADJ ? 0 : h / C;  // lanes with halves
    if (u < pu) {
        x.e[0] = u * C;
        x.e[1] = h + u * C;
        x.turn[0] = x.turn[1] = true;
        return x;
    }
    const int at = isv || ADJ ? 0 : R, n = (d - at) / C, n2 = (n + 1) / 2, j = u - pu;
    x.e[0] = j < n2 ? at + j * C : -1;
    x.e[1] = j < n2 && j + n2 < n ? at + (j + n2) * C : -1;
    x.turn[0] = ADJ && !isv && x.e[0] < R && x.e[0] >= 0;
    x.turn[1] = ADJ && !isv && x.e[1] < R && x.e[1] >= 0;
    return x;
}

// the rotation of a lane's elements by cs[pair] = (cos, sin), times scale already; BACK: transposed
template <int C, bool ADJ, bool BACK>
__device__ __forceinline__ void turn_held(const Held& H, const double2* z, double (&a)[C], double (&b)[C]) {
    if constexpr (ADJ) {
        if constexpr (C > 1) {
            auto one = [&](double (&x)[C], int e) __attribute__((always_inline)) {
#pragma unroll
                for (int i = 0; i < C; i += 2) {
                    const double2 q = z[(e + i) >> 1];
                    const double s = BACK ? -q.y : q.y, u = x[i], v = x[i + 1];
                    x[i] = __fma_rn(u, q.x, -(v * s));
                    x[i + 1] = __fma_rn(v, q.x, u * s);
                }
            };
            if (H.turn[0]) one(a, H.e[0]);
            if (H.turn[1]) one(b, H.e[1]);
        }
    } else if (H.turn[0]) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const double2 q = z[H.e[0] + i];
            const double s = BACK ? -q.y : q.y, u = a[i], v = b[i];
            a[i] = __fma_rn(u, q.x, -(v * s));
            b[i] = __fma_rn(v, q.x, u * s);
        }
    }
}

// (cos, sin) * scale of the block's tokens, pair by pair: the angle in half turns, its product's rounding error brought back
__device__ __forceinline__ void fill_turns(const ea_rotary& A, double2* cs, int64_t t0, int nt) {
    const int h = A.rot_dim / 2;
    for (int i = threadIdx.x; i < nt * h; i += NR_THREADS) {
        const int tk = i / h, p = i - tk * h;
        const int axis = A.axis_of_pair ? A.axis_of_pair[p] : 0;
        const double pos = (double)((int64_t)A.positions[axis * A.pos_axis_stride + t0 + tk] + A.pos_offset);
        const double w = A.half_turns[p];
        const double y = pos * w, e = __fma_rn(pos, w, -y);
        double sn, cn;
        sincospi((y - 2.0 * rint(0.5 * y)) + e, &sn, &cn);
        cs[i] = make_double2(cn * (double)A.scale, (A.inverse ? -sn : sn) * (double)A.scale);
    }
}

__device__ __forceinline__ double weight_at(const void* w, int fp32, int i) {
    return fp32 ? (double)((const float*)w)[i] : (double)__uint_as_float((uint32_t)((const uint16_t*)w)[i] << 16);
}

// over a head's L lanes (a power of two, aligned), in every one of them
__device__ __forceinline__ double head_sum(double x, int L) {
    for (int o = 1; o < L; o <<= 1) x += __shfl_xor(x, o, 64);
    return x;
}

// A double as the fp32 value that the conversion to 4 bits rounds as it would round the double: its upper 21 significant bits
// with the others' presence in the last one (round to odd). Past fp32's range an infinity.
__device__ __forceinline__ float odd21(double y) {
    const int hi = __double2hiint(y), lo = __double2loint(y);
    return (float)__hiloint2double(hi | (lo != 0 ? 1 : 0), 0);
}

// a head of one of q, k and v: where it comes from and goes
struct Row {
    const void* src;
    void* dst;
    uint8_t* scales;
    int64_t s, o;
    int kind;  // 0 q, 1 k, 2 v
    int tk;
    bool live;
};

// FULL: every lane holds two whole runs, and 32 elements lie with 4 lanes from a multiple of 4 (full_lanes)
template <int C, bool IN32, bool OUT32, bool KV4, bool ADJ, bool FULL>
__global__ void __launch_bounds__(NR_THREADS) ea_norm_rotary_kernel(ea_norm_rotary N, int tpb, int L) {
    extern __shared__ __align__(16) double2 cs[];  // tpb x pairs, then the weights of q and k (d each)
    __shared__ uint32_t s_max[FULL ? 1 : NR_THREADS];  // of a head's groups, at its lanes' places
    const ea_rotary& A = N.r;
    const int d = A.head_dim, R = A.rot_dim, h = R / 2, tid = threadIdx.x;
    const int64_t t0 = (int64_t)blockIdx.x * tpb;
    const int nt = (int)min((int64_t)tpb, A.num_tokens - t0);
    const bool norm = N.q_weight != nullptr;
    double* const wt = (double*)(cs + tpb * h);
    const int Hq = A.num_q_heads, Hk = A.num_kv_heads, I = Hq + Hk + (A.v ? Hk : 0);
    const int u = tid & (L - 1), base = tid & ~(L - 1);
    const int shift = KV4 && !(N.page_size & (N.page_size - 1)) ? __builtin_ctz(N.page_size) : -1;  // -1: a division
    auto row_of = [&](int it) __attribute__((always_inline)) {
        Row x;
        int g = it;
        for (x.tk = 0; g >= I; ++x.tk) g -= I;  // a few tokens
        const int64_t t = t0 + x.tk;
        x.scales = nullptr;
        if (g < Hq) {
            x.kind = 0;
            const int64_t r = A.q_rows ? A.q_rows[t] : t;
            x.live = r >= 0 && r < A.q_out_rows;
            x.src = A.q;
            x.dst = A.q_out;
            x.s = t * A.q_tok_stride + g * A.q_head_stride;
            x.o = r * A.qo_tok_stride + g * A.qo_head_stride;
            return x;
        }
        const int64_t r = A.dst_rows ? A.dst_rows[t] : t;
        x.live = r >= 0 && r < A.pool_rows;
        x.kind = g < Hq + Hk ? 1 : 2;
        g -= x.kind == 1 ? Hq : Hq + Hk;
        const bool v = x.kind == 2;
        x.src = v ? A.v : A.k;
        x.dst = v ? A.v_out : A.k_out;
        x.s = v ? t * A.v_tok_stride + g * A.v_head_stride : t * A.k_tok_stride + g * A.k_head_stride;
        const int64_t ts = v ? A.vo_tok_stride : A.ko_tok_stride, hs = v ? A.vo_head_stride : A.ko_head_stride;
        if constexpr (KV4) {
            x.scales = v ? N.v_scales : N.k_scales;
            const int64_t page = shift >= 0 ? r >> shift : r / N.page_size, slot = r - page * N.page_size;
            if (v) x.o = kv4_v_at(page * N.v_page_stride + g * hs, slot, kv4_width(d));
            else x.o = page * N.k_page_stride + slot * ts + g * hs;
        } else {
            x.o = r * ts + g * hs;
        }
        return x;
    };
    const int total = nt * I, step = (int)gridDim.y * (NR_THREADS / L);
    struct Work {
        Row row;
        Held H;
        Chunk<C, IN32> a, b;
    };
    auto fetch = [&](int it, Work& x) __attribute__((always_inline)) {
        x.row = row_of(it);
        x.H = held_by<C, ADJ>(u, d, R, x.row.kind == 2);
        if (!x.row.live) return;
        if (FULL || x.H.e[0] >= 0) x.a.load(x.row.src, x.row.s + x.H.e[0]);
        if (FULL || x.H.e[1] >= 0) x.b.load(x.row.src, x.row.s + x.H.e[1]);
    };
    auto finish = [&](Work& x) __attribute__((always_inline)) {
        if (!x.row.live) return;
        const Held& H = x.H;
        const bool has[2] = {FULL || H.e[0] >= 0, FULL || H.e[1] >= 0};
        const bool four = KV4 && x.row.kind != 0;
        if (!four && (x.row.kind == 2 || !(norm || H.turn[0] || H.turn[1]))) {  // as it is
            if (has[0]) store_as<C, IN32, OUT32>(x.a, x.row.dst, x.row.o + H.e[0]);
            if (has[1]) store_as<C, IN32, OUT32>(x.b, x.row.dst, x.row.o + H.e[1]);
            return;
        }
        double a[C], b[C];
#pragma unroll
        for (int i = 0; i < C; ++i) {
            a[i] = has[0] ? (double)x.a.get(i) : 0.0;
            b[i] = has[1] ? (double)x.b.get(i) : 0.0;
        }
        if (norm && x.row.kind != 2) {
            double s = 0.0;
#pragma unroll
            for (int i = 0; i < C; ++i) s = __fma_rn(a[i], a[i], __fma_rn(b[i], b[i], s));
            const double r = 1.0 / sqrt(head_sum(s, L) / (double)d + (double)N.eps);
            const double* const w = wt + (x.row.kind == 1 ? d : 0);
#pragma unroll
            for (int i = 0; i < C; ++i) {
                if (has[0]) a[i] = a[i] * r * w[H.e[0] + i];
                if (has[1]) b[i] = b[i] * r * w[H.e[1] + i];
            }
        }
        turn_held<C, ADJ, false>(H, cs + x.row.tk * h, a, b);
        if constexpr (KV4 && C > 1) {
            if (four) {
                float f[2][C];
                uint32_t m[2] = {0, 0};
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    f[0][i] = odd21(a[i]);
                    f[1][i] = odd21(b[i]);
                    m[0] = max(m[0], __float_as_uint(f[0][i]) & 0x7FFFFFFFu);  // magnitudes order as whole numbers, NaN last
                    m[1] = max(m[1], __float_as_uint(f[1][i]) & 0x7FFFFFFFu);
                }
                if constexpr (FULL) {
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        m[k] = max(m[k], (uint32_t)__builtin_amdgcn_mov_dpp((int)m[k], 0xB1, 0xF, 0xF, true));
                        m[k] = max(m[k], (uint32_t)__builtin_amdgcn_mov_dpp((int)m[k], 0x4E, 0xF, 0xF, true));
                    }
                } else {
                    // a head has at most as many groups as lanes, which all lie in one wave
                    s_max[tid] = 0;
                    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (has[k]) atomicMax(&s_max[base + (H.e[k] >> 5)], m[k]);
                    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
                    __builtin_amdgcn_wave_barrier();
#pragma unroll
                    for (int k = 0; k < 2; ++k)
                        if (has[k])
                            m[k] = __hip_atomic_load(&s_max[base + (H.e[k] >> 5)], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WAVEFRONT);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    if (!has[k]) continue;
                    const uint32_t top = m[k];
                    const int fld = (int)(top >> 23);
                    const int sc = fld == 255 ? 255 : min(max(fld - ((top & 0x7FFFFFu) < 0x600000u ? 2 : 1), 2), 252);
                    const float by = __uint_as_float((uint32_t)sc << 23);
                    uint32_t w = 0;
                    if (sc != 255) {
                        w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[k][0], f[k][1], by, 0);
                        if constexpr (C == 8) {
                            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[k][2], f[k][3], by, 1);
                            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[k][4], f[k][5], by, 2);
                            w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, f[k][6], f[k][7], by, 3);
                        }
                    }
                    uint8_t* const dst = (uint8_t*)x.row.dst;
                    if (x.row.kind == 2) {  // a byte for each pair of channels, 16 apart
#pragma unroll
                        for (int i = 0; i < C; i += 2) dst[x.row.o + 8 * (H.e[k] + i)] = (uint8_t)(w >> (4 * i));
                        if ((H.e[k] & 31) == 0) x.row.scales[kv4_vscale(x.row.o) + (H.e[k] >> 1)] = (uint8_t)sc;
                    } else {
                        const int64_t at = x.row.o + H.e[k];
                        if constexpr (C == 8) *(uint32_t*)(dst + (at >> 1)) = w;
                        else dst[at >> 1] = (uint8_t)w;
                        if ((H.e[k] & 31) == 0) x.row.scales[at >> 5] = (uint8_t)sc;
                    }
                }
                return;
            }
        }
        Chunk<C, OUT32> y;
        if (has[0]) {
            y.put_all(a);
            y.store(x.row.dst, x.row.o + H.e[0]);
        }
        if (has[1]) {
            y.put_all(b);
            y.store(x.row.dst, x.row.o + H.e[1]);
        }
    };
    int it = (int)blockIdx.y * (NR_THREADS / L) + tid / L;
    Work x;
    if (it < total) fetch(it, x);  // ahead of the sines
    if (h) fill_turns(A, cs, t0, nt);
    if (norm)
        for (int i = tid; i < 2 * d; i += NR_THREADS)
            wt[i] = i < d ? weight_at(N.q_weight, N.weights_fp32, i) : weight_at(N.k_weight, N.weights_fp32, i - d);
    __syncthreads();
    while (it < total) {
        finish(x);
        it += step;
        if (it < total) fetch(it, x);
    }
}

// The gradient. A block takes the q heads or the k heads (the first qblocks blocks those of q) of every so many tokens and keeps
// its sums of g xh, each lane those of its own elements; the lanes that held the same elements meet in LDS at the end.
template <int C, bool F32, bool ADJ, bool FULL>
__global__ void __launch_bounds__(NR_THREADS) ea_norm_rotary_grad_kernel(ea_norm_rotary_grad G, int tpb, int L, int qblocks) {
    extern __shared__ __align__(16) double2 cs[];  // tpb x pairs, the weight (d), and the lanes' sums (256 x 2 C) at the end
    const ea_rotary& A = G.r;
    const int d = A.head_dim, R = A.rot_dim, h = R / 2, tid = threadIdx.x;
    const bool isk = (int)blockIdx.x >= qblocks;
    const int blk = isk ? (int)blockIdx.x - qblocks : (int)blockIdx.x, nblk = isk ? (int)gridDim.x - qblocks : qblocks;
    const int heads = isk ? A.num_kv_heads : A.num_q_heads;
    double* const wt = (double*)(cs + tpb * h);
    const int u = tid & (L - 1);
    const Held H = held_by<C, ADJ>(u, d, R, false);
    const bool has[2] = {FULL || H.e[0] >= 0, FULL || H.e[1] >= 0};
    const void* const xs = isk ? A.k : A.q;
    const void* const gs = isk ? G.gk : G.gq;
    void* const os = isk ? A.k_out : A.q_out;
    const int64_t xt = isk ? A.k_tok_stride : A.q_tok_stride, xh = isk ? A.k_head_stride : A.q_head_stride;
    const int64_t gt = isk ? G.gk_tok_stride : G.gq_tok_stride, gh = isk ? G.gk_head_stride : G.gq_head_stride;
    const int64_t ot = isk ? A.ko_tok_stride : A.qo_tok_stride, oh = isk ? A.ko_head_stride : A.qo_head_stride;
    const bool sums = (isk ? G.dk_weight : G.dq_weight) != nullptr;
    double acc[2][C];
#pragma unroll
    for (int i = 0; i < C; ++i) acc[0][i] = acc[1][i] = 0.0;
    for (int i = tid; i < d; i += NR_THREADS) wt[i] = weight_at(isk ? G.k_weight : G.q_weight, G.weights_fp32, i);
    for (int64_t t0 = (int64_t)blk * tpb; t0 < A.num_tokens; t0 += (int64_t)nblk * tpb) {
        const int nt = (int)min((int64_t)tpb, A.num_tokens - t0);
        __syncthreads();  // the previous tokens' turns are done with
        fill_turns(A, cs, t0, nt);
        __syncthreads();
        for (int it = tid / L; it < nt * heads; it += NR_THREADS / L) {
            const int tk = it / heads, hd = it - tk * heads;
            const int64_t t = t0 + tk;
            Chunk<C, F32> x[2], g[2];
#pragma unroll
            for (int k = 0; k < 2; ++k)
                if (has[k]) {
                    x[k].load(xs, t * xt + hd * xh + H.e[k]);
                    g[k].load(gs, t * gt + hd * gh + H.e[k]);
                }
            double a[C], b[C];
            double s = 0.0, dot = 0.0;
#pragma unroll
            for (int i = 0; i < C; ++i) {
                a[i] = has[0] ? (double)g[0].get(i) : 0.0;
                b[i] = has[1] ? (double)g[1].get(i) : 0.0;
            }
            turn_held<C, ADJ, true>(H, cs + tk * h, a, b);
#pragma unroll
            for (int i = 0; i < C; ++i) {
                const double x0 = has[0] ? (double)x[0].get(i) : 0.0, x1 = has[1] ? (double)x[1].get(i) : 0.0;
                s = __fma_rn(x0, x0, __fma_rn(x1, x1, s));
                const double w0 = has[0] ? wt[H.e[0] + i] : 0.0, w1 = has[1] ? wt[H.e[1] + i] : 0.0;
                dot = __fma_rn(a[i] * w0, x0, __fma_rn(b[i] * w1, x1, dot));
            }
            s = head_sum(s, L);
            dot = head_sum(dot, L);
            const double r = 1.0 / sqrt(s / (double)d + (double)G.eps);
            const double m = dot * r * r / (double)d;  // x r^2 mean(g w xh) / r = x m, before the outer r
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                if (!has[k]) continue;
                Chunk<C, F32> o;
                double y[C];
#pragma unroll
                for (int i = 0; i < C; ++i) {
                    const double gi = k ? b[i] : a[i], xi = (double)x[k].get(i);
                    acc[k][i] = __fma_rn(gi, xi * r, acc[k][i]);
                    y[i] = r * __fma_rn(-xi, m, gi * wt[H.e[k] + i]);
                }
                o.put_all(y);
                o.store(os, t * ot + hd * oh + H.e[k]);
            }
        }
    }
    if (!sums) return;
    double* const red = wt + d;  // [256 / L][d]
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
        for (int i = 0; i < C; ++i)
            if (has[k]) red[(tid / L) * d + H.e[k] + i] = acc[k][i];
    __syncthreads();
    for (int i = tid; i < d; i += NR_THREADS) {
        double s = 0.0;
        for (int g = 0; g < NR_THREADS / L; ++g) s += red[g * d + i];
        G.partial[(int64_t)blockIdx.x * d + i] = s;
    }
}

// the blocks' partial sums to the weights' gradients: 32 elements a block, 32 threads each, in a fixed order
__global__ void __launch_bounds__(1024) ea_norm_weights_kernel(const double* partial, int d, int qblocks, int kblocks, void* dq,
                                                               void* dk, int fp32) {
    __shared__ double part[32][33];
    const int per = (d + 31) / 32;
    const bool isk = (int)blockIdx.x >= per;
    const int x = threadIdx.x & 31, i = ((int)blockIdx.x - (isk ? per : 0)) * 32 + x, y = threadIdx.x >> 5;
    void* const out = isk ? dk : dq;
    if (!out) return;
    const int b0 = isk ? qblocks : 0, n = isk ? kblocks : qblocks;
    double s[4] = {0.0, 0.0, 0.0, 0.0};
    if (i < d)
        for (int b = y; b < n; b += 128)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (b + 32 * k < n) s[k] += partial[(int64_t)(b0 + b + 32 * k) * d + i];
    part[y][x] = (s[0] + s[1]) + (s[2] + s[3]);
    for (int o = 16; o > 0; o >>= 1) {
        __syncthreads();
        if (y < o) part[y][x] += part[y + o][x];
    }
    if (y || i >= d) return;
    if (fp32) ((float*)out)[i] = (float)part[0][x];
    else ((uint16_t*)out)[i] = (uint16_t)f64_bf16(part[0][x]);
}

// rows of K to bf16, 8 elements a thread
__global__ void __launch_bounds__(256) ea_kv4_keys_kernel(int64_t n, int per, int groups, const uint8_t* codes, const uint8_t* scales,
                                                          uint16_t* out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / per;
        const int c = (int)(i - row * per);
        *(uint4*)(out + row * per * 8 + 8 * c) = kv4_load8(codes, scales, row * groups * 32 + 8 * c);
    }
}

// tiles of V to rows of bf16, 8 channels of a tile's 16 slots a thread: 16-byte reads, and writes that are whole rows over the lanes
// (a thread for 8 channels of one slot gathers bytes: 131072 slots of 128 channels 20 us, here 9)
__global__ void __launch_bounds__(256) ea_kv4_tiles_kernel(int64_t n, int per, int groups, const uint8_t* codes, const uint8_t* scales,
                                                           uint16_t* out) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int64_t tile = i / per;
        const int c = (int)(i - tile * per);
        const uint8_t* const p = codes + tile * groups * 256 + 64 * c;
        const uint4 w[4] = {*(const uint4*)p, *(const uint4*)(p + 16), *(const uint4*)(p + 32), *(const uint4*)(p + 48)};
        const uint4 s = *(const uint4*)(scales + tile * groups * 16 + 16 * (c >> 2));
        uint16_t* o = out + tile * 16 * per * 8 + 8 * c;
#pragma unroll
        for (int k = 0; k < 16; ++k, o += per * 8) {
            auto byte = [&](const uint4& x) { return ((k < 4 ? x.x : (k < 8 ? x.y : (k < 12 ? x.z : x.w))) >> (8 * (k & 3))) & 0xFFu; };
            const uint32_t sc = byte(s);
            *(uint4*)o = make_uint4(kv4_bf16x2<0>(byte(w[0]), sc), kv4_bf16x2<0>(byte(w[1]), sc), kv4_bf16x2<0>(byte(w[2]), sc),
                                    kv4_bf16x2<0>(byte(w[3]), sc));
        }
    }
}

// Elements a lane's run holds, 0 where there is no layout: what the rotation pairs stay in whole runs, and a head in 64 lanes
int run_of(int d, int R, bool adjacent, bool wide) {
    const int h = R / 2;
    if (wide && !(d & 7) && !((adjacent ? R : h) & 7)) return 8;
    if (!(d & 1) && (adjacent || !(h & 1))) return 2;
    return d <= 128 && !adjacent ? 1 : 0;
}
int lanes_of(int d, int C) {
    int L = 1;
    while (L * 2 * C < d) L *= 2;
    return L;
}

// every lane holds two whole runs of 8, 4 lanes 32 elements
bool full_lanes(int d, int R, bool adjacent, int C, int L) { return C == 8 && d == 16 * L && d % 64 == 0 && (adjacent || R % 64 == 0); }

template <int C, bool ADJ, bool FULL>
void launch(const ea_norm_rotary& a, dim3 grid, size_t lds, int tpb, int L, hipStream_t st) {
    const bool four = a.k_scales != nullptr;
    auto go = [&](auto* fn) { hipLaunchKernelGGL(fn, grid, dim3(NR_THREADS), lds, st, a, tpb, L); };
    if (!a.r.in_fp32) {
        if (four) go(ea_norm_rotary_kernel<C, false, false, true, ADJ, FULL>);
        else go(ea_norm_rotary_kernel<C, false, false, false, ADJ, FULL>);
    } else if (four) {
        go(ea_norm_rotary_kernel<C, true, false, true, ADJ, FULL>);
    } else if (a.r.out_fp32) {
        go(ea_norm_rotary_kernel<C, true, true, false, ADJ, FULL>);
    } else {
        go(ea_norm_rotary_kernel<C, true, false, false, ADJ, FULL>);
    }
}

// what both directions ask of ea_rotary's fields
int check_rotary(const ea_rotary& r) {
    const int d = r.head_dim, R = r.rot_dim;
    if (r.num_tokens < 0 || r.num_q_heads < 0 || r.num_kv_heads < 0) return -1;
    if (d <= 0 || d > 256 || R < 0 || R > d || (R & 1)) return -1;
    if (r.num_axes <= 0 || (r.num_axes > 1 && !r.axis_of_pair)) return -1;
    if ((r.in_fp32 | 1) != 1 || (r.out_fp32 | 1) != 1 || (r.out_fp32 && !r.in_fp32)) return -2;
    if (!(r.scale - r.scale == 0.0f)) return -2;
    return 0;
}

}  // namespace

extern "C" {

int ea_hip_norm_rotary(const ea_norm_rotary* a, ea_stream_t stream) {
    if (!a) return -1;
    const ea_rotary& r = a->r;
    const int rc = check_rotary(r);
    if (rc) return rc;
    const bool four = a->k_scales || a->v_scales, norm = a->q_weight || a->k_weight;
    if (norm && (!a->q_weight || !a->k_weight)) return -1;
    if (norm && (r.inverse || !(a->eps >= 0.0f) || !(a->eps - a->eps == 0.0f) || (a->weights_fp32 | 1) != 1)) return -2;
    if (!r.half_turns && r.rot_dim) return -1;
    if (four && (!a->k_scales || !a->v_scales || r.out_fp32 || a->page_size <= 0)) return -1;
    if (r.num_tokens == 0 || r.num_q_heads + r.num_kv_heads == 0) return 0;
    if ((r.rot_dim && !r.positions) || r.pool_rows < 0 || r.q_out_rows < 0) return -1;
    if (r.num_q_heads > 0 && (!r.q || !r.q_out)) return -1;
    if (r.num_kv_heads > 0 && (!r.k || !r.k_out || (r.v && !r.v_out))) return -1;
    const int d = r.head_dim, R = r.rot_dim;
    if (four) {
        if ((d & 7) || (R & 3)) return -1;
        if (((r.ko_tok_stride | r.ko_head_stride | a->k_page_stride) & 31) || ((r.vo_head_stride | a->v_page_stride) & 127)) return -1;
        if (r.v && (r.vo_tok_stride != kv4_width(d) || (a->page_size & 15))) return -1;
        if (((uintptr_t)r.k_out & 3) || (r.v && ((uintptr_t)r.v_out & 15))) return -1;
    }
    // 16-byte accesses: every row of every tensor starts on one (a 4-bit row's runs of 8 are 4 bytes)
    const int64_t in = r.in_fp32 ? 4 : 8, out = r.out_fp32 ? 4 : 8;
    uintptr_t ptr = 0;
    int64_t si = 0, so = 0;
    if (r.num_q_heads > 0) {
        ptr |= (uintptr_t)r.q | (uintptr_t)r.q_out;
        si |= r.q_tok_stride | r.q_head_stride;
        so |= r.qo_tok_stride | r.qo_head_stride;
    }
    if (r.num_kv_heads > 0) {
        ptr |= (uintptr_t)r.k | (r.v ? (uintptr_t)r.v : 0);
        si |= r.k_tok_stride | r.k_head_stride | (r.v ? r.v_tok_stride | r.v_head_stride : 0);
        if (!four) {
            ptr |= (uintptr_t)r.k_out | (r.v ? (uintptr_t)r.v_out : 0);
            so |= r.ko_tok_stride | r.ko_head_stride | (r.v ? r.vo_tok_stride | r.vo_head_stride : 0);
        }
    }
    const bool wide = !(ptr & 15) && !(si & (in - 1)) && !(so & (out - 1));
    const int C = run_of(d, R, r.adjacent != 0, wide);
    if (C == 0 || (four && C == 1)) return -1;
    const int L = lanes_of(d, C), per = NR_THREADS / L;
    const int items = r.num_q_heads + r.num_kv_heads * (r.v ? 2 : 1);
    // tokens a block: as the rotation alone takes them
    int tpb = 1;
    while (r.num_tokens >= 1536 && tpb < 4 && 2 * tpb * items <= per) tpb *= 2;
    if (r.num_tokens >= 8192) tpb = std::max(tpb, 2);
    if ((int64_t)items * tpb >= (int64_t)1 << 30) return -1;
    const int64_t slices = r.num_tokens < 768 ? std::min<int64_t>((items + per - 1) / per, 64) : 1;
    const dim3 grid((unsigned)(((int64_t)r.num_tokens + tpb - 1) / tpb), (unsigned)slices);
    const size_t lds = (size_t)tpb * (R / 2) * 16 + (size_t)2 * d * 8;
    const hipStream_t st = (hipStream_t)stream;
    const bool full = full_lanes(d, R, r.adjacent != 0, C, L);
    if (r.adjacent) {
        if (full) launch<8, true, true>(*a, grid, lds, tpb, L, st);
        else if (C == 8) launch<8, true, false>(*a, grid, lds, tpb, L, st);
        else launch<2, true, false>(*a, grid, lds, tpb, L, st);
    } else {
        if (full) launch<8, false, true>(*a, grid, lds, tpb, L, st);
        else if (C == 8) launch<8, false, false>(*a, grid, lds, tpb, L, st);
        else if (C == 2) launch<2, false, false>(*a, grid, lds, tpb, L, st);
        else launch<1, false, false>(*a, grid, lds, tpb, L, st);
    }
    return herr(hipGetLastError());
}

// blocks of the q heads and of the k heads, in proportion
static void grad_blocks(const ea_norm_rotary_grad& a, int tpb, int* q, int* k) {
    const int64_t steps = ((int64_t)a.r.num_tokens + tpb - 1) / tpb, H = (int64_t)a.r.num_q_heads + a.r.num_kv_heads;
    auto share = [&](int heads) {
        return heads ? (int)std::max<int64_t>(1, std::min<int64_t>(steps, (int64_t)NG_BLOCKS * heads / H)) : 0;
    };
    *q = share(a.r.num_q_heads);
    *k = share(a.r.num_kv_heads);
}
static const int NG_TOKENS = 4;

size_t ea_hip_norm_rotary_grad_size(const ea_norm_rotary_grad* a) {
    if (!a || a->r.num_tokens <= 0 || a->r.num_q_heads < 0 || a->r.num_kv_heads < 0 || a->r.head_dim <= 0 ||
        a->r.num_q_heads + a->r.num_kv_heads == 0)
        return 0;
    int q, k;
    grad_blocks(*a, NG_TOKENS, &q, &k);
    return (size_t)(q + k) * a->r.head_dim * 8;
}

int ea_hip_norm_rotary_grad(const ea_norm_rotary_grad* a, ea_stream_t stream) {
    if (!a) return -1;
    const ea_rotary& r = a->r;
    const int rc = check_rotary(r);
    if (rc) return rc;
    if (r.inverse || r.out_fp32 != r.in_fp32 || !(a->eps >= 0.0f) || !(a->eps - a->eps == 0.0f) || (a->weights_fp32 | 1) != 1) return -2;
    if (!a->q_weight || !a->k_weight || (r.rot_dim && !r.half_turns)) return -1;
    const hipStream_t st = (hipStream_t)stream;
    if (r.num_q_heads + r.num_kv_heads == 0) return 0;
    if (r.num_tokens > 0 && r.rot_dim && !r.positions) return -1;
    if (r.num_tokens > 0 && r.num_q_heads > 0 && (!r.q || !r.q_out || !a->gq || r.q == r.q_out)) return -1;
    if (r.num_tokens > 0 && r.num_kv_heads > 0 && (!r.k || !r.k_out || !a->gk || r.k == r.k_out)) return -1;
    const bool sums = a->dq_weight || a->dk_weight;
    if (r.num_tokens > 0 && sums && !a->partial) return -1;
    const int d = r.head_dim, R = r.rot_dim;
    int qb = 0, kb = 0;
    if (r.num_tokens > 0) {
        const int64_t al = r.in_fp32 ? 4 : 8;
        uintptr_t ptr = 0;
        int64_t s = 0;
        if (r.num_q_heads > 0) {
            ptr |= (uintptr_t)r.q | (uintptr_t)r.q_out | (uintptr_t)a->gq;
            s |= r.q_tok_stride | r.q_head_stride | r.qo_tok_stride | r.qo_head_stride | a->gq_tok_stride | a->gq_head_stride;
        }
        if (r.num_kv_heads > 0) {
            ptr |= (uintptr_t)r.k | (uintptr_t)r.k_out | (uintptr_t)a->gk;
            s |= r.k_tok_stride | r.k_head_stride | r.ko_tok_stride | r.ko_head_stride | a->gk_tok_stride | a->gk_head_stride;
        }
        const int C = run_of(d, R, r.adjacent != 0, !(ptr & 15) && !(s & (al - 1)));
        if (C == 0) return -1;
        const int L = lanes_of(d, C), tpb = NG_TOKENS;
        grad_blocks(*a, tpb, &qb, &kb);
        // 42 KB at most: 4 turns of 128 pairs, 256 weights, and 256 / L rows of d <= 16 L sums
        const size_t lds = (size_t)tpb * (R / 2) * 16 + (size_t)d * 8 + (sums ? (size_t)(NR_THREADS / L) * d * 8 : 0);
        auto go = [&](auto* fn) -> int {
            hipLaunchKernelGGL(fn, dim3((unsigned)(qb + kb)), dim3(NR_THREADS), lds, st, *a, tpb, L, qb);
            return herr(hipGetLastError());
        };
        auto both = [&](auto* wide, auto* narrow) -> int { return r.in_fp32 ? go(wide) : go(narrow); };
        const bool full = full_lanes(d, R, r.adjacent != 0, C, L);
        int e;
        if (r.adjacent) {
            if (full) e = both(ea_norm_rotary_grad_kernel<8, true, true, true>, ea_norm_rotary_grad_kernel<8, false, true, true>);
            else if (C == 8) e = both(ea_norm_rotary_grad_kernel<8, true, true, false>, ea_norm_rotary_grad_kernel<8, false, true, false>);
            else e = both(ea_norm_rotary_grad_kernel<2, true, true, false>, ea_norm_rotary_grad_kernel<2, false, true, false>);
        } else if (full) {
            e = both(ea_norm_rotary_grad_kernel<8, true, false, true>, ea_norm_rotary_grad_kernel<8, false, false, true>);
        } else if (C == 8) {
            e = both(ea_norm_rotary_grad_kernel<8, true, false, false>, ea_norm_rotary_grad_kernel<8, false, false, false>);
        } else if (C == 2) {
            e = both(ea_norm_rotary_grad_kernel<2, true, false, false>, ea_norm_rotary_grad_kernel<2, false, false, false>);
        } else {
            e = both(ea_norm_rotary_grad_kernel<1, true, false, false>, ea_norm_rotary_grad_kernel<1, false, false, false>);
        }
        if (e) return e;
    }
    if (sums) {
        hipLaunchKernelGGL(ea_norm_weights_kernel, dim3((unsigned)(2 * ((d + 31) / 32))), dim3(1024), 0, st, a->partial, d, qb, kb,
                           a->dq_weight, a->dk_weight, a->weights_fp32);
        return herr(hipGetLastError());
    }
    return 0;
}

int ea_hip_kv4_values(int64_t rows, int32_t head_dim, int32_t is_v, const uint8_t* codes, const uint8_t* scales, uint16_t* values,
                      ea_stream_t stream) {
    if (rows < 0 || head_dim <= 0 || (head_dim & 7) || (is_v && (rows & 15))) return -1;
    if (rows == 0) return 0;
    if (!codes || !scales || !values || ((uintptr_t)codes & 3) || ((uintptr_t)values & 15)) return -1;
    const int per = head_dim / 8;
    if (rows > (((int64_t)1 << 62) / head_dim)) return -1;
    const int64_t n = (is_v ? rows / 16 : rows) * per;
    const unsigned grid = (unsigned)std::min<int64_t>((n + 255) / 256, 8192);
    const auto fn = is_v ? ea_kv4_tiles_kernel : ea_kv4_keys_kernel;
    hipLaunchKernelGGL(fn, dim3(grid), dim3(256), 0, (hipStream_t)stream, n, per, (head_dim + 31) / 32, codes, scales, values);
    return herr(hipGetLastError());
}

}  // extern "C"

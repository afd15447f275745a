// Certified prefill on the CDNA4 int8 matrix cores (gfx950): exact q.k scores and P.V sums from
// v_mfma_i32_16x16x64_i8 over balanced radix-256 digits of the bf16 inputs.
//
// Reference behaviour: the tensor-core split program of src/exactattn/triton_kernels.py
// (_tc_logits :395-482, _tc_pv :512-648, slices.slice_rows :31-52) and the definition in
// docs/SPEC.md. The arithmetic here is designed for CDNA4, not translated:
//
//   digits  a bf16 vector (q row, K row, V row) becomes integers X_i = x_i / 2^lsb with
//           |X_i| < 2^30, lsb = (top bit position over the vector) - 29, rounded to nearest where
//           an element lies more than 22 binades below the vector's top (counted, bounded).
//           X splits into 4 balanced digits d_s in [-128, 127], X = sum_s d_s 256^s: the bytes of
//           X + 0x80808080 with their top bits flipped. q and K use digits 1..3 (24 bits) unless
//           a digit 0 is nonzero (per wave of 16 rows, per 16-key group); V uses all four.
//   scores  S^T = K Q^T per 16 keys x 16 rows: one MFMA per digit pair and 64 dims, digit pairs of
//           equal weight s + t share an int32 accumulator (|acc| < 2^23). The fp64 Horner fold of
//           the 7 accumulators is within 6.01 u sum_i A_q,i A_k,i of the exact integer, and the
//           certified t = RN32(alpha s) is taken from that interval (ea_device.h logit_cert);
//           undecided pairs are recomputed exactly in the lane (TwoSum over bf16 products).
//   weights w = RN24(2^t) = M 2^E in fp64 (tables + cubic, 128-bit enclosure when undecided).
//   P.V     the S^T output layout leaves each lane 16 keys of one row, which is the A-operand
//           layout of the P.V MFMA (rows x keys): no transpose. Per row a base exponent; the
//           weight of key j enters as Wf = RN(M 2^(E + vlsb_j - base)) <= 2^38 (the V row's lsb
//           folded into the weight), as 5 balanced digits read straight out of the fp64 sum
//           Wf + 0x8080808080 + 1.5 * 2^52. acc_c = sum_j Wf_j X_jc over digit pairs s + t >= 2
//           (the 3 omitted pairs are bounded: 513 * 2^20 per tile), int32 accumulators kept
//           across tiles and folded into fp64 only when a row's base must move (a weight above
//           2^38) or after 256 tiles. Error bound per (row, channel):
//             |N/2^base - acc| <= sum_j |X_jc| / 2 + (2^38 + 1)/2 * (inexact V elements)
//                                 + omitted pairs + fold roundings.
//   Z       fp64 sum of the exact weights 2^(E - base), bound (n + 8) u' Z.
//   final   RN(N/Z) certified per channel (certify_round); rows with an undecided pair or
//           channel go to the device tier 2 work list, NaN/inf and logit overflow are flag 2.
//
// Kernels: ea_pf_qslice (q rows -> digits), ea_pf_kvslice (K/V pages -> 64-key digit tiles with
// per-key and per-channel metadata: the KV-cache slice format), ea_pf_main (one block of 4 waves
// per 64 rows of a segment, 16 rows per wave, K/V digit tiles DMA'd to LDS and double-buffered).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>
#include <mutex>

#include "ea_params.h"
#include "ea_pf_common.h"
#include "ea_pf_main.h"

using namespace ea;
using namespace ea::pf;

namespace {


__device__ __forceinline__ void bf16_dec(uint32_t x, int* m, int* e, int* bad) {
    int f = (x >> 7) & 0xFF;
    int mm = (int)(x & 0x7F) | (f ? 0x80 : 0);
    *m = (x & 0x8000) ? -mm : mm;
    *e = (f ? f : 1) - 134;
    *bad = f == 0xFF;
}

__device__ __forceinline__ int lead_of(int m, int e) {
    int a = m < 0 ? -m : m;
    return e + 31 - __clz(a);
}

// X = RN(m 2^(e - lsb)) (half away from zero), with |m 2^(e - lsb)| < 2^30 guaranteed by lsb
__device__ __forceinline__ int to_fixed(int m, int e, int lsb, int* inexact) {
    int sh = e - lsb;
    int a = m < 0 ? -m : m;
    int r;
    if (sh >= 0) {
        r = a << sh;
        *inexact = 0;
    } else {
        int s = -sh;
        if (s > 10) {
            r = 0;
            *inexact = a != 0;
        } else {
            r = (a + (1 << (s - 1))) >> s;
            *inexact = (r << s) != a;
        }
    }
    return m < 0 ? -r : r;
}

// digit bytes of X (|X| < 2^30): byte s is digit s, in two's complement
__device__ __forceinline__ uint32_t digits_of(int X) { return ((uint32_t)X + 0x80808080u) ^ 0x80808080u; }
// sum_s |d_s| 256^s: every byte's magnitude (at most 128) in place, below 2^32
__device__ __forceinline__ uint32_t digit_abs(uint32_t v) {
    const uint32_t neg = (v >> 7) & 0x01010101u;
    return (v ^ (neg * 255u)) + neg;
}

// ------------------------------------------------------------------------------------------------
// Digits of NE consecutive bf16 elements held by one lane; the G = 128 / NE adjacent lanes of a
// group (lane & (G - 1)) cover a 128-element vector. Returns the vector's lsb (group-uniform) and
// the digit bytes (4 planes x NE bytes, as NE / 4 dwords per plane). K/V rows take NE = 32 (a quad
// per key); q rows NE = 8 (16 lanes per row: four times the lanes, a quarter of the chain). All of it in integers:
// with magnitudes as fp64 sums, digits picked byte by byte and shuffles through LDS 65536 q rows took 20.9
// us (now 17 to 19) and the K and V of 8 x 4096 keys 30.3 (25.9).
// ------------------------------------------------------------------------------------------------
template <int NE>
struct SliceN {
    int lsb, bad, inex, need4, xmax;
    double amax, asum;
    uint32_t dig[4][NE / 4];
};
using Slice32 = SliceN<32>;

// over the group's G lanes, in every one of them: rotations within a row of 16 lanes, or permutations within a
// quad
template <int G, typename F>
__device__ __forceinline__ int grp_all(int x, F f) {
    static_assert(G == 16 || G == 4, "a DPP row or quad");
    if constexpr (G == 16) {
        x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x128, 0xF, 0xF, false));  // row_ror 8, 4, 2, 1
        x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x124, 0xF, 0xF, false));
        x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x122, 0xF, 0xF, false));
        return f(x, __builtin_amdgcn_update_dpp(0, x, 0x121, 0xF, 0xF, false));
    } else {
        x = f(x, __builtin_amdgcn_update_dpp(0, x, 0xB1, 0xF, 0xF, false));  // quad_perm 1 0 3 2, 2 3 0 1
        return f(x, __builtin_amdgcn_update_dpp(0, x, 0x4E, 0xF, 0xF, false));
    }
}
template <int G>
__device__ __forceinline__ int grp_max(int x) {
    return grp_all<G>(x, [](int a, int b) { return max(a, b); });
}
template <int G>
__device__ __forceinline__ int grp_sum(int x) {
    return grp_all<G>(x, [](int a, int b) { return a + b; });
}

// src: NE bf16 values (any alignment of 2 bytes); valid = false gives an all-zero vector.
// lost[c] (optional) receives 1 for each element that is not exact in 30 bits. have: the elements there
// are, a multiple of 8 (negative: none); the others are zeros.
template <int NE>
__device__ __forceinline__ void slice_n(const uint16_t* src, bool valid, SliceN<NE>& S, int* lost = nullptr, int have = NE) {
    constexpr int G = 128 / NE;
    int m[NE], e[NE];
    int bad = 0, lead = INT_MIN;
    // the 2 NE bytes as 16-byte loads when they start on a 16-byte boundary (the usual cache
    // strides), else element by element
    uint32_t raw[NE / 2];
    if (valid && ((uintptr_t)src & 15) == 0) {
#pragma unroll
        for (int i = 0; i < NE / 8; ++i) {
            const uint4 v = 8 * i < have ? ((const uint4*)src)[i] : make_uint4(0, 0, 0, 0);
            raw[4 * i] = v.x;
            raw[4 * i + 1] = v.y;
            raw[4 * i + 2] = v.z;
            raw[4 * i + 3] = v.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < NE / 2; ++i)
            raw[i] = valid && 2 * i < have ? ((uint32_t)src[2 * i] | ((uint32_t)src[2 * i + 1] << 16)) : 0u;
    }
#pragma unroll
    for (int k = 0; k < NE; ++k) {
        int bk;
        bf16_dec((raw[k >> 1] >> (16 * (k & 1))) & 0xFFFFu, &m[k], &e[k], &bk);
        bad |= bk;
        if (m[k] && !bk) lead = max(lead, lead_of(m[k], e[k]));
    }
    lead = grp_max<G>(lead);
    bad = grp_max<G>(bad);
    const int lsb = (lead == INT_MIN) ? 0 : lead - 29;
    int inex = 0, xmax = 0;
    uint32_t amax = 0, low = 0;
    uint64_t asum = 0;
#pragma unroll
    for (int w4 = 0; w4 < NE / 4; ++w4) {
        uint32_t v[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int kk = 4 * w4 + k;
            int ie = 0;
            const int X = (bad || m[kk] == 0) ? 0 : to_fixed(m[kk], e[kk], lsb, &ie);
            inex += ie;
            if (lost) lost[kk] = ie;
            v[k] = digits_of(X);
            low |= v[k] & 0xFFu;
            const uint32_t a = digit_abs(v[k]);
            amax = max(amax, a);
            asum += a;
            xmax = max(xmax, X < 0 ? -X : X);
        }
        // plane s: byte k of dword w4 = digit s of element 4 w4 + k, a transposition of 4 x 4 bytes
        const uint32_t lo01 = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u), hi01 = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);
        const uint32_t lo23 = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u), hi23 = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
        S.dig[0][w4] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100u);
        S.dig[1][w4] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302u);
        S.dig[2][w4] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100u);
        S.dig[3][w4] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302u);
    }
    S.lsb = lsb;
    S.bad = bad;
    S.inex = grp_sum<G>(inex);
    S.need4 = grp_max<G>(low != 0);
    S.xmax = grp_max<G>(xmax);
    S.amax = (double)(uint32_t)grp_all<G>((int)amax, [](int a, int b) { return (int)max((uint32_t)a, (uint32_t)b); });
    const int hi = grp_sum<G>((int)(asum >> 20)), lo = grp_sum<G>((int)(asum & 0xFFFFF));
    S.asum = (double)hi * 0x1p20 + (double)lo;  // exact: integers below 2^41
}
__device__ __forceinline__ void slice32(const uint16_t* src, bool valid, Slice32& S, int* lost = nullptr, int have = 32) {
    slice_n<32>(src, valid, S, lost, have);
}

}  // namespace

// ------------------------------------------------------------------------------------------------
// q rows -> digit planes: 16 rows per block, 16 lanes per row (8 dims each: a short chain per lane,
// which is what a step of few rows, such as tree verification, waits on). Also clears the tier-2
// work-list counter (this is the step's first kernel on the prefill path).
// ------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(256) ea_pf_qslice(Params P) {
    if (blockIdx.x == 0 && threadIdx.x < EA_T2_CNT) P.wl_cnt[threadIdx.x] = 0;
    const int q16 = threadIdx.x & 15;
    const int64_t row = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (row >= P.rows) return;  // whole 16-lane groups leave together
    const int Hq = P.g.num_q_heads, T = P.g.num_tokens;
    const int64_t b = row / ((int64_t)T * Hq);
    const int t = (int)((row / Hq) % T), hq = (int)(row % Hq);
    const uint16_t* qr = P.q + b * P.g.q_seq_stride + (int64_t)t * P.g.q_tok_stride + (int64_t)hq * P.g.q_head_stride;
    SliceN<8> S;
    slice_n<8>(qr + 8 * q16, 8 * q16 < P.g.head_dim, S);  // dims past the head's are zeros
    uint8_t* dst = P.pfq + row * 512 + 8 * q16;
#pragma unroll
    for (int sp = 0; sp < 4; ++sp) *(uint2*)(dst + 128 * sp) = make_uint2(S.dig[sp][0], S.dig[sp][1]);
    if (q16 == 0) {
        PfQMeta* qm = (PfQMeta*)P.pfqm + row;
        qm->lsb = S.lsb;
        qm->flags = S.need4 | (S.bad << 1) | (min(S.inex, 255) << 8);
        qm->qA = S.asum;
        qm->qX = (double)S.xmax;
        qm->a = ldexp(P.alpha, S.lsb);
    }
}

// ------------------------------------------------------------------------------------------------
// K/V pages -> one 64-key digit tile per block (segment-major), in the LDS layout of ea_pf_main.
// Lane quad (key = tid / 4) covers the key's 128 dims and 128 channels. K planes are written
// straight to memory in 16-byte chunks; the V planes (keys interleaved per channel) are
// assembled in LDS and copied out in 16-byte chunks.
// ------------------------------------------------------------------------------------------------
// MOD (score modifications): tiles wholly before the first key that a token of the sequence sees are left
// out; no row of ea_pf_main reads them. Heads of fewer dims or channels than 128 are padded with zeros.
template <bool MOD>
__global__ void __launch_bounds__(256) ea_pf_kvslice(Params P) {
    __shared__ __align__(16) uint8_t s_v[32768];
    __shared__ int s_lc[128];
    __shared__ int s_tfl;
    const int tid = threadIdx.x, q4 = tid & 3, key = tid >> 2;
    int seg, tile;
    if (P.kvd_begin) {
        // cache update: block i of a segment re-slices the i-th tile that holds an appended key
        seg = blockIdx.x / P.kvd_span;
        const int bs = seg / P.g.num_kv_heads;
        const int kb = max(P.kvd_begin[bs], 0), ke = P.kvd_end[bs];
        tile = kb / 64 + (int)(blockIdx.x % P.kvd_span);
        if (ke <= kb || tile * 64 >= ke || tile >= P.pf_ntiles) return;  // uniform: the whole block
    } else {
        seg = blockIdx.x / P.pf_ntiles;
        tile = blockIdx.x % P.pf_ntiles;
    }
    const int Hkv = P.g.num_kv_heads;
    const int64_t b = seg / Hkv;
    const int hk = seg % Hkv;
    if constexpr (MOD) {
        int first = INT_MAX;
        for (int t = tid; t < P.g.num_tokens; t += 256) {
            const int64_t tok = b * P.g.num_tokens + t;
            const int kvl = P.kv_len[tok];
            first = min(first, key_span(vis_begin(P, tok, kvl), kvl, P.seq_len[b], P.tree_mask ? P.tree_mask[tok] : 0ull,
                                        P.tree_mask ? P.tree_base[b] : 0).beg);
        }
        if (!__syncthreads_or(first < 64 * (tile + 1))) return;
    }
    uint8_t* T = P.pfkv + ((int64_t)seg * P.pf_ntiles + tile) * EA_PF_TILE_BYTES;
    PfTileMeta* TM = (PfTileMeta*)(T + EA_PF_META_OFF);
    if (tid < 128) s_lc[tid] = 0;
    if (tid == 0) s_tfl = 0;
    __syncthreads();
    const int64_t n = (int64_t)tile * 64 + key;
    const bool valid = n < P.seq_len[b];
    const uint16_t* kr = P.k + (valid ? kv_off(P, b, n, hk, 0) : 0) + 32 * q4;
    const uint16_t* vr = P.v + (valid ? kv_off(P, b, n, hk, 1) : 0) + 32 * q4;
    int bad;
    {
        Slice32 S;
        slice32(kr, valid, S, nullptr, MOD ? P.g.head_dim - 32 * q4 : 32);
#pragma unroll
        for (int sp = 0; sp < 4; ++sp) {
#pragma unroll
            for (int hh = 0; hh < 2; ++hh) {
                const int c = 2 * q4 + hh;  // 16-byte chunk of dims 16c .. 16c+15
                *(uint4*)(T + sp * 8192 + key * 128 + ((c ^ (key & 7)) << 4)) =
                    make_uint4(S.dig[sp][4 * hh], S.dig[sp][4 * hh + 1], S.dig[sp][4 * hh + 2], S.dig[sp][4 * hh + 3]);
            }
        }
        bad = S.bad;
        if (q4 == 0) {
            TM->lsbk[key] = S.lsb;
            TM->kA[key] = ldexp(S.amax, S.lsb);  // in absolute units: the score bound needs no rescale
            TM->kX[key] = (double)S.xmax;
        }
        int tf = (S.need4 ? 1 : 0) << (key >> 4);
        if (S.inex) tf |= 32;
        if (q4 == 0 && tf) atomicOr(&s_tfl, tf);
        bad |= 0;
        if (q4 == 0) TM->kfl[key] = min(S.inex, 255) << 8;  // bit 0 set below with V
    }
    {
        Slice32 S;
        int lost[32];
        slice32(vr, valid, S, lost, MOD ? P.g.head_dim_v - 32 * q4 : 32);
        const int gq = (key >> 2) & 3, kt = key >> 4, ii = key & 3;
#pragma unroll
        for (int sp = 0; sp < 4; ++sp)
#pragma unroll
            for (int k = 0; k < 32; ++k) {
                const int ch = 32 * q4 + k;
                s_v[sp * 8192 + ch * 64 + ((gq ^ ((ch >> 1) & 3)) << 4) + 4 * kt + ii] =
                    (uint8_t)(S.dig[sp][k >> 2] >> (8 * (k & 3)));
            }
        if (S.inex) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
                if (lost[k]) atomicAdd(&s_lc[32 * q4 + k], 1);
        }
        bad = grp_max<4>(bad | S.bad);
        if (q4 == 0) {
            TM->vlsb[key] = S.lsb;
            if (bad) {
                TM->kfl[key] |= 1;
                atomicOr(&s_tfl, 16);
            }
        }
    }
    __syncthreads();
    const uint4* sv4 = (const uint4*)s_v;
    uint4* dv4 = (uint4*)(T + 32768);
#pragma unroll
    for (int i = 0; i < 8; ++i) dv4[tid + 256 * i] = sv4[tid + 256 * i];
    if (tid < 128) TM->EV[tid] = 0.5 * (0x1p38 + 1.0) * (double)s_lc[tid];
    const int tot = tid < 64 ? wave_scan_dpp(s_lc[tid] + s_lc[tid + 64]) : 0;
    if (tid == 63) {
        TM->tfl = s_tfl;
        TM->pad = 0;
        TM->EVt = 0.5 * (0x1p38 + 1.0) * (double)tot;
    }
}

// ------------------------------------------------------------------------------------------------
// Merge of the key splits' partials (pf_nsplit > 1) and the certified final rounding, one block of
// 128 threads per row (thread = channel). Per split s with keys: Z_s and N_s in units 2^base_s with
// bounds (nv_s + 8) u' Z_s + (nv_s + 64) 2^-1074 (the sums of the split's weights, as the kernel's
// own epilogue bounds them) and en_s. Rescaled to the largest base B by exact powers of two (an
// underflowing rescale loses at most 2^-1074 per term, added), then summed: ns - 1 more roundings
// of at most u of the sum of magnitudes. q = N RN(1/Z) and its radius as in ea_pf_main's epilogue,
// then certify_round; rows that fail go to the tier-2 work list.
// ------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) ea_pf_combine(Params P) {
    const int64_t row = blockIdx.x;
    const int c = threadIdx.x;
    const int ns = P.pf_nsplit;
    const PfPart* const parts = (const PfPart*)P.pf_part;
    const double2* const ent = (const double2*)(parts + (int64_t)ns * P.rows);
    int B = INT_MIN, nv = 0, fl = 0;
    for (int s = 0; s < ns; ++s) {
        const PfPart pr = parts[(int64_t)s * P.rows + row];
        fl |= pr.fl;
        if (pr.nv > 0) {
            B = max(B, pr.base);
            nv += pr.nv;
        }
    }
    uint32_t bits = 0;
    bool fin = false;
    if (nv > 0 && !fl) {
        double z = 0.0, ezs = 0.0, nn = 0.0, an = 0.0, en = 0.0;
        for (int s = 0; s < ns; ++s) {
            const PfPart pr = parts[(int64_t)s * P.rows + row];
            if (pr.nv <= 0) continue;
            const int dsh = max(pr.base - B, -1100);
            const double zs = ldexp(pr.z, dsh);
            z += zs;
            ezs += (double)(pr.nv + 8) * PF_U * zs + (double)(pr.nv + 65) * 0x1p-1074;
            const double2 e = ent[((int64_t)s * P.rows + row) * 128 + c];
            const double v = ldexp(e.x, dsh);
            nn += v;
            an += fabs(v);
            en += ldexp(e.y, dsh) + 0x1p-1074;
        }
        // the merge's own roundings (ns - 1 additions each for Z and N, sums of positive bounds
        // rounded up by the (1 + 2^-40) factors)
        const double eZ = (ezs + (double)ns * PF_U * z) * (1.0 + 0x1p-40);
        en = (en + (double)ns * 0x1p-52 * an) * (1.0 + 0x1p-40);
        const bool zok = z > 2.0 * eZ && isfinite(z);
        const double rz = zok ? 1.0 / z : 0.0, rze = zok ? 1.0 / (z - eZ) : 0.0;
        const double q = nn * rz;
        double delta = (en * (1.0 + 0x1p-40) + fabs(q) * eZ) * rze * (1.0 + 0x1p-40) + fabs(q) * 0x1p-51 + 0x1p-1070;
        if (!isfinite(q) || !isfinite(delta) || !zok) delta = __builtin_inf();
        fin = c < P.g.head_dim_v && !certify_round(q, delta, P.out_fp32, &bits);
        if (fin) bits = 0;
    }
    const bool anyfin = __syncthreads_or(fin) != 0;  // every thread reaches this barrier
    const int flag = (fl & 1) ? 2 : (((fl & 2) || anyfin) ? 1 : 0);
    const int Hq = P.g.num_q_heads, T = P.g.num_tokens;
    const int64_t b = row / ((int64_t)T * Hq);
    const int t = (int)((row / Hq) % T), hq = (int)(row % Hq);
    const int64_t o = b * P.g.o_seq_stride + (int64_t)t * P.g.o_tok_stride + (int64_t)hq * P.g.o_head_stride + c;
    if (flag) bits = 0;
    if (c < P.g.head_dim_v) {
        if (P.out_fp32) ((uint32_t*)P.out)[o] = bits;
        else ((uint16_t*)P.out)[o] = (uint16_t)bits;
    }
    if (c == 0) {
        P.flags[row] = (uint8_t)flag;
        if (flag == 1) {
            const int slot = atomicAdd(P.wl_cnt, 1);
            P.wl[slot] = (int32_t)row;
        }
        if (P.stats && flag) {
            atomicAdd((unsigned long long*)&P.stats[1], 1ull);
            if (flag == 2) atomicAdd((unsigned long long*)&P.stats[4], 1ull);
            if (flag == 1 && !(fl & 2)) atomicAdd((unsigned long long*)&P.stats[7], 1ull);
        }
    }
}

namespace {
// kernel shape: 32 rows per block; 8 waves (2 row groups x 4 waves, 2 waves per SIMD, 256
// registers each) by default, ea_options.prefill_waves = 4 selects 4 waves (2 x 2, 1 wave per SIMD)
constexpr int PF_RPB = 32;
}  // namespace

int ea::ea_prefill_eligible(const ea_geometry& g, int grp, int kernel, int* ntiles, int* nrb, bool padded) {
    if (kernel == EA_KERNEL_DECODE || kernel == EA_KERNEL_GENERAL) return 0;
    const bool force = kernel == EA_KERNEL_PREFILL;
    if ((g.head_dim != 128 || g.head_dim_v != 128) && (!padded || (g.head_dim_v & 7))) return 0;
    const int64_t r_seg = (int64_t)g.num_tokens * grp;
    // Rows of one (sequence, KV head) that fill a 32-row block (64 tokens, or fewer tokens with a
    // wider GQA group: speculative trees, chunked prefill) read each K/V tile once here, against
    // once per 1-2 rows in the decode kernel (C4: 0.82 ms here, 2.57 ms there with 4-row blocks)
    // Segments of 24-31 rows (verification of 12-15 draft tokens at GQA 2) come here too when
    // there is enough work: measured on MI355X against the decode kernel (2-row blocks, a
    // segment's row blocks on one XCD; contiguous K/V, graph replays), which took the other steps
    // then, the int8 kernel is 14-45%
    // faster at 24 rows with 8K+ keys on 16+ segments or 32K+ keys on any; at 16 rows the decode
    // kernel is as fast or faster everywhere measured (up to 1.9x at 2K keys, within 3% at 64
    // segments of 32K keys). The multi-row kernel takes the steps left now: of 12 to 20 rows, 2K to
    // 32K keys and 8 to 256 segments all are slower here when K and V are sliced in the step (20 rows,
    // 256 segments of 8K keys 1362 against 797 us); with the tiles cached 12 to 16 rows are even (within
    // 10%) on 32 segments of 8K keys and more, and 20 rows faster here from 32K keys on 8 segments, 8K on 32
    // or 2K on 128 on (448 against 797). The line at 24 rows has not been drawn again.
    const int64_t nseg = (int64_t)g.num_seqs * g.num_kv_heads;
    const bool mid = r_seg >= 24 && g.max_seq_len >= 8192 && (nseg >= 16 || g.max_seq_len >= 32768);
    if (!force && g.num_tokens < 64 && r_seg < PF_RPB && !mid) return 0;
    if (r_seg >= (1 << 30) || (int64_t)g.max_seq_len + 64 >= (1 << 30)) return 0;
    const int rpb = PF_RPB;
    *ntiles = (g.max_seq_len + 63) / 64;
    *nrb = (int)((r_seg + rpb - 1) / rpb);
    return 1;
}

int ea::ea_launch_prefill(const Params& P, hipStream_t st) {
    static std::once_flag once;
    static hipError_t attr_err = hipSuccess;
    std::call_once(once, [] {
        const void* fns[7] = {(const void*)ea_pf_main<4, false>, (const void*)ea_pf_main<4, true>,
                              (const void*)ea_pf_main<8, false>, (const void*)ea_pf_main<8, true>,
                              ea_pf_mod_fn(1), ea_pf_mod_fn(2), ea_pf_mod_fn(3)};
        for (const void* f : fns)
            if (attr_err == hipSuccess)
                attr_err = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, PF_LDS);
    });
    if (attr_err != hipSuccess) return -100 - (int)attr_err;
    Params Pc = P;
    hipLaunchKernelGGL(ea_pf_qslice, dim3((unsigned)((P.rows + 15) / 16)), dim3(256), 0, st, Pc);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return -100 - (int)e;
    if (P.nseg > 0 && P.pf_ntiles > 0 && !P.pf_kv_cached) {
        const dim3 grid((unsigned)(P.nseg * P.pf_ntiles));
        if (P.mods) hipLaunchKernelGGL(ea_pf_kvslice<true>, grid, dim3(256), 0, st, Pc);
        else hipLaunchKernelGGL(ea_pf_kvslice<false>, grid, dim3(256), 0, st, Pc);
        e = hipGetLastError();
        if (e != hipSuccess) return -100 - (int)e;
    }
    return 0;
}

int ea::ea_launch_kv_digits(const Params& P, hipStream_t st) {
    if (P.nseg <= 0 || P.kvd_span <= 0) return 0;
    Params Pc = P;
    hipLaunchKernelGGL(ea_pf_kvslice<false>, dim3((unsigned)(P.nseg * P.kvd_span)), dim3(256), 0, st, Pc);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : -100 - (int)e;
}

int ea::ea_launch_prefill_main(const Params& P, hipStream_t st) {
    Params Pc = P;
    if (P.nseg > 0 && P.pf_nrb > 0) {
        const int items = P.nseg * P.pf_nrb * P.pf_nsplit;
        const dim3 grid((unsigned)items);
        if (P.mods) {
            // a block fills a CU's LDS: as many blocks as CUs, a multiple of the 8 XCDs, take all items
            static std::atomic<int> cus[64];
            int dev = 0;
            hipError_t e = hipGetDevice(&dev);
            if (e != hipSuccess) return -100 - (int)e;
            if (dev < 0 || dev >= 64) return -1;
            int n = cus[dev].load();
            if (!n) {
                if ((e = hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev)) != hipSuccess)
                    return -100 - (int)e;
                cus[dev].store(n);
            }
            void* args[] = {(void*)&Pc};
            e = hipLaunchKernel(ea_pf_mod_fn(P.mods), dim3((unsigned)std::min(items, std::max(n & ~7, 8))), dim3(512), args, PF_LDS, st);
            if (e != hipSuccess) return -100 - (int)e;
        } else if (P.pf_waves != 4) {
            if (P.timers) hipLaunchKernelGGL((ea_pf_main<8, true>), grid, dim3(512), PF_LDS, st, Pc);
            else hipLaunchKernelGGL((ea_pf_main<8, false>), grid, dim3(512), PF_LDS, st, Pc);
        } else {
            if (P.timers) hipLaunchKernelGGL((ea_pf_main<4, true>), grid, dim3(256), PF_LDS, st, Pc);
            else hipLaunchKernelGGL((ea_pf_main<4, false>), grid, dim3(256), PF_LDS, st, Pc);
        }
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return -100 - (int)e;
    }
    return 0;
}

int ea::ea_launch_prefill_combine(const Params& P, hipStream_t st) {
    if (P.pf_nsplit <= 1 || P.rows == 0) return 0;
    Params Pc = P;
    hipLaunchKernelGGL(ea_pf_combine, dim3((unsigned)P.rows), dim3(128), 0, st, Pc);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? 0 : -100 - (int)e;
}

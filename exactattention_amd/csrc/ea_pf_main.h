// The main kernel of the int8 prefill path (ea_prefill.hip): a header, because its variants with score
// modifications are compiled by themselves (ea_prefill_mod.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "ea_params.h"
#include "ea_pf_common.h"

using namespace ea;
using namespace ea::pf;

// The next digit, of weight 256^-1, of 16 q elements: the signed byte nearest 256 (q 2^-lsb - X). planes: the
// elements' bytes of digit plane 0; the first `have` of them exist, the others are zeros.
static __device__ __forceinline__ uint4 rest_digits(const uint16_t* q, const uint8_t* planes, int lsb, int have) {
    uint64_t lo = 0, hi = 0;
#pragma unroll 1
    for (int k = 0; k < min(have, 16); ++k) {
        int X = 0;
        for (int sp = 3; sp >= 0; --sp) X = X * 256 + (int)(int8_t)planes[128 * sp + k];
        const double r = ldexp((double)__uint_as_float((uint32_t)q[k] << 16), -lsb) - (double)X;
        const uint64_t d = (uint64_t)(min((int)rint(r * 256.0), 127) & 0xFF) << (8 * (k & 7));
        if (k < 8) lo |= d;
        else hi |= d;
    }
    return make_uint4((uint32_t)lo, (uint32_t)(lo >> 32), (uint32_t)hi, (uint32_t)(hi >> 32));
}

// ------------------------------------------------------------------------------------------------
// Main kernel. Block = NWB waves over 32 consecutive rows (tokens x query heads of one KV head):
// two row groups rg of 16 rows, SPLIT = NWB / 2 waves each. Wave hh of a row group takes the
// scores and weights of key groups kt = NKT hh .. NKT hh + NKT - 1 of each 64-key tile and the
// P.V sums of channel tiles ct = NCT hh .. NCT hh + NCT - 1 (NWB = 8: one key group and two
// channel tiles per wave; NWB = 4: two and four). Lane (g = lane / 16, j = lane % 16):
//   score layout  row j, keys 16 kt + 4 g + i (i = 0..3)
//   P.V layout    rows 4 g + i, channels 16 ct + j
// Software pipeline, one step per tile it, two barriers:
//   B1    K(it), its metadata and V(it-1) landed; the row maxima of tile it-1 are in sX
//         score MFMAs of tile it (K planes and q digits from LDS); while they run, the base move
//         (epoch fold when a base moves) and the weight digits of tile it-1 to sWD
//   B2    every wave has read the K planes of tile it and written its digits: row group 0's
//         waves issue the DMAs of K(it+1) with its metadata and of V(it) while row group 1's go
//         on; fp64 scores; P.V MFMAs of tile it-1 (digits from sWD), certification of tile it,
//         cold path; row maxima of tile it to sX
// V and the metadata are double-buffered (the two parities are two copies of the step). The DMAs
// are issued as inline asm, so the compiler adds no waits of its own; barriers are s_barrier after
// lgkmcnt(0) (no vmcnt(0): DMAs stay in flight across them) and the DMA waits are vmcnt(NKI)
// before B1 (K(it) and its metadata) and vmcnt(0) before B2 (V(it-1)).
// ------------------------------------------------------------------------------------------------
struct PfX {
    int32_t a, b;
    double c;
};

// LDS layout (dynamic): the DMA targets first, all below 104 KB
constexpr int PF_OFF_K = 0;
constexpr int PF_OFF_V0 = 32768;
constexpr int PF_OFF_V1 = 65536;
constexpr int PF_OFF_M0 = 98304;
constexpr int PF_OFF_M1 = PF_OFF_M0 + 4096;
constexpr int PF_QROW = 656;                 // q digit row stride in LDS: 640 bytes + 16 of padding
constexpr int PF_OFF_Q = PF_OFF_M1 + 4096;  // 32 rows x PF_QROW bytes
constexpr int PF_OFF_T = PF_OFF_Q + 32 * PF_QROW;
constexpr int PF_OFF_WD = PF_OFF_T + 4096;  // 5 planes x 4 key groups x 2 row groups x 64 lanes x 4 B
constexpr int PF_OFF_X = PF_OFF_WD + 10240;  // up to 8 waves x 64 lanes x 16 bytes
constexpr int PF_OFF_KEND = PF_OFF_X + 8192;
constexpr int PF_LDS = PF_OFF_KEND + 16;

// MOD: a row's base leaves its largest weight at 2^23 to 2^24 times 2^PF_MOD_TOP0 of 2^38, with room for
// larger ones to come; one that has to move shows scores of a wide spread, whose many small weights lose
// bits below the base, and leaves it at PF_MOD_TOP. fp32 outputs need every bit there is: PF_MOD_TOP32.
constexpr int PF_MOD_TOP0 = 11, PF_MOD_TOP = 13, PF_MOD_TOP32 = 14;

template <int N>
struct PfPar {
    static constexpr int value = N;
};

// MOD: with score modifications (ea_mod.h): 1 key ranges alone, 2 with a bias, 3 with a cap; a block's tiles then start at
// its rows' first visible key, and its last key split takes every tile past the others.
template <int NWB, bool TIMERS, int MOD = 0>
__global__ void __launch_bounds__(64 * NWB, 1) ea_pf_main(Params A) {
    const Params& P = A;
    // phase clocks (TIMERS build): shader cycles summed over waves into P.timers[i]. Per tile:
    // [14] DMA wait before B1, [0] B1, [1] EV reads and score MFMAs, [2] base move and weight
    // digits, [3] B2, DMA issue, fp64 scores and digit reads, [4] pair metadata, P.V and
    // certification, [5] cold path, [6] pair exchange, [7] the rest. Per block: [15] prologue,
    // [9] drain, [10] row totals, [11] earlier epochs and reciprocals, [12] normal-range rounding
    // of every entry, [13] the general test for the rest. [8] counts tiles (lane 0 of each wave).
    uint64_t tclk[16] = {0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0, 0};
    uint64_t tprev = TIMERS ? __builtin_amdgcn_s_memtime() : 0;
    auto tick = [&](int ph) __attribute__((always_inline)) {
        if (TIMERS) {
            const uint64_t t = __builtin_amdgcn_s_memtime();
            tclk[ph] += t - tprev;
            tprev = t;
        }
    };
    // the clocks into P.timers, once per wave (slot 8 counts the wave's tiles)
    auto flush_timers = [&](int ntile) __attribute__((always_inline)) {
        if (TIMERS && (threadIdx.x & 63) == 0) {
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (i != 8) atomicAdd((unsigned long long*)&P.timers[i], (unsigned long long)tclk[i]);
            atomicAdd((unsigned long long*)&P.timers[8], (unsigned long long)ntile);
        }
    };
    constexpr int SPLIT = NWB / 2;         // waves per row group of 16 rows
    constexpr int RPB = 16 * NWB / SPLIT;  // rows per block (32)
    constexpr int NKT = 4 / SPLIT;         // key groups of 16 per wave
    constexpr int NCT = 8 / SPLIT;         // channel tiles of 16 per wave
    constexpr int NKI = 64 / NWB;          // K (and V) DMA instructions per issuing wave and tile
    extern __shared__ __align__(16) unsigned char smem[];
    uint8_t* const sK = smem + PF_OFF_K;     // K planes of the current tile
    uint8_t* const sV0 = smem + PF_OFF_V0;   // V planes, even tiles
    uint8_t* const sV1 = smem + PF_OFF_V1;   // V planes, odd tiles
    uint8_t* const sM0 = smem + PF_OFF_M0;   // tile metadata, even tiles
    uint8_t* const sM1 = smem + PF_OFF_M1;   // tile metadata, odd tiles
    uint8_t* const sQ = smem + PF_OFF_Q;     // q digits of the block's rows
    double* const sT1 = (double*)(smem + PF_OFF_T);  // T1 * 2^23, then T2
    double* const sT2 = sT1 + 256;
    uint32_t* const sWD = (uint32_t*)(smem + PF_OFF_WD);  // weight digits [wave][plane 5][2][lane]
    PfX* const sX = (PfX*)(smem + PF_OFF_X);              // pair exchange [wave][lane]
    int& s_kend = *(int*)(smem + PF_OFF_KEND);
    int& s_kbeg = *(int*)(smem + PF_OFF_KEND + 4);
    int& s_next = *(int*)(smem + PF_OFF_KEND + 8);
    // Items: a segment's row block and key split, the longest first. With modifications, where the items are more
    // than the blocks, which then fill the device, a block takes another one of its XCD (item % 8) when it is
    // done: the 4 us between one block's end and the next one's first load are saved (documents of 4096 tokens,
    // 2048 items of some 39 us: 392 -> 377 us a step). The plain kernel spills in such a loop (4096 causal rows
    // 908 -> 976 us), or, compiled as those variants are, loses as much in the tile loop (940).
    for (uint32_t item = blockIdx.x;;) {
    int taken = INT_MAX / 16;  // of the items past the grid's, the one the block has next
    {
    // MOD: what follows from the arguments or the thread is made anew for each item, not kept over its loop
    typedef const __attribute__((address_space(4))) Params* kernarg_t;
    kernarg_t args = (kernarg_t)__builtin_amdgcn_kernarg_segment_ptr();
    int tid = threadIdx.x;
    if constexpr (MOD) {
        asm volatile("" : "+s"(args));
        asm volatile("" : "+v"(tid));
    }
    const Params& P = MOD ? *(const Params*)args : A;
    const int nseg = P.nseg;
    const int lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rg = w / SPLIT, hh = w % SPLIT;
    const int g = lane >> 4, j = lane & 15;
    const int seg = item % nseg;
    const int split = (int)(item / nseg) % P.pf_nsplit;  // key split (tile range)
    const int rbk = P.pf_nrb - 1 - (int)(item / nseg) / P.pf_nsplit;
    const int Hkv = P.g.num_kv_heads;
    const int64_t b = seg / Hkv;
    const int hk = seg % Hkv;
    // the segment's K/V tiles: its own in the workspace, or its slot's in the caller's cache
    const int64_t kseg = (P.pf_kv_cached && P.pf_kv_slot) ? (int64_t)P.pf_kv_slot[b] * Hkv + hk : (int64_t)seg;
    const int T = P.g.num_tokens;
    constexpr int WDS = 5 * NKT * 64;  // digit dwords per wave: [plane 5][NKT][lane 64]
    uint32_t* const wd_w = sWD + w * WDS + lane;                    // this wave's digit planes
    const uint32_t* const wd_r = sWD + (rg * SPLIT) * WDS + lane;  // the row group's, by key group
    // per-lane scratch: fp64 sums of completed epochs, then the final quotients
    double* const scr = P.pfscr + (((int64_t)blockIdx.x * NWB + w) * 64 + lane) * (8 * NCT);

    if (tid == 0) {
        s_kend = 0;
        if constexpr (MOD) s_kbeg = INT_MAX;
    }
    if ((!MOD || item == blockIdx.x) && tid < 256) {
        sT1[tid] = u64_as_f64(EA_T1_BITS[tid]) * 8388608.0;  // 2^23: exact
        sT2[tid] = u64_as_f64(EA_T2_BITS[tid]);
    }
    // step 0 runs the P.V of "tile -1" on zero weight digits and adds the zero EV of sM1
    for (int c = tid; c < NWB * WDS; c += 64 * NWB) sWD[c] = 0u;
    if (tid < 128) ((PfTileMeta*)sM1)->EV[tid] = 0.0;
    // ---- this lane's row in the score layout
    const int lr = rbk * RPB + rg * 16 + j;
    const bool rvalid = lr < P.r_seg;
    const int lrc = rvalid ? lr : P.r_seg - 1;
    int tq;
    const int64_t grow = seg_row(P, b, hk, lrc, &tq);
    const int64_t tok = b * T + tq;
    const int kvl = rvalid ? P.kv_len[tok] : 0;
    const uint64_t tmk = (rvalid && P.tree_mask) ? P.tree_mask[tok] : 0ull;
    const int tbase = P.tree_mask ? P.tree_base[b] : 0;
    const int slen = P.seq_len[b];
    int ve = kvl;
    if (tmk) ve = max(ve, tbase + 64 - (int)__clzll(tmk));
    ve = min(ve, slen);
    // keys below kvmin are visible to every row of the wave (and of its partner)
    const int kvmin = wave_min_i(rvalid ? min(kvl, slen) : INT_MAX);
    int kvb = 0, mpos = 0, kbmax = 0;
    float mslope = 0.0f;
    int vb = INT_MAX;
    if constexpr (MOD) {
        kvb = vis_begin(P, tok, kvl);
        mpos = mod_pos(P, tok, kvl);
        mslope = mod_slope(P, hk * P.grp + lrc % P.grp);
        kbmax = wave_max_i(rvalid ? kvb : 0);
        const KeySpan ks = key_span(kvb, kvl, slen, tmk, tbase);
        vb = ks.beg;
        ve = ks.end;
    }
    __syncthreads();  // s_kend initialised
    {
        const int kw = wave_max_i(ve);
        if (lane == 0) atomicMax(&s_kend, kw);
        if constexpr (MOD) {
            const int kb0 = wave_min_i(vb);
            if (lane == 0) atomicMin(&s_kbeg, kb0);
        }
    }
    // q digits of the block's rows into LDS: [row][plane 5][128 bytes] with rows PF_QROW = 656
    // bytes apart, so the 16 rows a 16-lane group reads start 4 banks apart (164 dwords = 36 mod 64)
    // and a 16-byte read per lane touches every bank once; rows past the segment repeat its last row.
    // The last plane is read for rows with elements rounded at slicing alone (score_rest)
    for (int c = tid; c < RPB * 32; c += 64 * NWB) {
        const int r = c >> 5, q16 = c & 31;
        const int lrr = min(rbk * RPB + r, P.r_seg - 1);
        int tt;
        const int64_t gr = seg_row(P, b, hk, lrr, &tt);
        *(uint4*)(sQ + r * PF_QROW + q16 * 16) = *(const uint4*)(P.pfq + gr * 512 + q16 * 16);
        if (q16 < 8) {
            uint4 rest = make_uint4(0, 0, 0, 0);
            const PfQMeta& m = ((const PfQMeta*)P.pfqm)[gr];
            if ((m.flags >> 8) & 0xFF)
                rest = rest_digits(P.q + b * P.g.q_seq_stride + (int64_t)tt * P.g.q_tok_stride +
                                       (int64_t)(hk * P.grp + lrr % P.grp) * P.g.q_head_stride + 16 * q16,
                                   P.pfq + gr * 512 + 16 * q16, m.lsb, P.g.head_dim - 16 * q16);
            *(uint4*)(sQ + r * PF_QROW + 512 + q16 * 16) = rest;
        }
    }
    // this lane's q digits (B operand of the score MFMA): row j, dims 64 h + 16 g .. + 15, plane s:
    // chunk 8 s + 4 h + g of the row
    const uint8_t* const qlds = sQ + (rg * 16 + j) * PF_QROW;
    const uint8_t* const qb[2] = {qlds + (g << 4), qlds + ((4 + g) << 4)};
    // K operand: key 16 kt + j, chunk (4 h + g) ^ (j & 7), plane t at + 8192 t, key group at + 2048 kt
    const uint8_t* const kb[2] = {sK + j * 128 + ((g ^ (j & 7)) << 4), sK + j * 128 + (((4 + g) ^ (j & 7)) << 4)};
    const PfQMeta qm = ((const PfQMeta*)P.pfqm)[grow];
    const bool needq = __ballot(rvalid && (qm.flags & 1)) != 0;
    // the score bound per pair is adq * kA 2^lk: |a| times the fold error factor 6.01 u times
    // sum_i A_q,i, with 2^-48 of slack for the roundings of this product and of adq * kAs
    const double adq = fabs(qm.a) * (6.01 * 0x1p-53) * qm.qA * (1.0 + 0x1p-48);
    // Elements of q rounded at slicing: each is within half a unit of 2^lsbq, and with its next digit, which
    // such rows' scores take in (score_rest), within 1/256, times a K element of at most kX; K's lowest digit,
    // which that product leaves out, is below 64 units, 2^-23 kX. With half a unit 6% of such a row's pairs
    // (normal values: one row of 128 dims in some 5000) took the cold path one after another, and its block
    // 4 times the others' time: 10000 rows of up to 2500 keys 505 us, 175 with the digit.
    const double aqL = fabs(qm.a) * 0x1.01p-8 * (double)((qm.flags >> 8) & 0xFF);
    const double aqX = fabs(qm.a) * 0.5 * (qm.qX + 1.0);
    const bool lossy_q = __ballot(rvalid && ((qm.flags >> 8) & 0xFF)) != 0;
    const bool qbad = (qm.flags & 2) != 0;
    int dom = (rvalid && qbad) ? 1 : 0;  // NaN/inf in q: a domain error (docs/SPEC.md)
    int unc = 0;
    int nslow = 0, nunc_s = 0, nunc_w = 0;
    // wave-uniform event counts, added to the stats once at the end: an atomic inside the tile loop
    // would make the next wait for vector memory (vmcnt) also wait for its round trip
    int nfold = 0, ncold = 0;
    __syncthreads();  // s_kend final, tables and q digits visible
    const int kend = s_kend;
    const int ntiles = (kend + 63) >> 6;
    // this block's key split: tiles [t0, t1) of the rows' visible range
    int t0 = min(split * P.pf_tps, ntiles), t1 = min(t0 + P.pf_tps, ntiles);
    if constexpr (MOD) {
        const int tb0 = min(s_kbeg >> 6, ntiles);
        t0 = min(tb0 + split * P.pf_tps, ntiles);
        t1 = split == P.pf_nsplit - 1 ? ntiles : min(t0 + P.pf_tps, ntiles);
    }
    const int nt = t1 - t0;
    const double* const T1s = sT1;
    const double* const T2 = sT2;

    // tile DMA: only the SPLIT waves of row group 0 issue, each NKI instructions of 1 KB for the K
    // (or V) planes and its share of the 4 KB of metadata. A wave stalls at a DMA instruction until
    // the texture path accepts it (about 2,000 cycles for a tile's 68 instructions); with one
    // issuing wave per SIMD the other wave on that SIMD, of row group 1, runs its P.V and
    // certification meanwhile instead of stalling beside it. Issued through pf_dma (inline asm),
    // so the compiler inserts no waits of its own before the LDS reads: every read of a DMA'd
    // buffer follows an explicit vmcnt wait for that buffer (row group 1 has nothing in flight).
    auto rsrc = [&](int tile) __attribute__((always_inline)) {
        const uint64_t src = (uint64_t)(P.pfkv + (kseg * P.pf_ntiles + tile) * EA_PF_TILE_BYTES);
        v4i r = {(int)(uint32_t)src, (int)((uint32_t)(src >> 32) & 0xFFFFu), EA_PF_TILE_BYTES, 0x00020000};
        r.x = __builtin_amdgcn_readfirstlane(r.x);
        r.y = __builtin_amdgcn_readfirstlane(r.y);
        return r;
    };
    const int vlane = lane * 16;  // one lane offset; the per-instruction offset goes in soffset
    const uint32_t aK = lds_addr(sK), aV0 = lds_addr(sV0), aV1 = lds_addr(sV1), aM0 = lds_addr(sM0),
                   aM1 = lds_addr(sM1);
    auto issue_k = [&](int tile, uint32_t mdst) __attribute__((always_inline)) {
        if (rg != 0) return;
        const v4i rs = rsrc(tile);
#pragma unroll
        for (int q = 0; q < NKI; ++q) {
            const int off = (q * SPLIT + hh) * 1024;
            pf_dma(rs, aK + off, vlane, off);
        }
#pragma unroll
        for (int m = hh; m < 4; m += SPLIT) pf_dma(rs, mdst + m * 1024, vlane, EA_PF_META_OFF + m * 1024);
    };
    auto issue_v = [&](int tile, uint32_t vdst) __attribute__((always_inline)) {
        if (rg != 0) return;
        const v4i rs = rsrc(tile);
#pragma unroll
        for (int q = 0; q < NKI; ++q) {
            const int off = (q * SPLIT + hh) * 1024;
            pf_dma(rs, vdst + off, vlane, 32768 + off);
        }
    };

    // per-row state (score layout; the 4 lanes of a row, and both waves of the pair, hold the
    // same base)
    int base = INT_MIN;
    double z = 0.0;  // this wave's keys
    int nv = 0;
    int nfrac = 0;   // this wave's keys of the current epoch whose scaled weight may have a fraction
    // MOD: instead of their number, the sum of what rounding the scaled weights moved them by in the epoch. Of
    // large scores most weights lie far below the base, where that is the weight and not a half
    float dsum = 0.0f;
    // The row's sum over its 4 lanes, times |X| < 2^30 of a key's V row: two additions here, SPLIT before and
    // the up to 1024 of each lane lose less than 2^-10 of it
    auto frac_total = [&](float pair) __attribute__((always_inline)) {
        pair += __shfl_xor(pair, 16, 64);
        return (pair + __shfl_xor(pair, 32, 64)) * (0x1p30f * (1.0f + 0x1p-10f));
    };
    // P.V state (P.V layout): int32 accumulators of digit weights 256^1 .. 256^7, 4 channel tiles
    v4i pacc[NCT][7];
#pragma unroll
    for (int cc = 0; cc < NCT; ++cc)
#pragma unroll
        for (int k = 0; k < 7; ++k) pacc[cc][k] = (v4i){0, 0, 0, 0};
    double EVs[NCT];  // per channel: inexact V elements of the epoch's tiles, times (2^38 + 1) / 2
#pragma unroll
    for (int cc = 0; cc < NCT; ++cc) EVs[cc] = 0.0;
    int ep_tiles = 0;
    bool had_fold = false;  // scr holds the sums of earlier epochs
    // MOD: the bound of what earlier epochs left out, per row (score layout), and the tiles since the base
    // last moved for the accumulators' sake
    float err = 0.0f;
    int since = 0;
    uint32_t failbits = 0;

    // fp64 value of the int32 P.V accumulators of (channel tile cc, row 4 g + i) in units 2^base,
    // and the bound of everything the epoch left out: fold roundings (6.02 u sum |acc|), inexact V
    // elements (EVs), the omitted digit pair (0, 0) (2^20 per tile), weight roundings below the
    // base (fr_i = 2^29 per key: 2^30 / 2)
    auto epoch_sum = [&](int cc, int i, double fr_i, double omit, double* en) __attribute__((always_inline)) {
        double h = (double)pacc[cc][6][i], ha = fabs(h);
#pragma unroll
        for (int k = 5; k >= 0; --k) {
            const double a = (double)pacc[cc][k][i];
            h = __fma_rn(h, 256.0, a);
            ha = __fma_rn(ha, 256.0, fabs(a));
        }
        *en = 6.02 * 0x1p-53 * (ha * 256.0) + EVs[cc] + omit + fr_i;
        return h * 256.0;
    };
    // ---- MOD: the epoch's sums back into the accumulators at the new bases nb. Modified scores move the
    // base often (large scores: 5 times a wave in 20 tiles), and a fold to memory costs 14,000 cycles
    // there, a round trip per entry. The sum, units 2^base 256, is cut into three parts 24 bits apart, the
    // slots 256^7, 256^4 and 256^1: |N| <= 2^74 per tile of 64 keys (weights to 2^38, |X| < 2^30), so the top
    // one stays below 2^30 for 4096 tiles, and with the 2^28 that 256 tiles add below 2^31. The rest is a
    // rounding of 2^7. What the epoch left out becomes one bound per row, the largest over the wave's channels.
    auto refold = [&](float ds_pair, int nb) __attribute__((always_inline)) {
        ++nfold;
        const float ft = frac_total(ds_pair);
        dsum = 0.0f;
        const double omit = (double)ep_tiles * 0x1p20;
        const int sh = base == INT_MIN ? 0 : max(base - nb, -1100);  // of the row in the score layout
        int er = 0;  // row j's bound as fp32 bits, in the score layout
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const double fr = (double)__shfl(ft, 4 * g + i, 64);
            const int dsh = __shfl(sh, 4 * g + i, 64);
            double e = 0.0;
#pragma unroll
            for (int cc = 0; cc < NCT; ++cc) {
                double en;
                const double nn = epoch_sum(cc, i, fr, omit, &en);
                e = fmax(e, en);
                double v = ldexp(nn, dsh - 8);
                const double A = rint(v * 0x1p-48);
                v = __fma_rn(-A, 0x1p48, v);
                const double B = rint(v * 0x1p-24);
                v = __fma_rn(-B, 0x1p24, v);
#pragma unroll
                for (int k = 0; k < 7; ++k) pacc[cc][k][i] = 0;
                pacc[cc][6][i] = (int)A;
                pacc[cc][3][i] = (int)B;
                pacc[cc][0][i] = (int)rint(v);
            }
            const float ef = (float)((ldexp(e, dsh) + 0x1p8) * (1.0 + 0x1p-20));
            const int em = row16_max(__float_as_int(ef));  // the 16 channels of row 4 g + i; bounds are positive
            const int mine = __shfl(em, 16 * (j >> 2), 64);
            er = (j & 3) == i ? mine : er;
        }
        err = (ldexpf(err, sh) + __int_as_float(er)) * (1.0f + 0x1p-20f);
#pragma unroll
        for (int cc = 0; cc < NCT; ++cc) EVs[cc] = 0.0;
        ep_tiles = 0;
    };
    // ---- fold the epoch into the per-lane fp64 sums in scr, rescaled to the new bases nb
    auto fold = [&](int nf_pair, int nb) __attribute__((always_inline)) {
        ++nfold;
        int nf = nf_pair + __shfl_xor(nf_pair, 16, 64);
        nf += __shfl_xor(nf, 32, 64);
        double fr[4];
        int bo[4], bn[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bo[i] = __shfl(base, 4 * g + i, 64);
            bn[i] = __shfl(nb, 4 * g + i, 64);
            fr[i] = 0x1p29 * (double)__shfl(nf, 4 * g + i, 64);
        }
        nfrac = 0;
        const double omit = (double)ep_tiles * 0x1p20;  // pair (0, 0): 64 keys x 2^14
#pragma unroll
        for (int cc = 0; cc < NCT; ++cc) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                double en;
                double nn = epoch_sum(cc, i, fr[i], omit, &en);
                double2* sp = (double2*)(scr + 2 * (4 * cc + i));
                if (had_fold) {
                    const double2 o = *sp;
                    nn += o.x;
                    en += o.y;
                }
                en += fabs(nn) * 0x1p-52;
                if (bo[i] != INT_MIN && bn[i] != bo[i]) {
                    const int dsh = max(bo[i] - bn[i], -1100);
                    nn = ldexp(nn, dsh);
                    en = ldexp(en, dsh) + 0x1p-1074;
                }
                *sp = make_double2(nn, en);
#pragma unroll
                for (int k = 0; k < 7; ++k) pacc[cc][k][i] = 0;
            }
        }
#pragma unroll
        for (int cc = 0; cc < NCT; ++cc) EVs[cc] = 0.0;
        ep_tiles = 0;
        had_fold = true;
        wait_vm<0>();  // the scr stores are complete (keeps the DMA counts exact)
    };

    // ---- P.V of the tile whose digits are in sWD and V planes in vbuf: pacc[cc][s + t - 1] +=
    // W digits s x V digits t (all pairs but (0, 0)). Channel 16 (NCT hh + cc) + j: the 16-byte
    // slot swizzle (ch >> 1) & 3 = (j >> 1) & 3 does not depend on cc, so every read is one lane
    // base plus a constant.
    auto pv_mfma = [&](const v4i (&Wd)[5], const uint8_t* vbuf, int c0, int c1) __attribute__((always_inline)) {
        const uint8_t* Vt = vbuf + (16 * NCT * hh + j) * 64 + ((g ^ ((j >> 1) & 3)) << 4);
#pragma unroll
        for (int cc = c0; cc < c1; ++cc) {
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const v4i B = *(const v4i*)(Vt + t * 8192 + cc * 1024);
#pragma unroll
                for (int s = 0; s < 5; ++s) {
                    if (s + t < 1) continue;
                    pacc[cc][s + t - 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(Wd[s], B, pacc[cc][s + t - 1], 0, 0, 0);
                }
            }
        }
    };
    auto read_wd = [&](v4i (&Wd)[5]) __attribute__((always_inline)) {
#pragma unroll
        for (int s = 0; s < 5; ++s)
#pragma unroll
            for (int kt = 0; kt < 4; ++kt) Wd[s][kt] = (int)wd_r[(kt / NKT) * WDS + (s * NKT + kt % NKT) * 64];
    };

    // ---- weights of the previous tile (certified in the previous step) and this wave's row maxima
    v4i cMk[NKT], cEk[NKT], cvl[NKT];
    int cgm = INT_MIN;
    // ---- after B1: the row group's maxima of the previous tile are in sX. Move the base (folding
    // the epoch first when it moves or is 256 tiles old), add the previous tile's inexact-V
    // counts, then write the previous tile's weight digits (A operand of the P.V MFMA) to sWD.
    auto rebase_digits = [&](const double (&evp)[NCT]) __attribute__((always_inline)) {
        int gm = cgm;
        int nf_pair = nfrac;  // the row group's keys (all SPLIT waves) of the epoch
        float ds_pair = dsum;
#pragma unroll
        for (int o = 1; o < SPLIT; ++o) {
            const PfX x = sX[(rg * SPLIT + (hh + o) % SPLIT) * 64 + lane];
            gm = max(gm, x.a);
            if constexpr (MOD) ds_pair += __int_as_float(x.b);
            else nf_pair += x.b;
        }
        // the base moves when a weight would exceed 2^38 (G - base > 14 for G = E + vlsb)
        const bool need_rb = gm != INT_MIN && (base == INT_MIN || gm > base + 14);
        int nb = need_rb ? gm - (!MOD ? 10 : (P.out_fp32 ? PF_MOD_TOP32 : (base == INT_MIN ? PF_MOD_TOP0 : PF_MOD_TOP))) : base;
        if constexpr (MOD) {
            if (++since > 4096 && base != INT_MIN) nb = max(nb, base + 8);
            if (ep_tiles > 0 && (__ballot(nb != base) != 0 || ep_tiles >= 256)) refold(ds_pair, nb);
            if (since > 4096) since = 0;
        } else {
            if (ep_tiles > 0 && (__ballot(need_rb) != 0 || ep_tiles >= 256)) fold(nf_pair, nb);
        }
#pragma unroll
        for (int cc = 0; cc < NCT; ++cc) EVs[cc] += evp[cc];
        if (nb != base && base != INT_MIN) z = ldexp(z, max(base - nb, -1100));
        base = nb;
    #pragma unroll
            for (int kk = 0; kk < NKT; ++kk) {
                uint32_t L[4], H[4];
    #pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int Mp = cMk[kk][i];
                    const int sc = cEk[kk][i] - base;
                    const double md = (double)Mp;
                    const double wsc = ldexp(md, sc + cvl[kk][i]);  // <= 2^38
                    z += ldexp(md, sc);                             // md = 0 for masked pairs
                    nv += Mp ? 1 : 0;
                    const double yw = wsc + PF_C40;
                    if constexpr (MOD) dsum += fabsf((float)(wsc - (yw - PF_C40)));
                    else nfrac += (Mp && sc + cvl[kk][i] < 0) ? 1 : 0;
                    const uint64_t yb = f64_as_u64(yw);
                    L[i] = (uint32_t)yb;
                    H[i] = (uint32_t)(yb >> 32);
                }
                const uint32_t a01 = __builtin_amdgcn_perm(L[1], L[0], 0x05010400u);
                const uint32_t b01 = __builtin_amdgcn_perm(L[1], L[0], 0x07030602u);
                const uint32_t a23 = __builtin_amdgcn_perm(L[3], L[2], 0x05010400u);
                const uint32_t b23 = __builtin_amdgcn_perm(L[3], L[2], 0x07030602u);
                const uint32_t e01 = __builtin_amdgcn_perm(H[1], H[0], 0x05010400u);
                const uint32_t e23 = __builtin_amdgcn_perm(H[3], H[2], 0x05010400u);
                uint32_t* wd = wd_w + kk * 64;
                wd[0 * 64 * NKT] = __builtin_amdgcn_perm(a23, a01, 0x05040100u) ^ 0x80808080u;
                wd[1 * 64 * NKT] = __builtin_amdgcn_perm(a23, a01, 0x07060302u) ^ 0x80808080u;
                wd[2 * 64 * NKT] = __builtin_amdgcn_perm(b23, b01, 0x05040100u) ^ 0x80808080u;
                wd[3 * 64 * NKT] = __builtin_amdgcn_perm(b23, b01, 0x07060302u) ^ 0x80808080u;
                wd[4 * 64 * NKT] = __builtin_amdgcn_perm(e23, e01, 0x05040100u) ^ 0x80808080u;
            }
    };

    // ---- one pipeline step, tile it (B1, score MFMAs beside the base move and digits of tile
    // it-1, B2, DMAs of K(it+1) and V(it), P.V of tile it-1, certification of tile it)
    auto step = [&](auto par, int it) __attribute__((always_inline)) {
        constexpr int PA = decltype(par)::value;
        const uint8_t* const sVp = PA ? sV0 : sV1;  // V(it - 1)
        const uint32_t aVc = PA ? aV1 : aV0;        // V(it) loads into the buffer V(it - 2) used
        const PfTileMeta* const TMc = (const PfTileMeta*)(PA ? sM1 : sM0);
        const PfTileMeta* const TMp = (const PfTileMeta*)(PA ? sM0 : sM1);
        const uint32_t aMn = PA ? aM0 : aM1;        // metadata of tile it + 1
        const bool k_next = it + 1 < t1;
        tick(7);
        // K(it) and its metadata landed. V(it - 1), issued after them, is first read after B2 and
        // is waited for there; at the first tile nothing else is in flight.
        if (it > t0) wait_vm<NKI>();
        else wait_vm<0>();
        tick(14);
        pf_bar();      // B1
        tick(0);
        const int tfl = TMc->tfl;
        // the previous tile's inexact-V counts, read before its metadata buffer is reloaded
        double evp[NCT];
#pragma unroll
        for (int cc = 0; cc < NCT; ++cc) evp[cc] = TMp->EV[16 * (NCT * hh + cc) + j];
        // ---- score MFMAs of tile it, then (while they run) the previous tile's base move and
        // weight digits
        v4i sacc[NKT][7];
#pragma unroll
        for (int kk = 0; kk < NKT; ++kk)
#pragma unroll
            for (int k = 0; k < 7; ++k) sacc[kk][k] = (v4i){0, 0, 0, 0};
        const bool wide = needq || ((tfl >> (NKT * hh)) & ((1 << NKT) - 1));
        auto scores = [&]() __attribute__((always_inline)) {
            if (lossy_q) {
#pragma unroll
                for (int kk = 0; kk < NKT; ++kk) score_rest(kb, qb, NKT * hh + kk, sacc[kk]);
            }
            if (wide) {
#pragma unroll
                for (int kk = 0; kk < NKT; ++kk) score_mfma<true>(kb, qb, NKT * hh + kk, sacc[kk]);
            } else {
#pragma unroll
                for (int kk = 0; kk < NKT; ++kk) score_mfma<false>(kb, qb, NKT * hh + kk, sacc[kk]);
            }
        };
        scores();
        tick(1);
        if (it > t0) rebase_digits(evp);
        tick(2);
        // every wave has read the K planes of tile it and written the weight digits of tile it - 1,
        // and V(it - 1) has landed: K(it + 1) with its metadata and V(it) start loading
        wait_vm<0>();
        pf_bar();
        if (k_next) issue_k(it + 1, aMn);
        issue_v(it, aVc);
        v4i lk4[NKT];
        double xs[NKT][4];
#pragma unroll
        for (int kk = 0; kk < NKT; ++kk) {
            lk4[kk] = *(const v4i*)&TMc->lsbk[16 * (NKT * hh + kk) + 4 * g];
            score_fold(sacc[kk], lk4[kk], xs[kk]);
        }
        v4i Wd[5];
        read_wd(Wd);  // zero at it = t0
        if (it > t0) ++ep_tiles;
        tick(3);
        // ---- per-pair metadata, score bounds and visibility of tile it
        v4i vl4[NKT];
        double adel[NKT][4];
#pragma unroll
        for (int kk = 0; kk < NKT; ++kk) {
            const int kt = NKT * hh + kk;
            vl4[kk] = *(const v4i*)&TMc->vlsb[16 * kt + 4 * g];
            const double2 kA01 = *(const double2*)&TMc->kA[16 * kt + 4 * g];
            const double2 kA23 = *(const double2*)&TMc->kA[16 * kt + 4 * g + 2];
            adel[kk][0] = adq * kA01.x;
            adel[kk][1] = adq * kA01.y;
            adel[kk][2] = adq * kA23.x;
            adel[kk][3] = adq * kA23.y;
        }
        if (lossy_q || (tfl & 32)) {
            // elements rounded at slicing: |k_i - K_i| <= 2^lsbk / 2, and q's as aqL has them
#pragma unroll
            for (int kk = 0; kk < NKT; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int key = 16 * (NKT * hh + kk) + 4 * g + i;
                    const double e = __fma_rn(aqL, TMc->kX[key] + 1.0, (double)(TMc->kfl[key] >> 8) * aqX);
                    adel[kk][i] = (adel[kk][i] + ldexp(e, lk4[kk][i])) * (1.0 + 0x1p-50);
                }
        }
        uint32_t vism = rvalid ? 0xFFu : 0u;  // bit 4 kk + i: pair visible
        if (!((it + 1) * 64 <= kvmin) || (MOD && it * 64 < kbmax)) {
            vism = 0;
#pragma unroll
            for (int kk = 0; kk < NKT; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = it * 64 + 16 * (NKT * hh + kk) + 4 * g + i;
                    const int ti = n - tbase;
                    const bool intree = ((unsigned)ti < 64u) & (((tmk >> (ti & 63)) & 1ull) != 0);
                    bool pre = n < kvl;
                    if constexpr (MOD) pre = pre & (n >= kvb);
                    vism |= ((n < slen) & (pre | intree)) ? (1u << (4 * kk + i)) : 0u;
                }
        }
        if (tfl & 16) {
            // NaN/inf in a key's K or V row: a domain error for the rows that see it
#pragma unroll
            for (int kk = 0; kk < NKT; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int bit = 1 << (4 * kk + i);
                    if (TMc->kfl[16 * (NKT * hh + kk) + 4 * g + i] & 1) {
                        if (vism & bit) dom = 1;
                        vism &= ~(uint32_t)bit;
                    }
                }
        }
        // ---- P.V of tile it - 1 (zero digits at it = t0) beside the certification of tile it
        v4i Mk[NKT], Ek[NKT];
        uint32_t slowmask = 0;  // pairs the fast path left undecided (cold path below)
        int gm = INT_MIN;
#pragma unroll
        for (int kk = 0; kk < NKT; ++kk) {
            pv_mfma(Wd, sVp, kk * (NCT / NKT), (kk + 1) * (NCT / NKT));
            int M[4], E[4];
            bool ok[4];
            if constexpr (MOD >= 2) {
                float m4[4];
                int dist[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    m4[i] = mslope;
                    dist[i] = it * 64 + 16 * (NKT * hh + kk) + 4 * g + i - mpos;
                }
                cert_pairs<4, MOD>(xs[kk], adel[kk], qm.a, T1s, T2, M, E, ok, P.cap, m4, dist);
            } else {
                cert_pairs<4>(xs[kk], adel[kk], qm.a, T1s, T2, M, E, ok);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const bool vis = (vism >> (4 * kk + i)) & 1;
                const bool good = vis & ok[i];
                slowmask |= (vis & !ok[i]) ? (1u << (4 * kk + i)) : 0u;
                Mk[kk][i] = good ? M[i] : 0;
                Ek[kk][i] = E[i];
                gm = max(gm, good ? E[i] + vl4[kk][i] : INT_MIN);
            }
        }
        tick(4);
        // ---- cold path: exact decision for the pairs the fast path left undecided. The exact
        // integer score comes from the tile's digit planes (no bf16 reads); only pairs whose
        // digits are inexact (elements rounded at slicing) read the bf16 inputs.
        if (__builtin_expect(__ballot(slowmask != 0) != 0, 0)) {
            ++ncold;
            const int8_t* Kg = (const int8_t*)(P.pfkv + (kseg * P.pf_ntiles + it) * EA_PF_TILE_BYTES);
            for (int p = 0; p < 4 * NKT; ++p) {
                if (!((slowmask >> p) & 1)) continue;
                const int kk = p >> 2, i = p & 3;
                const int key = 16 * (NKT * hh + kk) + 4 * g + i;
                const int n = it * 64 + key;
                const int kf = TMc->kfl[key];
                ++nslow;
                // the pair's exact decision, out of line: from the tile's digit planes when every
                // element was sliced exactly, else from the bf16 inputs
                const int mode = qbad ? 2 : ((!((qm.flags >> 8) & 0xFF) && !(kf >> 8)) ? 0 : 1);
                const uint16_t* qr = nullptr;
                const uint16_t* kr = nullptr;
                if (mode == 1) {
                    qr = P.q + b * P.g.q_seq_stride + (int64_t)tq * P.g.q_tok_stride +
                         (int64_t)(hk * P.grp + lrc % P.grp) * P.g.q_head_stride;
                    kr = P.k + kv_off(P, b, n, hk, 0);
                }
                const int3 cw = pf_cold_pair<(MOD >= 2)>(mode, qlds, 0, (const uint8_t*)Kg + key * 128, key & 7, qr, kr, P.am,
                                                  P.ae + qm.lsb + TMc->lsbk[key], P.alpha, T1s, T2, P.cap, mslope, n - mpos,
                                                  MOD ? P.g.head_dim : 128);
                const bool live = cw.x == 0;
                const int32_t M = cw.y, E = cw.z;
                if (cw.x == 2) dom = 1;
                if (cw.x == 3) {
                    unc = 1;
                    ++nunc_s;
                }
                if (cw.x == 4) {
                    unc = 1;
                    ++nunc_w;
                }
#pragma unroll
                for (int q = 0; q < NKT; ++q)
                    if (q == kk) {
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if (r == i) {
                                Mk[q][r] = live ? M : 0;
                                Ek[q][r] = E;
                            }
                    }
                if (live) gm = max(gm, E + TMc->vlsb[key]);
            }
        }
        tick(5);
        // ---- the row's largest weight in this tile (this wave's 4 lanes of the row), for the
        // row group's exchange after the next B1
        gm = max(gm, __shfl_xor(gm, 16, 64));
        gm = max(gm, __shfl_xor(gm, 32, 64));
        sX[w * 64 + lane] = PfX{gm, MOD ? __float_as_int(dsum) : nfrac, 0.0};
        cgm = gm;
#pragma unroll
        for (int kk = 0; kk < NKT; ++kk) {
            cMk[kk] = Mk[kk];
            cEk[kk] = Ek[kk];
            cvl[kk] = vl4[kk];
        }
        tick(6);
    };

    wait_vm<0>();  // the prologue's global loads: from here on vmcnt counts DMAs (and folds)
    if (nt > 0) issue_k(t0, aM0);
    tick(15);
    for (int it = t0; it < t1; it += 2) {
        step(PfPar<0>{}, it);
        if (it + 1 < t1) step(PfPar<1>{}, it + 1);
    }
    tick(7);
    // the block's next item, asked for while the last tile's sums and the rounding are ahead: at the start, a block
    // with a long item would take one that another is free for sooner (2375 tokens of documents, 298 items: 138
    // us a step so, 167 then, 146 on as many blocks as items)
    if (MOD && tid == 0 && nseg * P.pf_nrb * P.pf_nsplit > (int)gridDim.x)
        taken = atomicAdd(&P.wl_cnt[EA_PF_NEXT + (blockIdx.x & 7)], 1);
    // ---- drain: digits and P.V of the last tile
    if (nt > 0) {
        wait_vm<0>();
        pf_bar();
        const bool odd = (nt - 1) & 1;
        const PfTileMeta* TMl = (const PfTileMeta*)(odd ? sM1 : sM0);
        double evp[NCT];
#pragma unroll
        for (int cc = 0; cc < NCT; ++cc) evp[cc] = TMl->EV[16 * (NCT * hh + cc) + j];
        rebase_digits(evp);
        pf_bar();
        v4i Wd[5];
        read_wd(Wd);
        ++ep_tiles;
        pv_mfma(Wd, odd ? sV1 : sV0, 0, NCT);
    }
    tick(9);
    // ---- row totals for the final rounding: this wave's 4 lanes of the row, then the partner
    z += __shfl_xor(z, 16, 64);
    z += __shfl_xor(z, 32, 64);
    nv += __shfl_xor(nv, 16, 64);
    nv += __shfl_xor(nv, 32, 64);
    dom |= __shfl_xor(dom, 16, 64);
    dom |= __shfl_xor(dom, 32, 64);
    unc |= __shfl_xor(unc, 16, 64);
    unc |= __shfl_xor(unc, 32, 64);
    // MOD: the flags in the last bits of the sum, rounded up
    const int fdom = (__float_as_int(dsum) & ~3) + 4;
    sX[w * 64 + lane] = MOD ? PfX{nv, fdom | dom | (unc << 1), z} : PfX{nv, nfrac | (dom << 24) | (unc << 25), z};
    pf_bar();
    int nf_pair = nfrac;
    float ds_pair = __int_as_float(fdom);
    {
#pragma unroll
        for (int o = 1; o < SPLIT; ++o) {
            const PfX x = sX[(rg * SPLIT + (hh + o) % SPLIT) * 64 + lane];
            nv += x.a;
            if constexpr (MOD) {
                ds_pair += __int_as_float(x.b & ~3);
                dom |= x.b & 1;
                unc |= (x.b >> 1) & 1;
            } else {
                nf_pair += x.b & 0xFFFFFF;
                dom |= (x.b >> 24) & 1;
                unc |= (x.b >> 25) & 1;
            }
            z += x.c;
        }
    }
    tick(10);
    const float ft = MOD ? frac_total(ds_pair) : 0.0f;
    if (P.pf_nsplit > 1) {
        // ---- key splits: this split's (N, bound) per (row, channel) and (base, nv, flags, Z) per
        // row, in units 2^base; ea_pf_combine merges the splits and rounds. Every record a
        // combine reads is written here (a split with no tile writes nv = 0 and its flags).
        PfPart* const parts = (PfPart*)P.pf_part;
        double2* const ent = (double2*)(parts + (int64_t)P.pf_nsplit * P.rows);
        if (nt > 0) {
            int nf = nf_pair + __shfl_xor(nf_pair, 16, 64);
            nf += __shfl_xor(nf, 32, 64);
            const double omit = (double)ep_tiles * 0x1p20;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int lri = rbk * RPB + rg * 16 + 4 * g + i;
                if (lri >= P.r_seg) continue;
                int ti;
                const int64_t gr = seg_row(P, b, hk, lri, &ti);
                double fri = 0x1p29 * (double)__shfl(nf, 4 * g + i, 64);
                if constexpr (MOD) fri = (double)__shfl(ft, 4 * g + i, 64) + (double)__shfl(err, 4 * g + i, 64);
#pragma unroll
                for (int cc = 0; cc < NCT; ++cc) {
                    double en;
                    double nn = epoch_sum(cc, i, fri, omit, &en);
                    if (!MOD && had_fold) {
                        const double2 o = *(const double2*)(scr + 2 * (4 * cc + i));
                        nn += o.x;
                        en += o.y;
                    }
                    en += fabs(nn) * 0x1p-52;
                    ent[((int64_t)split * P.rows + gr) * 128 + 16 * (NCT * hh + cc) + j] = make_double2(nn, en);
                }
            }
        }
        if (g == 0 && hh == 0 && rvalid) {
            PfPart pr;
            pr.base = nv > 0 ? base : INT_MIN;
            pr.nv = nv;
            pr.fl = (dom ? 1 : 0) | (unc ? 2 : 0);
            pr.pad = 0;
            pr.z = z;
            pr.pad2 = 0.0;
            parts[(int64_t)split * P.rows + grow] = pr;
        }
        if (P.stats) {
            const int st5 = wave_sum_i(nunc_s), st6 = wave_sum_i(nunc_w), st8 = wave_sum_i(nslow);
            // rows are counted once, by the blocks of split 0
            const int cr = wave_sum_i((split == 0 && g == 0 && hh == 0 && rvalid) ? 1 : 0);
            if (lane == 0) {
                if (st5) atomicAdd((unsigned long long*)&P.stats[5], (unsigned long long)st5);
                if (st6) atomicAdd((unsigned long long*)&P.stats[6], (unsigned long long)st6);
                if (st8) atomicAdd((unsigned long long*)&P.stats[8], (unsigned long long)st8);
                if (nfold) atomicAdd((unsigned long long*)&P.stats[11], (unsigned long long)nfold);
                if (ncold) atomicAdd((unsigned long long*)&P.stats[12], (unsigned long long)ncold);
                if (cr) {
                    atomicAdd((unsigned long long*)&P.stats[0], (unsigned long long)cr);
                    atomicAdd((unsigned long long*)&P.stats[10], (unsigned long long)cr);
                }
            }
        }
        flush_timers(nt);  // loop phases, prologue, drain and row totals (no final rounding here)
        goto done;
    }
    // ---- the last epoch plus the earlier ones, then RN(N/Z) per (row, channel), certified:
    // q = N * RN(1/Z) (two roundings: below 2^-51.9 |q|, inside the 2^-51 |q| term) and
    // delta >= |N/Z - q| from the N bound en and the Z bound eZ
    if (nt > 0) {
        double2 prev[4 * NCT];
#pragma unroll
        for (int e = 0; e < 4 * NCT; ++e)
            prev[e] = !MOD && had_fold ? *(const double2*)(scr + 2 * e) : make_double2(0.0, 0.0);
        int nf = nf_pair + __shfl_xor(nf_pair, 16, 64);
        nf += __shfl_xor(nf, 32, 64);
        double fr[4], Zr[4], eZr[4], rz[4], rze[4];
        bool skip[4], live[4];  // skip: empty row, domain error or undecided pair (no output here)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            fr[i] = 0x1p29 * (double)__shfl(nf, 4 * g + i, 64);
            if constexpr (MOD) fr[i] = (double)__shfl(ft, 4 * g + i, 64) + (double)__shfl(err, 4 * g + i, 64);
            Zr[i] = __shfl(z, 4 * g + i, 64);
            const int nvr = __shfl(nv, 4 * g + i, 64);
            eZr[i] = (double)(nvr + 8) * PF_U * Zr[i] + (double)(nvr + 64) * 0x1p-1074;
            skip[i] = !(nvr > 0 && !__shfl(dom | unc, 4 * g + i, 64));
            const bool zok = Zr[i] > 2.0 * eZr[i] && isfinite(Zr[i]);
            rz[i] = zok ? 1.0 / Zr[i] : 0.0;
            rze[i] = zok ? 1.0 / (Zr[i] - eZr[i]) : 0.0;
            live[i] = !skip[i] && zok;
        }
        // output offsets of this lane's 4 rows (channel j of its first channel tile)
        int64_t orow[4];
        bool ovalid[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int lri = rbk * RPB + rg * 16 + 4 * g + i;
            ovalid[i] = lri < P.r_seg;
            const int lrv = ovalid[i] ? lri : 0;
            const int hq = hk * P.grp + lrv % P.grp;
            orow[i] = b * P.g.o_seq_stride + (int64_t)(lrv / P.grp) * P.g.o_tok_stride +
                      (int64_t)hq * P.g.o_head_stride + 16 * NCT * hh + j;
        }
        const int nch = MOD ? P.g.head_dim_v - 16 * NCT * hh - j : 128;  // channel 16 cc of this lane is there below it
        auto store_out = [&](int i, int cc, uint32_t bits) __attribute__((always_inline)) {
            if (P.out_fp32) ((uint32_t*)P.out)[orow[i] + 16 * cc] = bits;
            else ((uint16_t*)P.out)[orow[i] + 16 * cc] = (uint16_t)bits;
        };
        // every entry first tries the normal-range rounding (a few integer operations, no
        // branches); the entries it cannot decide go through LDS (the K and V buffers are idle:
        // no DMA is in flight) to one rolled loop of the general test
        double2* const qd = (double2*)smem + tid;  // entry e at qd[64 NWB e]
        uint32_t slow = 0;
        tick(11);
        const double omit = (double)ep_tiles * 0x1p20;
#pragma unroll
        for (int cc = 0; cc < NCT; ++cc) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                double en;
                const double nn = epoch_sum(cc, i, fr[i], omit, &en) + prev[4 * cc + i].x;
                en += prev[4 * cc + i].y;
                en += fabs(nn) * 0x1p-52;
                const double q = nn * rz[i];
                double delta = (en * (1.0 + 0x1p-40) + fabs(q) * eZr[i]) * rze[i] * (1.0 + 0x1p-40) +
                               fabs(q) * 0x1p-51 + 0x1p-1070;
                if (!isfinite(q) || !isfinite(delta) || !live[i]) delta = __builtin_inf();
                uint32_t bits = 0;
                const bool ok = !skip[i] && certify_round_normal(q, delta, P.out_fp32, &bits);
                const bool there = !MOD || 16 * cc < nch;
                if (ok && ovalid[i] && there) store_out(i, cc, bits);
                if (!skip[i] && !ok && there) {
                    slow |= 1u << (4 * cc + i);
                    qd[64 * NWB * (4 * cc + i)] = make_double2(q, delta);
                }
            }
        }
        tick(12);
        if (slow) {
#pragma unroll 1
            for (int e = 0; e < 4 * NCT; ++e) {
                if (!((slow >> e) & 1)) continue;
                const int cc = e >> 2, i = e & 3;
                const double2 v = qd[64 * NWB * e];
                uint32_t bits = 0;
                if (!certify_round_general(v.x, v.y, P.out_fp32, &bits)) {
                    failbits |= 1u << (8 * i + cc);
                    continue;
                }
                if (ovalid[i]) store_out(i, cc, bits);
            }
        }
    }
    tick(13);
    flush_timers(nt);
    if (P.stats) {
        const int st5 = wave_sum_i(nunc_s), st6 = wave_sum_i(nunc_w), st8 = wave_sum_i(nslow);
        if (lane == 0) {
            if (st5) atomicAdd((unsigned long long*)&P.stats[5], (unsigned long long)st5);
            if (st6) atomicAdd((unsigned long long*)&P.stats[6], (unsigned long long)st6);
            if (st8) atomicAdd((unsigned long long*)&P.stats[8], (unsigned long long)st8);
            if (nfold) atomicAdd((unsigned long long*)&P.stats[11], (unsigned long long)nfold);
            if (ncold) atomicAdd((unsigned long long*)&P.stats[12], (unsigned long long)ncold);
        }
    }
    if (nt == 0) {
        // no key visible to any row of the block: every row is empty (+0) or a q domain error
        nv = 0;
        unc = 0;
    }
    // ---- row flags: a row fails when any channel of either wave of the pair failed
    {
        uint32_t fb = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint64_t bal = __ballot(((failbits >> (8 * i)) & 0xFF) != 0);
            if (((bal >> (16 * g)) & 0xFFFFull) != 0) fb |= 1u << i;
        }
        pf_bar();  // sX reuse
        sX[w * 64 + lane].a = (int)fb;
        pf_bar();
#pragma unroll
        for (int o = 1; o < SPLIT; ++o) fb |= (uint32_t)sX[(rg * SPLIT + (hh + o) % SPLIT) * 64 + lane].a;
        failbits = fb;
    }
    int c_rows = 0, c_flag = 0, c_dom = 0, c_fin = 0;  // this lane's rows, added per wave below
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int di = __shfl(dom, 4 * g + i, 64), ui = __shfl(unc, 4 * g + i, 64), nvr = __shfl(nv, 4 * g + i, 64);
        const bool fin = !di && !ui && ((failbits >> i) & 1);  // a final rounding failed
        const int flag = di ? 2 : ((ui || fin) ? 1 : 0);
        const int lri = rbk * RPB + rg * 16 + 4 * g + i;
        if (lri >= P.r_seg) continue;
        if (flag || nvr == 0) {
            const int hq = hk * P.grp + lri % P.grp;
            const int64_t o = b * P.g.o_seq_stride + (int64_t)(lri / P.grp) * P.g.o_tok_stride +
                              (int64_t)hq * P.g.o_head_stride + 16 * NCT * hh + j;
#pragma unroll
            for (int cc = 0; cc < NCT; ++cc) {
                if (MOD && 16 * (NCT * hh + cc) + j >= P.g.head_dim_v) continue;
                if (P.out_fp32) ((uint32_t*)P.out)[o + 16 * cc] = 0u;
                else ((uint16_t*)P.out)[o + 16 * cc] = 0;
            }
        }
        if (j == 0 && hh == 0) {
            int ti;
            const int64_t gr = seg_row(P, b, hk, lri, &ti);
            P.flags[gr] = (uint8_t)flag;
            if (flag == 1) {
                const int slot = atomicAdd(P.wl_cnt, 1);
                P.wl[slot] = (int32_t)gr;
            }
            ++c_rows;
            c_flag += flag ? 1 : 0;
            c_dom += flag == 2 ? 1 : 0;
            c_fin += fin ? 1 : 0;
        }
    }
    // one atomic per counter and wave (same-address atomics per row would serialise)
    if (P.stats && hh == 0) {
        c_rows = wave_sum_i(c_rows);
        c_flag = wave_sum_i(c_flag);
        c_dom = wave_sum_i(c_dom);
        c_fin = wave_sum_i(c_fin);
        if (lane == 0) {
            if (c_rows) {
                atomicAdd((unsigned long long*)&P.stats[0], (unsigned long long)c_rows);
                atomicAdd((unsigned long long*)&P.stats[10], (unsigned long long)c_rows);
            }
            if (c_flag) atomicAdd((unsigned long long*)&P.stats[1], (unsigned long long)c_flag);
            if (c_dom) atomicAdd((unsigned long long*)&P.stats[4], (unsigned long long)c_dom);
            if (c_fin) atomicAdd((unsigned long long*)&P.stats[7], (unsigned long long)c_fin);
        }
    }
    }
done:
    if constexpr (!MOD) {
        return;
    } else {
        if (threadIdx.x == 0) s_next = (int)(blockIdx.x & 7) + 8 * ((int)gridDim.x / 8 + taken);
        __syncthreads();  // s_next written, and this item's LDS reads done
        item = __builtin_amdgcn_readfirstlane(s_next);
        if (item >= (uint32_t)(A.nseg * A.pf_nrb * A.pf_nsplit)) return;
    }
    }
}

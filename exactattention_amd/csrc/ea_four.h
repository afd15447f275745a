// Tier-1 split kernel for caches held in 4 bits (ea_kv4.h) on the low-precision matrix instructions (gfx950): certified sums, as
// the other split kernels', whose partials the same combine merges.
//
// What a 4-bit cache changes: a key's element is a 4-bit float under a power of two, which v_mfma_scale_f32_16x16x128_f8f6f4
// multiplies as it stands, scale included. The fp64 kernels convert every element and pay 16 MACs a cycle and SIMD; here a key's 128
// elements are one instruction of 16 cycles for 16 columns.
//
//   scores   q is cut once into 6 balanced digits of 5 bits, -16 .. 15, each a 6-bit float (3 of mantissa: the code of a
//            magnitude is the magnitude). A product of a digit and an element is a whole number of halves, at most 192; 128 of
//            them, and scales up to 2^9 apart, are below 2^24 units: the instruction's fp32 sum is exact, in any order. The 6 sums join
//            in fp64 exactly, 49 bits, so the score of a pair is exact, and the certified logit almost always decided. What elements
//            far below the row's top leave (one of a row's 128 is 2^-20 of the largest in some rows of every step) takes 6 digits
//            more, in blocks of rows that have any; what those leave is counted and bounded. Keys whose scales lie further apart are
//            left to the exact path.
//   weights  w = RN24(2^t) = M 2^E (cert_pairs), their exponents against a base per row
//   P.V      V's scale belongs to its key, a summand: it moves into the weight. For each group of 32 channels the weight
//            W = RN(M 2^(E + b - G - base)) <= 2^46 (b the scale's byte, G the group's largest) becomes 6 balanced digits of 8 bits,
//            read out of an fp64 sum with 2^52, and v_mfma_i32_16x16x64_i8 sums them over 64 keys with the elements as
//            whole numbers (-12 .. 12, byte lookups). int32 sums are exact; a base that must move folds them into fp64.
//            The rounding of W is the one error: half a unit of 2^(base + G) a key.
//
// What bounds it is the VALU, and HBM where a block has 2 rows: of a tile of 64 keys and 4 rows 55 instructions for the scores, 135 for the
// weights, 37 a group of 32 channels for their digits and 44 for V's bytes; 2 waves a SIMD (the int32 sums alone are 64 registers; 8 rows
// a wave took 96, spilled, and then waited for every load: a 1500-token chunk 770 us, 680 with 4). A step of 32 ragged sequences to
// 4096 keys, 32/8 heads: 59 us, 69 on the fp64 matrix instructions; 8 of 30000 to 131072, 16/8 heads: 172 (4.8 TB/s), 437; a chunk of
// 1500 tokens behind 2500, 16/8 heads: 579, 718.
//
// Layout. A block is 4 waves over one (segment, block of rows, key range). WR = 1: RS = 2 or 4 rows, wave w takes 64-key tiles w, w +
// 4, .. and meets the others in the epilogue only. WR = 4: 16 rows, a wave takes 4 of them and every tile. Lane l: g = l / 16, n = l % 16;
// its pairs are those of its row, with the keys 4 n + u (u = 0..3) of the tile: row g of the wave's, or of 2 rows row g / 2 and half of the
// keys.
//   q     digits in registers, the A operand (M = a row's digit, K = dim): with M = 4 g + i in the order of the rows, the 4 sums of
//         D that a lane gets are digits of its own row: 2 instructions a key of 4 rows, and nothing passes between lanes; 1 of 2
//         rows, whose lanes swap halves
//   K     lane loads dims 32 g .. + 31 of the keys 4 n + u (16 bytes and a scale each): the B operand (K = dim, N = key)
//   W     digits to LDS, [plane][row][64 keys]; A operand (M = plane and row, K = key): 4 rows: planes 0, 1 and 2..5
//   V     l = 0..3: lane loads channels 32 l + 2 n and + 1 of keys 16 g .. + 15 (16 bytes): two B operands (K = key, N = channel)
//   O     fp64 sums, in LDS: they change only where int32 sums are folded into them
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <type_traits>

#include "ea_kv4.h"
#include "ea_params.h"
#include "ea_pf_common.h"

using namespace ea;

namespace {

constexpr int F4_THREADS = 256;
constexpr int F4_NONE = -1200000000;  // base of a row without a visible key so far
constexpr int F4_BITS = 22;           // a weight's exponent E may exceed the base by this: M < 2^24 then gives 46 bits
constexpr int F4_HEAD = 2;            // room left when the base moves
constexpr int F4_SPREAD = 9;          // of a key's scales, for exact sums
constexpr int F4_LIST = 64;
constexpr int F4_EPOCH = 16384;       // tiles between folds at most: 2^14 x 64 keys x 128 x 12 < 2^31
constexpr int F4_WROW = 20;           // dwords a row of 64 digits takes (16 and 4 that spread the rows over the banks)
typedef int f4_i8 __attribute__((ext_vector_type(8)));
typedef int f4_i4 __attribute__((ext_vector_type(4)));
typedef float f4_f4 __attribute__((ext_vector_type(4)));
typedef uint32_t f4_u4 __attribute__((ext_vector_type(4)));
typedef uint32_t f4_u2 __attribute__((ext_vector_type(2)));
typedef unsigned short f4_h2 __attribute__((ext_vector_type(2)));

template <int RS, int NG, int WR>
struct FourSmem {
    static constexpr int RB = RS * WR;  // rows of the block
    uint32_t q6[2][RB * 6 * 24];  // q's digits [row][digit][32-dim block][6 dwords], and those of what they leave
    uint32_t zero[8];
    double T1[256], T2[256];  // exp2 tables, T1 times 2^23
    double rq[RB], rqe[RB];   // alpha 2^(lsb + 3); |alpha| times the sum of |q| that both rounds lost
    int bad[RB], more[RB], kvl[RB];
    uint64_t tmk[RB];
    int kvb[RB], pos[RB];  // with score modifications
    float slope[RB];
    double wZ[4][RS], we[4][RS];
    int wR[4][RS], wf[4][RS], wn[4];
    uint32_t wv[4][4];  // per wave and group: the reference, no key's scale is larger
    uint32_t list[4][F4_LIST + 64 * RS];
    double O[4][RS][32 * NG];  // per wave: of channel 32 l + 2 n + h at 32 l + 16 h + n
    union alignas(16) {
        uint32_t W[4][NG][6 * RS * F4_WROW];
        uint8_t dig[2][RB * 6 * 128];
    };
};

// x of the lane 16 (32) lanes away
__device__ __forceinline__ double xor16(double x) { return __shfl_xor(x, 16, 64); }
__device__ __forceinline__ double xor32(double x) { return __shfl_xor(x, 32, 64); }
__device__ __forceinline__ f4_h2 pk_max(f4_h2 a, f4_h2 b) { return __builtin_elementwise_max(a, b); }

// The bytes of 4 elements, whole numbers of halves, from the low (HI = false) or high halves of 4 bytes: 0, 1, 2, 3, 4, 6, 8, 12 and
// their negatives. A byte permutation looks up 8 entries; selectors 8 to 11 give the signs of the table's odd entries (0 or 0xFF), 12
// gives 0 and 13 to 15 0xFF. So P[x] ^ N[x ^ 8] has both halves of the code in one place, each table holding its entries XORed with what the
// other one gives there:
//   P[i] = v_i ^ b_i, b_0..3 the signs of N[1], N[3], N[5], N[7], b_4 = 0, b_5..7 = 0xFF; N[i] = -v_i ^ a_i, a from P's signs alike
//   P[5] = ~6 and P[7] = ~12 are negative, N[5] = ~-6 = 5 and N[7] = ~-12 = 11 positive: b_2 = b_3 = 0, so P[3] = 3, a_1 = 0 and
//   N[1] = -1: b_0 = 0xFF; a_3 = 0xFF makes N[3] = ~-3 = 2 positive: b_1 = 0 and P[1] = 1, a_0 = 0; a_2 = 0xFF
template <bool HI>
__device__ __forceinline__ uint32_t four_bytes(uint32_t w) {
    constexpr uint32_t M = 0x0F0F0F0Fu;
    constexpr uint32_t p[8] = {0, 1, 2, 3, 4, 6, 8, 12};
    constexpr auto neg = [](uint32_t x) { return (0u - x) & 0xFFu; };
    constexpr uint32_t P0 = (p[0] ^ 0xFFu) | p[1] << 8 | p[2] << 16 | p[3] << 24;
    constexpr uint32_t P1 = p[4] | (p[5] ^ 0xFFu) << 8 | (p[6] ^ 0xFFu) << 16 | (p[7] ^ 0xFFu) << 24;
    constexpr uint32_t N0 = neg(p[0]) | neg(p[1]) << 8 | (neg(p[2]) ^ 0xFFu) << 16 | (neg(p[3]) ^ 0xFFu) << 24;
    constexpr uint32_t N1 = neg(p[4]) | (neg(p[5]) ^ 0xFFu) << 8 | (neg(p[6]) ^ 0xFFu) << 16 | (neg(p[7]) ^ 0xFFu) << 24;
    const uint32_t s = HI ? w >> 4 : w;
    const uint32_t x = s & M, y = (s & M) ^ 0x08080808u;
    return __builtin_amdgcn_perm(P1, P0, x) ^ __builtin_amdgcn_perm(N1, N0, y);
}

// Certified weights of exact sums: w = RN24(2^t), t = RN32(x), x within |p| rel + adel of p = a xs: t is decided when both ends of
// that interval round to it. |t| <= 2^-25 gives 1. 2^t from the tables and the cubic of pf::cert_pairs, with its bound: t is cut at
// multiples of 2^-16 by an addition (of t - 2^-17, which is exact; a multiple may go down, and leaves r = 2^-16). w = Y 2^(fl - 23), Y in
// 2^23 .. 2^24; not ok: left to the exact path.
template <int NP>
__device__ __forceinline__ void four_weights(const double (&xs)[NP], double a, double rel, double adel, const double* T1s, const double* T2, double (&Y)[NP],
                                             int (&fl)[NP], bool (&ok)[NP]) {
    const double c1 = u64_as_f64(EA_C_BITS[0]), c2 = u64_as_f64(EA_C_BITS[1]), c3 = u64_as_f64(EA_C_BITS[2]);
    constexpr double CUT = 0x1.8p36;
    double r[NP], aa[NP];
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const double p = a * xs[i], e = __fma_rn(fabs(p), rel, adel);
        const float lo = (float)(p - e), hi = (float)(p + e);
        ok[i] = (lo == hi) & (fabsf(hi) < 0x1p29f);
        const double t = (double)(fabsf(hi) <= 0x1p-25f ? 0.0f : hi);
        const double X = (t - 0x1p-17) + CUT;
        r[i] = t - (X - CUT);
        const uint32_t k = (uint32_t)__double2loint(X);  // t in units of 2^-16, its low half the fraction
        fl[i] = (int)__builtin_amdgcn_alignbit((uint32_t)__double2hiint(X), k, 16);
        aa[i] = T1s[(k >> 8) & 255u] * T2[k & 255u];
    }
#pragma unroll
    for (int i = 0; i < NP; ++i) {
        const double y = __fma_rn(aa[i], r[i] * __fma_rn(r[i], __fma_rn(r[i], c3, c2), c1), aa[i]);
        Y[i] = (y + 0x1.8p52) - 0x1.8p52;
        ok[i] = ok[i] & (fabs(y - Y[i]) <= 0.5 - 0x1p-26);
    }
}

}  // namespace

// MOD: with score modifications (ea_mod.h): 1 key ranges alone, 2 with a bias, 3 with a cap; a unit's key range is then counted from its
// rows' first visible key, down to a whole tile, and on uniform splits the last split takes every key past the others.
template <int RS, int NG, int MOD, int WR>
__global__ void __launch_bounds__(F4_THREADS, 2) ea_four(Params P) {
    constexpr int KL = RS;               // keys of a lane
    constexpr int NMF = RS == 2 ? 1 : 2;  // matrix instructions for 6 digits of the rows
    constexpr int RB = RS * WR;           // rows of the block
    constexpr int STEP = WR == 1 ? 256 : 64;  // from a wave's tile to its next
    typedef FourSmem<RS, NG, WR> Smem;
    extern __shared__ __align__(16) unsigned char smem_raw[];
    Smem& S = *reinterpret_cast<Smem*>(smem_raw);
    const int tid = (int)threadIdx.x;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int d = P.g.head_dim, dv = P.g.head_dim_v;
    const int wid = kv4_width(dv), ng = NG == 2 ? wid >> 5 : NG;  // V's channels in whole groups: NG, or 1 with NG = 2

    S.T1[tid] = u64_as_f64(EA_T1_BITS[tid]) * 8388608.0;  // 2^23: exact
    S.T2[tid] = u64_as_f64(EA_T2_BITS[tid]);
    if (tid < 8) S.zero[tid] = 0;
    if (blockIdx.x == 0 && blockIdx.y == 0) {
        // on uniform splits the step's first kernel clears the tier-2 work list and chunk counts
        if (!P.dq_stream && tid < EA_T2_CNT) P.wl_cnt[tid] = 0;
        if (tid == 0 && P.stats) atomicAdd((unsigned long long*)&P.stats[9], (unsigned long long)P.rows);
        if (tid == 0 && P.stats_x) atomicAdd((unsigned long long*)&P.stats_x[0], (unsigned long long)P.rows);
    }

    // One piece: keys [kA, kB) of unit `item` (segment, row block), clipped to the unit's visible end, as partial slot `split`.
    auto piece = [&](const int item, const int split, int kA, int kB) __attribute__((always_inline)) {
        // what follows from the lane is found anew for every piece: kept over the pieces it spills, and a reload waits for the loads of
        // the first tile
        int lane = tid & 63;
        asm volatile("" : "+v"(lane));
        const int g = lane >> 4, n = lane & 15;
        const int seg = item / P.nrb, rbk = item % P.nrb;
        const int Hkv = P.g.num_kv_heads;
        const int b = seg / Hkv, hk = seg % Hkv;
        const int row0 = rbk * RB;
        const int nrow = min(RB, P.r_seg - row0);
        const int wrow = WR == 1 ? 0 : RS * w;  // the first of the wave's rows
        auto q_row = [&](int r) __attribute__((always_inline)) {
            const int lr = row0 + r, t = lr / P.grp, gi = lr % P.grp;
            return P.q + (int64_t)b * P.g.q_seq_stride + (int64_t)t * P.g.q_tok_stride + (int64_t)(hk * P.grp + gi) * P.g.q_head_stride;
        };
        // what the digits are cut from, requested before anything waits
        uint32_t qv[(RB + 3) / 4][2];
#pragma unroll
        for (int r4 = 0; r4 < RB; r4 += 4)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int i = 2 * lane + h;
                qv[r4 / 4][h] = r4 + w < nrow && i < d ? q_row(r4 + w)[i] : 0u;
            }
        // ---- the rows' visible keys: prefix and tree mask in LDS (tiles inside every prefix do not read them), the last
        // visible key and the shortest prefix of the block
        const int slen = P.seq_len[b];
        const int tb = P.tree_mask ? P.tree_base[b] : 0;
        int kend = 0, kvmin = INT_MAX;
        int kbeg = INT_MAX, kbmax = 0;  // MOD: the rows' first visible key, their last prefix start
        {
            const int r = lane & (RB - 1);
            const int tok = b * P.g.num_tokens + (row0 + min(r, nrow - 1)) / P.grp;
            const int kvl = P.kv_len[tok];
            const uint64_t tmk = P.tree_mask ? P.tree_mask[tok] : 0ull;
            kend = tmk ? max(kvl, tb + 64 - (int)__clzll(tmk)) : kvl;
            kvmin = kvl;
            if constexpr (MOD) {
                const int kvb = vis_begin(P, tok, kvl);
                kbmax = kvb;
                const KeySpan ks = key_span(kvb, kvl, slen, tmk, tb);
                kbeg = ks.beg;
                kend = ks.end;
                if (w == 0 && lane < RB) {
                    S.kvb[r] = kvb;
                    S.pos[r] = mod_pos(P, tok, kvl);
                    const int lr = row0 + min(r, nrow - 1);
                    S.slope[r] = mod_slope(P, hk * P.grp + lr % P.grp);
                }
            }
            if (w == 0 && lane < RB) {
                S.kvl[r] = r < nrow ? kvl : INT_MIN;
                S.tmk[r] = r < nrow ? tmk : 0ull;
            }
        }
        kend = min(wave_max_dpp(kend), slen);
        kvmin = min(-wave_max_dpp(-kvmin), slen);
        if constexpr (MOD) {
            kbeg = -wave_max_dpp(-kbeg);
            kbmax = wave_max_dpp(kbmax);
            const int k0 = kend > 0 ? tile_floor(kbeg) : 0;
            kA += k0;
            kB += k0;
        }
        const int k1 = min(kB, kend);
        const int k0w = WR == 1 ? kA + 64 * w : kA;  // this wave's tiles: k0w + STEP it
        const int nst = k1 > k0w && wrow < nrow ? (k1 - k0w + STEP - 1) / STEP : 0;
        const int row = RS == 2 ? g >> 1 : g;       // the lane's row
        const int sub = RS == 2 ? 2 * (g & 1) : 0;  // its keys of a tile: 4 n + sub + i
        constexpr int RLANES = RS == 2 ? 32 : 16;   // lanes of a row
        const bool head = n == 0 && sub == 0;       // the first of them
        // Loads of a tile stand under no branch: one that waits for older loads could not tell how many younger ones there are, and
        // would wait for all. So caches without pages look one up (and do not use it), and the last tile requests its last run again.
        cint_t* btb = P.bt ? (cint_t*)P.bt + (P.bt_off ? P.bt_off[b] : (int64_t)b * P.g.block_table_stride) : (cint_t*)P.seq_len;
        const int bmask = P.bt ? -1 : 0;
        const int pshift = P.pshift, pmask = (1 << pshift) - 1;
        // 16 consecutive keys from a multiple of 16 (a run) lie in one page (page size >= 16) and are one tile of V. Runs past the
        // last key (or, MOD, before the first) read the last one's again, as keys past the last one do within theirs, and weigh
        // nothing. Offsets count 32 elements: 16 bytes, or one scale.
        auto run_of = [&](int n0, int at) __attribute__((always_inline)) {
            int m = min(n0 + 16 * at, k1 - 1);
            if constexpr (MOD) m = max(m, kbeg);
            return m & ~15;
        };
        struct Pages {
            int k, v;
        };
        auto pages_of = [&](int n0) __attribute__((always_inline)) {
            const int pk = btb[(run_of(n0, n >> 2) >> pshift) & bmask], pv = btb[(run_of(n0, g) >> pshift) & bmask];
            return (Pages){P.bt ? pk : b, P.bt ? pv : b};
        };
        auto times = [](int x, int64_t stride) __attribute__((always_inline)) {  // x >= 0
            return (uint64_t)(uint32_t)x * (uint32_t)stride + ((uint64_t)((uint32_t)x * (uint32_t)(stride >> 32)) << 32);
        };
        struct KR {
            f4_u4 k[4];
            uint32_t s[4];
        };
        struct VR {
            f4_u4 v[NG];
            uint32_t s[NG];
        };
        const int64_t kps = P.g.k_page_stride >> 5, kss = P.g.k_slot_stride >> 5, vps = P.g.v_page_stride >> 5;
        const int gk = min(g, (d - 1) >> 5);  // blocks past the head: q's digits are zeros there
        const char* const kbase = (const char*)P.k + (((int64_t)hk * P.g.k_head_stride) >> 1) + 16 * gk;
        const uint8_t* const ksbase = P.ks + (((int64_t)hk * P.g.k_head_stride) >> 5) + gk;
        const char* const vbase = (const char*)P.v + (((int64_t)hk * P.g.v_head_stride) >> 1) + 16 * n;
        const uint8_t* const vsbase = P.vs + (((int64_t)hk * P.g.v_head_stride) >> 5) + 4 * (n & 3) + sub;
        auto issue_k = [&](int n0, const Pages& p, KR& x) __attribute__((always_inline)) {
            const int run = run_of(n0, n >> 2), lim = k1 - 1 - run;
            const uint64_t at = times(p.k, kps) + times(P.bt ? run & pmask : run, kss);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint64_t to = at + (uint64_t)((uint32_t)min(4 * (n & 3) + u, lim) * (uint32_t)kss);
                x.k[u] = *(const f4_u4*)(kbase + (to << 4));
                x.s[u] = ksbase[to];
            }
        };
        auto issue_v = [&](int n0, const Pages& p, VR& x) __attribute__((always_inline)) {
            const int rv = run_of(n0, g), rs = run_of(n0, n >> 2);
            const uint64_t at = times(p.v, vps) + times((P.bt ? rv & pmask : rv) >> 4, wid >> 1);
            const uint64_t as = times(p.k, vps) + times((P.bt ? rs & pmask : rs) >> 4, wid >> 1);
            const char* const vc = vbase + (at << 4);
            const uint8_t* const vs = vsbase + as;
#pragma unroll
            for (int l = 0; l < NG; ++l) {
                const int lx = min(l, ng - 1);
                x.v[l] = *(const f4_u4*)(vc + 256 * lx);
                x.s[l] = KL == 4 ? *(const uint32_t*)(vs + 16 * lx) : *(const uint16_t*)(vs + 16 * lx);
            }
        };

        // the first tile is requested before the digits are cut
        KR kr;
        VR vr;
        Pages nx = {0, 0};  // of the next tile
        auto begin = [&](int n0) __attribute__((always_inline)) {
            const Pages p = pages_of(n0);
            nx = pages_of(n0 + STEP);
            issue_k(n0, p, kr);
            issue_v(n0, p, vr);
        };
        if (nst > 0) begin(k0w);
        // ---- q's digits: X = q / 2^lsb, |X| < 2^28, in 6 digits of 5 bits
#pragma unroll
        for (int r4 = 0; r4 < RB; r4 += 4) {
            const int r = r4 + w;
            if (r >= RB) break;
            int m[2] = {0, 0}, e[2] = {0, 0}, bad = 0, lead = INT_MIN;
            if (r < nrow) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint32_t x = qv[r4 / 4][h];
                    const int f = (x >> 7) & 0xFF;
                    bad |= f == 0xFF;
                    m[h] = (int)(x & 0x7F) | (f ? 0x80 : 0);
                    e[h] = (f ? f : 1) - 134;
                    if (m[h]) lead = max(lead, e[h] + 31 - __clz(m[h]));
                    if (x & 0x8000) m[h] = -m[h];
                }
            }
            lead = wave_max_dpp(lead);
            bad = wave_max_dpp(bad);
            const int lsb = lead == INT_MIN ? 0 : lead - 27;
            // two rounds: q in units of 2^lsb, then what that leaves in units of 2^(lsb - 28): half a unit of the first at most,
            // and nothing in most rows (with one round, a row whose smallest element is 20 binades below its largest leaves an
            // eighth of its pairs to the exact path)
            int lost = 0, more = 0;
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2) {
                uint32_t y[2];
                lost = 0;
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int a = m[h] < 0 ? -m[h] : m[h], sh = e[h] - lsb + 28 * k2;
                    int X = 0, rest = 0;
                    if (a && !bad) {
                        if (sh >= 0) {
                            X = a << sh;
                        } else {
                            X = sh >= -10 ? (a + (1 << (-sh - 1))) >> -sh : 0;
                            rest = sh >= -10 ? a - (X << -sh) : a;
                        }
                    }
                    y[h] = (uint32_t)(m[h] < 0 ? -X : X) + 0x21084210u;
                    m[h] = m[h] < 0 ? -rest : rest;
                    lost += rest != 0;
                }
#pragma unroll
                for (int k = 0; k < 6; ++k) {
                    uint32_t c2 = 0;
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const int dk = (int)((y[h] >> (5 * k)) & 31u) - 16;
                        c2 |= (dk < 0 ? 32u | (uint32_t)-dk : (uint32_t)dk) << (8 * h);
                    }
                    *(uint16_t*)&S.dig[k2][(r * 6 + k) * 128 + 2 * lane] = (uint16_t)c2;
                }
                if (k2 == 0) more = __ballot(lost != 0) != 0;
            }
            lost = wave_sum_i(lost);
            if (lane == 0) {
                S.bad[r] = bad;
                S.more[r] = more;
                S.rq[r] = ldexp(P.alpha, lsb + 3);
                S.rqe[r] = fabs(P.alpha) * (double)lost * ldexp(0.5 * (1.0 + 0x1p-20), lsb - 28);
            }
        }
        __syncthreads();  // the digits are in LDS: 32 of a block to 24 bytes
        int any = 0, two = 0;  // does a row of the block, of the wave, need the second round?
#pragma unroll
        for (int r = 0; r < RB; ++r) any |= S.more[r];
#pragma unroll
        for (int r = 0; r < RS; ++r) two |= S.more[wrow + r];
        any = __builtin_amdgcn_readfirstlane(any);
        two = __builtin_amdgcn_readfirstlane(two);
        for (int x0 = tid; x0 < RB * 24 * (1 + any); x0 += F4_THREADS) {
            const int k2 = x0 >= RB * 24, x = x0 - (k2 ? RB * 24 : 0);
            const uint32_t* src = (const uint32_t*)&S.dig[k2][(x >> 2) * 128 + 32 * (x & 3)];
            uint32_t c[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const uint32_t y = src[j];  // 4 codes of 6 bits in bytes
                c[j] = (y & 0x3Fu) | (y >> 2 & 0xFC0u) | (y >> 4 & 0x3F000u) | (y >> 6 & 0xFC0000u);
            }
            f4_u2* const o = (f4_u2*)&S.q6[k2][x * 6];
            o[0] = (f4_u2){c[0] | c[1] << 24, c[1] >> 8 | c[2] << 16};
            o[1] = (f4_u2){c[2] >> 16 | c[3] << 8, c[4] | c[5] << 24};
            o[2] = (f4_u2){c[5] >> 8 | c[6] << 16, c[6] >> 16 | c[7] << 8};
        }
        __syncthreads();
        // the lane's part of a row block's digits, instruction j: M = n is digit 4 j + n % 4 of the digits of the rows of n / 4
        auto q_part = [&](int k2, int j) __attribute__((always_inline)) {
            const int c = RS == 2 ? n & 7 : 4 * j + (n & 3);
            const int qr = wrow + (RS == 2 ? n >> 3 : n >> 2);
            const uint32_t* const p = c >= 6 ? S.zero : &S.q6[k2][((qr * 6 + c) * 4 + g) * 6];
            const f4_u2 x = *(const f4_u2*)p, y = *(const f4_u2*)(p + 2), t = *(const f4_u2*)(p + 4);
            return (f4_i8){(int)x.x, (int)x.y, (int)y.x, (int)y.y, (int)t.x, (int)t.y, 0, 0};
        };
        f4_i8 qd[NMF];
#pragma unroll
        for (int j = 0; j < NMF; ++j) qd[j] = q_part(0, j);
        const double alpha = P.alpha;
        int rfl = S.bad[wrow + row];  // the row is left to tier 2
        int base = F4_NONE;    // of the row
        double z = 0.0, lostw = 0.0;  // the weights' sum, and what rounding took from their whole numbers
        int G[NG];             // the groups' references, uniform
#pragma unroll
        for (int l = 0; l < NG; ++l) G[l] = 0;
        int lo = 120;          // scales of keys in [lo, lo + F4_SPREAD] need no closer look: at first 2^-7 .. 2^2
        int kexp = 2;          // 6 2^kexp bounds |k| of such keys
        f4_i4 acc[NMF][2 * NG];
        // the lane's own sums: [c], or with 2 rows those of c = 2 l + g % 2
        constexpr int OC = RS == 2 ? NG : 2 * NG, OS = RS == 2 ? 32 : 16;
        double* const O = &S.O[w][row][8 * sub + n];
#pragma unroll
        for (int c = 0; c < 2 * NG; ++c) {
#pragma unroll
            for (int j = 0; j < NMF; ++j) acc[j][c] = (f4_i4){0, 0, 0, 0};
            if (c < OC) O[OS * c] = 0.0;
        }
        int since = 0, folds = 0;
        int n5 = 0, n6 = 0, n8 = 0, cnt = 0;  // wave-uniform
        const double gw = RS == 2 ? (g == 0 ? 1.0 : (g == 1 ? 0x1p16 : 0x1p32)) : (g == 0 ? 1.0 : (g == 1 ? 0x1p8 : (g == 2 ? 0x1p16 : 0x1p24)));

        // the int32 sums into the fp64 ones: digits joined, the lanes' parts added up, each lane left with its own rows
        auto fold = [&]() __attribute__((always_inline)) {
#pragma unroll
            for (int l = 0; l < NG; ++l) {
                const double unit = ldexp(gw, G[l] - 128);  // in halves of 2^(G - 127)
                if constexpr (RS == 2) {
                    double a[2];
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const f4_i4 x = acc[0][2 * l + h];
                        const double t0 = __fma_rn((double)x[2], 256.0, (double)x[0]) * unit, t1 = __fma_rn((double)x[3], 256.0, (double)x[1]) * unit;
                        a[h] = (row ? t1 : t0) + xor32(row ? t0 : t1);
                        acc[0][2 * l + h] = (f4_i4){0, 0, 0, 0};
                    }
                    O[32 * l] += (sub ? a[1] : a[0]) + xor16(sub ? a[0] : a[1]);
                    continue;
                }
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int c = 2 * l + h;
                    double t[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        double x = (double)acc[NMF - 1][c][i];
#pragma unroll
                        for (int j = NMF - 2; j >= 0; --j) x = __fma_rn(x, 65536.0, (double)acc[j][c][i]);
                        t[i] = x * unit;
                    }
                    const bool up = g >= 2;
                    double a = up ? t[2] : t[0], e = up ? t[3] : t[1];
                    a += xor32(up ? t[0] : t[2]);
                    e += xor32(up ? t[1] : t[3]);
                    const bool odd = g & 1;
                    O[16 * c] += (odd ? e : a) + xor16(odd ? a : e);
#pragma unroll
                    for (int j = 0; j < NMF; ++j) acc[j][c] = (f4_i4){0, 0, 0, 0};
                }
            }
            ++folds;
            since = 0;
        };
        // a row's base to nb (the same in every lane of the row), after a fold
        auto rebase = [&](int nb) __attribute__((always_inline)) {
            double f = 1.0;
            if (nb != base) {
                if (base != F4_NONE) {
                    if (!MOD && base - nb < -900) rfl = 1;
                    f = ldexp(1.0, max(base - nb, -1000));
                    z *= f;
                    lostw *= f;
                }
                base = nb;
            }
#pragma unroll
            for (int c = 0; c < OC; ++c) O[OS * c] *= f;
        };

        auto tile = [&](int n0) __attribute__((always_inline)) {
            const Pages after = pages_of(n0 + 2 * STEP);
            // ---- are the scales near enough to each other for exact sums?
            uint32_t wide = 0;  // bit u: key 4 n + u is left to the exact path
            {
                uint32_t far = 0;
#pragma unroll
                for (int u = 0; u < 4; ++u) far |= (uint32_t)((int)kr.s[u] - lo) > F4_SPREAD ? 1u : 0u;
                if (__builtin_expect(__ballot(far != 0) != 0, 0)) {
                    int top = 0;
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t any = (kr.k[u].x | kr.k[u].y | kr.k[u].z | kr.k[u].w) & 0x77777777u;
                        const bool has = any != 0 || kr.s[u] == 255;  // groups of zeros take any scale
                        int mx = has ? (int)kr.s[u] : 0, mn = has ? (int)kr.s[u] : 1000;
                        mx = max(mx, __shfl_xor(mx, 16, 64));
                        mn = min(mn, __shfl_xor(mn, 16, 64));
                        mx = max(mx, __shfl_xor(mx, 32, 64));
                        mn = min(mn, __shfl_xor(mn, 32, 64));
                        // sums far from fp32's ends, too
                        const bool off = mn != 1000 && (mx - mn > F4_SPREAD || mn < 40 || mx > 230);
                        if (!has) kr.s[u] = 127;
                        if (off) {
                            wide |= 1u << u;
                        } else if (mn != 1000) {
                            top = max(top, mx);
                        }
                    }
                    top = wave_max_dpp(top);
                    if (top > 0) lo = __builtin_amdgcn_readfirstlane(max(top - (F4_SPREAD - 1), 40));
                    kexp = max(kexp, __builtin_amdgcn_readfirstlane(max(top, lo + F4_SPREAD)) - 127);
                }
            }
            const bool edge = n0 + 64 > min(kvmin, k1) || (MOD && n0 < kbmax);
            const bool cut = n0 + 64 > k1 || (MOD && n0 < kbeg);
            const int kn = n0 + 4 * n + sub;  // the first of the lane's keys
            if constexpr (KL == 2) wide >>= sub;
            // ---- scores: 6 exact sums for every pair
            double sc[4];
            auto products = [&](const f4_i8 (&qa)[NMF], double (&x)[4]) __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const f4_i8 B = {(int)kr.k[u].x, (int)kr.k[u].y, (int)kr.k[u].z, (int)kr.k[u].w, 0, 0, 0, 0};
                    f4_f4 D[NMF];
#pragma unroll
                    for (int j = 0; j < NMF; ++j)
                        D[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(qa[j], B, (f4_f4){0.0f, 0.0f, 0.0f, 0.0f}, 2, 4, 0, 127, 0,
                                                                                (int)kr.s[u]);
                    constexpr int LAST = RS == 2 ? 3 : 5;
                    x[u] = (double)D[LAST >> 2][LAST & 3];
#pragma unroll
                    for (int k = LAST - 1; k >= 0; --k) x[u] = __fma_rn(x[u], 32.0, (double)D[k >> 2][k & 3]);
                    if constexpr (RS == 2) x[u] *= sub ? 0x1p20 : 1.0;
                }
                if constexpr (RS == 2) {
                    // digits 0..3 of a row's sums lie 16 lanes before digits 4 and 5: the first lane takes keys 0 and 1, the other 2 and 3
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const auto lo = __builtin_amdgcn_permlane16_swap(__double2loint(x[u]), __double2loint(x[u + 2]), false, false);
                        const auto hi = __builtin_amdgcn_permlane16_swap(__double2hiint(x[u]), __double2hiint(x[u + 2]), false, false);
                        x[u] = __hiloint2double((int)hi[0], (int)lo[0]) + __hiloint2double((int)hi[1], (int)lo[1]);
                    }
                }
            };
            products(qd, sc);
            if (__builtin_expect(two, 0)) {
                f4_i8 q2[NMF];
                double s2[4];
#pragma unroll
                for (int j = 0; j < NMF; ++j) q2[j] = q_part(1, j);
                products(q2, s2);
#pragma unroll
                for (int i = 0; i < KL; ++i) sc[i] = __fma_rn(s2[i], 0x1p-28, sc[i]);  // one rounding, in the weights' bound
            }
            issue_k(n0 + STEP, nx, kr);
            double md[KL];  // the weights: md 2^(base + ex)
            int ex[KL];
            constexpr uint32_t ALL = (1u << KL) - 1u;
            // ---- certified weights
            const double adel = S.rqe[wrow + row] * ldexp(6.0, kexp), rq = S.rq[wrow + row];
            bool ok[KL];
            double x[KL];
#pragma unroll
            for (int i = 0; i < KL; ++i) x[i] = sc[i];
            if constexpr (MOD >= 2) {
                float sl[KL];
                int dist[KL], Mi[KL];
                double ad[KL];
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    sl[i] = S.slope[wrow + row];
                    dist[i] = kn + i - S.pos[wrow + row];
                    ad[i] = __fma_rn(fabs(x[i] * rq), 0x1p-52, adel);
                }
                pf::cert_pairs<KL, MOD>(x, ad, rq, S.T1, S.T2, Mi, ex, ok, P.cap, sl, dist);
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    md[i] = (double)Mi[i];
                    ok[i] &= ex[i] < (1 << 29) && ex[i] > -(1 << 29) - 23;  // differences from a base fit an int
                    ex[i] -= base;
                }
            } else {
                four_weights<KL>(x, rq, 0x1p-49, adel, S.T1, S.T2, md, ex, ok);
#pragma unroll
                for (int i = 0; i < KL; ++i) ex[i] -= base + 23;
            }
            // ---- which of the pairs are visible (rows past the last one weigh what they like)
            uint32_t vis = ALL;
            if (edge) {
                vis = 0;
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    const int key = kn + i, ti = key - tb;
                    const bool in = ((unsigned)ti < 64u) & (((S.tmk[wrow + row] >> (ti & 63)) & 1ull) != 0);
                    bool pre = key < S.kvl[wrow + row];
                    if constexpr (MOD) pre = pre & (key >= S.kvb[wrow + row]);
                    vis |= ((key < k1) & (pre | in)) ? (1u << i) : 0u;
                }
            }
            bool all = (vis == ALL) & (wide == 0);
#pragma unroll
            for (int i = 0; i < KL; ++i) all = all & ok[i];
            if (__ballot(!all) != 0) {
                if constexpr (MOD < 2) {
                    // A score of few bits may lie on a tie of t: 1 pair in 2^14 of normal q and K. Where the product is exact, too, it
                    // rounds to even like any other
#pragma unroll
                    for (int i = 0; i < KL; ++i) {
                        const bool tie = !two && !ok[i] && adel == 0.0 && __fma_rn(rq, x[i], -(rq * x[i])) == 0.0;
                        if (__ballot(tie) != 0) {
                            const double xt[1] = {x[i]};
                            double yt[1];
                            int ft[1];
                            bool okt[1];
                            four_weights<1>(xt, rq, 0.0, 0.0, S.T1, S.T2, yt, ft, okt);
                            const bool take = tie && okt[0];
                            ok[i] = ok[i] | take;
                            md[i] = take ? yt[0] : md[i];
                            ex[i] = take ? ft[0] - (base + 23) : ex[i];
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                }
                uint32_t gd = 0;
#pragma unroll
                for (int i = 0; i < KL; ++i) gd |= ok[i] ? (1u << i) : 0u;
                gd &= ~wide;
                const uint32_t slow = wrow + row < nrow ? vis & ~gd : 0u;
                gd &= vis;
                if (__builtin_expect(__ballot(slow != 0) != 0, 0)) {
                    // undecided pairs wait in the wave's list for flush(); a row that is flagged already needs no more of them
#pragma unroll
                    for (int i = 0; i < KL; ++i) {
                        const bool put = ((slow >> i) & 1) && !rfl;
                        const uint64_t m = __ballot(put);
                        if (put)
                            S.list[w][cnt + __builtin_amdgcn_mbcnt_hi((uint32_t)(m >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)m, 0))] =
                                (uint32_t)(row) << 29 | (uint32_t)(kn + i - kA);
                        cnt += (int)__popcll(m);
                    }
                }
#pragma unroll
                for (int i = 0; i < KL; ++i) {  // the others weigh nothing
                    const bool y = (gd >> i) & 1;
                    md[i] = y ? md[i] : 0.0;
                    ex[i] = y ? ex[i] : F4_BITS;
                }
            }
            // ---- bases and references move when a weight or a scale passes them
            if (cut) {  // scales of slots past the last key (or before the first) may be anything
                uint32_t keep = 0;
#pragma unroll
                for (int i = 0; i < KL; ++i) keep |= (kn + i < k1 && (!MOD || kn + i >= kbeg)) ? 0xFFu << (8 * i) : 0u;
#pragma unroll
                for (int l = 0; l < NG; ++l) vr.s[l] &= keep;
            }
            int most = ex[0];
#pragma unroll
            for (int i = 1; i < KL; ++i) most = max(most, ex[i]);
            f4_h2 top[NG];  // of the scales of even and odd keys
            uint32_t past = 0;
#pragma unroll
            for (int l = 0; l < NG; ++l) {
                const uint32_t x = vr.s[l];
                top[l] = pk_max(__builtin_bit_cast(f4_h2, x & 0x00FF00FFu), __builtin_bit_cast(f4_h2, x >> 8 & 0x00FF00FFu));
                const f4_h2 ref = __builtin_bit_cast(f4_h2, (uint32_t)G[l] * 0x10001u);
                past |= __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(top[l], ref));
            }
            if (__ballot(most > F4_BITS || past != 0) != 0 || since >= F4_EPOCH) {
                if (since) fold();
#pragma unroll
                for (int l = 0; l < NG; ++l) {
                    const int m = wave_max_dpp((int)max(top[l].x, top[l].y));
                    G[l] = max(G[l], m >= G[l] ? min(m + 1, 255) : 0);  // one binade of room
                }
                int m = 0;
#pragma unroll
                for (int i = 0; i < KL; ++i) m = max(m, ex[i]);  // pairs that weigh nothing have F4_BITS
                for (int o = 1; o < RLANES; o <<= 1) m = max(m, __shfl_xor(m, o, 64));
                const int up = m > F4_BITS ? m - (F4_BITS - F4_HEAD) : 0;
#pragma unroll
                for (int i = 0; i < KL; ++i) ex[i] = md[i] != 0.0 ? ex[i] - up : F4_BITS;
                if (folds) {
                    rebase(base + up);
                } else {
                    base += up;  // nothing summed yet
                }
            }
            ++since;
            if constexpr (KL == 2) z += ldexp(md[0], ex[0]) + ldexp(md[1], ex[1]);
            else z += (ldexp(md[0], ex[0]) + ldexp(md[1], ex[1])) + (ldexp(md[KL - 2], ex[KL - 2]) + ldexp(md[KL - 1], ex[KL - 1]));
            // ---- P.V: a phase writes the digits of its groups and reads them back; the next one writes them anew (a wave's LDS
            // accesses keep their order)
            auto digits = [&](const int l) __attribute__((always_inline)) {
                uint32_t* const W = S.W[w][l];
                constexpr double BIG = 0x1.8p52 + 141289400074368.0;  // and 0x808080808080
                const uint32_t below = (uint32_t)G[l] * (KL == 4 ? 0x01010101u : 0x0101u) - vr.s[l];  // bytes, none of them negative
                uint32_t L[KL], H[KL];
                double xw[KL], y[KL];
                int least = 0;
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    const int sh = ex[i] - (int)(below >> (8 * i) & 0xFFu);
                    least = min(least, sh);
                    xw[i] = ldexp(md[i], sh);
                    y[i] = xw[i] + BIG;
                    L[i] = (uint32_t)__double2loint(y[i]);
                    H[i] = (uint32_t)__double2hiint(y[i]);
                }
                if (__builtin_expect(__ballot(least < 0) != 0, 0)) {
#pragma unroll
                    for (int i = 0; i < KL; ++i) lostw += fabs(xw[i] - (y[i] - BIG));
                }
                // byte p of the sums is plane p: transpositions of 4 x 4 and 4 x 2 bytes, or 2 x 4 and 2 x 2
                const uint32_t l01 = __builtin_amdgcn_perm(L[1], L[0], 0x05010400u), h01 = __builtin_amdgcn_perm(L[1], L[0], 0x07030602u);
                const uint32_t t01 = __builtin_amdgcn_perm(H[1], H[0], 0x05010400u);
                if constexpr (KL == 2) {
                    const uint32_t pp[3] = {l01 ^ 0x80808080u, h01 ^ 0x80808080u, t01 ^ 0x80808080u};
                    uint16_t* const at = (uint16_t*)&W[row * F4_WROW + n] + (sub >> 1);
#pragma unroll
                    for (int p = 0; p < 6; ++p) at[p * 2 * RS * F4_WROW] = (uint16_t)(pp[p >> 1] >> (16 * (p & 1)));
                } else {
                    const uint32_t l23 = __builtin_amdgcn_perm(L[KL - 1], L[KL - 2], 0x05010400u);
                    const uint32_t h23 = __builtin_amdgcn_perm(L[KL - 1], L[KL - 2], 0x07030602u);
                    const uint32_t t23 = __builtin_amdgcn_perm(H[KL - 1], H[KL - 2], 0x05010400u);
                    const uint32_t pl[6] = {__builtin_amdgcn_perm(l23, l01, 0x05040100u), __builtin_amdgcn_perm(l23, l01, 0x07060302u),
                                            __builtin_amdgcn_perm(h23, h01, 0x05040100u), __builtin_amdgcn_perm(h23, h01, 0x07060302u),
                                            __builtin_amdgcn_perm(t23, t01, 0x05040100u), __builtin_amdgcn_perm(t23, t01, 0x07060302u)};
                    const int at = row * F4_WROW + n;
#pragma unroll
                    for (int p = 0; p < 6; ++p) W[p * RS * F4_WROW + at] = pl[p] ^ 0x80808080u;
                }
            };
            auto multiply = [&](const int l) __attribute__((always_inline)) {
                const uint32_t* const W = S.W[w][l];
                f4_i4 A[NMF];
                if constexpr (RS == 2) {
                    const uint32_t* const a0 = n < 12 ? &W[n * F4_WROW + 4 * g] : S.zero;
                    A[0] = __builtin_bit_cast(f4_i4, *(const f4_u4*)a0);
                } else {
                    const uint32_t* const a0 = n < 8 ? &W[n * F4_WROW + 4 * g] : S.zero;
                    A[0] = __builtin_bit_cast(f4_i4, *(const f4_u4*)a0);
                    A[NMF - 1] = __builtin_bit_cast(f4_i4, *(const f4_u4*)&W[(8 + n) * F4_WROW + 4 * g]);
                }
                f4_i4 B0, B1;
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    B0[x] = (int)four_bytes<false>(vr.v[l][x]);
                    B1[x] = (int)four_bytes<true>(vr.v[l][x]);
                }
#pragma unroll
                for (int j = 0; j < NMF; ++j) {
                    acc[j][2 * l] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[j], B0, acc[j][2 * l], 0, 0, 0);
                    acc[j][2 * l + 1] = __builtin_amdgcn_mfma_i32_16x16x64_i8(A[j], B1, acc[j][2 * l + 1], 0, 0, 0);
                }
            };
#pragma unroll
            for (int l = 0; l < NG; ++l)
                if (l < ng) digits(l);
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int l = 0; l < NG; ++l)
                if (l < ng) multiply(l);
            __builtin_amdgcn_sched_barrier(0);
            issue_v(n0 + STEP, nx, vr);
            nx = after;
            __builtin_amdgcn_sched_barrier(0);
        };

        // ---- the pairs waiting in the list, 4 at a time and 16 lanes a pair: every product of the score separately,
        // TwoSum-accumulated, the certified weight, then one pair after another into the row's fp64 sums. (A lane a pair took 8 us of a
        // step with one such pair, most of it waiting for 16 loads in turn.)
        auto flush = [&]() __attribute__((always_inline)) {
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (int at = 0; at < cnt; at += 4) {
                const bool have = at + g < cnt;
                const uint32_t en = have ? S.list[w][at + g] : 0u;
                const int er = (int)(en >> 29), ek = kA + (int)(en & 0x1FFFFFFFu);
                double ss = 0.0, es = 0.0, ea = 0.0;
                if (have && 8 * n < d) {
                    const uint16_t* qr = q_row(wrow + er) + 8 * n;
                    const uint4 kv = kv4_load8(P.k, P.ks, kv_off(P, b, ek, hk, 0) + 8 * n);
                    const uint32_t wd[4] = {kv.x, kv.y, kv.z, kv.w};
                    uint32_t qw[8];
#pragma unroll
                    for (int h = 0; h < 8; ++h) qw[h] = qr[h];
#pragma unroll
                    for (int h = 0; h < 4; ++h) {
                        double e0, e1;
                        ss = two_sum(ss, (double)__uint_as_float(qw[2 * h] << 16) * bf16lo_f64(wd[h]), &e0);
                        ss = two_sum(ss, (double)__uint_as_float(qw[2 * h + 1] << 16) * bf16hi_f64(wd[h]), &e1);
                        es += e0 + e1;
                        ea += fabs(e0) + fabs(e1);
                    }
                }
#pragma unroll
                for (int o = 1; o < 16; o <<= 1) {  // alike in both lanes: a sum and its error do not depend on the order
                    double e;
                    ss = two_sum(ss, __shfl_xor(ss, o, 64), &e);
                    es = (es + __shfl_xor(es, o, 64)) + e;
                    ea = (ea + __shfl_xor(ea, o, 64)) + fabs(e);
                }
                int32_t Mi = 0, Ei = 0;
                bool live = false;
                int why = 0;  // 1 score not certified, 2 weight not certified
                const bool fin = have && isfinite(ss);
                if (have) {
                    uint32_t tbits = 0;
                    int ls = 3;
                    if (fin) {
                        const bool zero = ss == 0.0 && es == 0.0 && ea == 0.0;
                        ls = zero ? 1 : logit_cert(alpha, ss, es, ea * 0x1p-44, &tbits);
                        if (ls == 1) tbits = 0;
                        if constexpr (MOD >= 2) ls = mod_logit(ls, zero, P.cap, S.slope[wrow + er], ek - S.pos[wrow + er], S.T1, 23, &tbits);
                    }
                    if (ls == 2 || ls == 3) {
                        why = 1;  // undecided, or an overflow (tier 2 reports the domain error)
                    } else if (pf::table_weight(tbits, S.T1, S.T2, &Mi, &Ei)) {
                        live = true;
                    } else {
                        int64_t E2 = 0;
                        live = weight_wide(tbits, &Mi, &E2) == 0 && E2 > -(1LL << 30) && E2 < (1LL << 30);
                        if (!live) why = 2;
                        Ei = (int32_t)E2;
                    }
                }
                const uint64_t lead4 = 0x0001000100010001ull;  // a lane of each pair
                n5 += (int)__popcll(__ballot(why == 1) & lead4);
                n6 += (int)__popcll(__ballot(why == 2) & lead4);
                n8 += (int)__popcll(__ballot(fin) & lead4);
                for (uint64_t m = __ballot(have && !live) & lead4; m; m &= m - 1) {
                    const int r = __builtin_amdgcn_readlane(er, __builtin_ctzll(m));
                    if (row == r) rfl = 1;
                }
                for (uint64_t lv = __ballot(live) & lead4; lv; lv &= lv - 1) {
                    const int ln = __builtin_ctzll(lv);
                    const int r = __builtin_amdgcn_readlane(er, ln), key = __builtin_amdgcn_readlane(ek, ln);
                    const int Mr = __builtin_amdgcn_readlane(Mi, ln), Er = __builtin_amdgcn_readlane(Ei, ln);
                    const int64_t vc = kv4_v(P, b, key, hk);
                    uint32_t v2[NG];
#pragma unroll
                    for (int l = 0; l < NG; ++l) v2[l] = l < ng ? kv4_vload2(P.v, P.vs, vc, 32 * l + 2 * n) : 0u;
                    if (row == r) {
                        if (Er > base + F4_BITS) rebase(Er - (F4_BITS - F4_HEAD));
                        const int de = Er - base;
                        if (!MOD && de < -1000) rfl = 1;
                        const double om = de < -1000 ? 0.0 : ldexp((double)Mr, de);
                        z += head ? om : 0.0;
#pragma unroll
                        for (int l = 0; l < NG; ++l) {
                            if (l >= ng) break;
                            double* const o = &O[32 * l];
                            if constexpr (RS == 2) {
                                o[0] = __fma_rn(om, sub ? bf16hi_f64(v2[l]) : bf16lo_f64(v2[l]), o[0]);
                                continue;
                            }
                            o[0] = __fma_rn(om, bf16lo_f64(v2[l]), o[0]);
                            o[16] = __fma_rn(om, bf16hi_f64(v2[l]), o[16]);
                        }
                    }
                    ++folds;
                }
            }
            cnt = 0;
        };

        // ---- the wave's tiles: K of the next one is requested once the scores have read this one's registers, V once P.V has;
        // pages are looked up a tile before that. A flush (rare) drops the loads in flight and starts over
        for (int it = 0; it < nst;) {
#pragma unroll 1
            for (; it < nst && cnt < F4_LIST; ++it) tile(k0w + STEP * it);
            if (since) fold();
            if (cnt > 0) {
                flush();
                if (it < nst) begin(k0w + STEP * it);
            }
        }

        // ---- epilogue: row totals of the wave, then the 4 waves' partials at the rows' largest base (exact powers of two), two
        // additions deep
        {
            double zs = z, ls = lostw;
            int fl = rfl;
            for (int o = 1; o < RLANES; o <<= 1) {
                zs += __shfl_xor(zs, o, 64);
                ls += __shfl_xor(ls, o, 64);
                fl |= __shfl_xor(fl, o, 64);
            }
            if (head) {
                S.wR[w][row] = base;
                S.wZ[w][row] = zs;
                S.we[w][row] = ls;
                S.wf[w][row] = fl;
            }
            if (lane == 0) S.wn[w] = folds;
#pragma unroll
            for (int l = 0; l < NG; ++l)
                if (lane == 0) S.wv[w][l] = (uint32_t)G[l];
        }
        __syncthreads();
        const int64_t pbase = (int64_t)split * P.rows;
        // WR = 1: the waves' factors to the row's largest base; otherwise one wave has it
        auto sums_at = [&](int r, double (&f)[4]) __attribute__((always_inline)) {
            int Rm = F4_NONE, far = 0;
            if constexpr (WR > 1) return S.wR[r / RS][r % RS];
            for (int ww = 0; ww < 4; ++ww) Rm = max(Rm, S.wR[ww][r]);
#pragma unroll
            for (int ww = 0; ww < 4; ++ww) {
                const bool any = S.wR[ww][r] != F4_NONE;
                const int sh = any ? S.wR[ww][r] - Rm : 0;
                far |= !MOD && sh < -900;
                f[ww] = any ? ldexp(1.0, max(sh, -1000)) : 0.0;
            }
            return far ? INT_MIN : Rm;
        };
        // a thread 2 channels of a row at a time
        for (int x = tid; x < nrow * 16 * NG; x += F4_THREADS) {
            const int r = x / (16 * NG), p = x % (16 * NG), l = p >> 4, c = p & 15;
            if (2 * p >= dv) continue;
            double f[4], o[2];
            if constexpr (WR == 1) sums_at(r, f);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int at = 32 * l + 16 * h + c;
                if constexpr (WR > 1) o[h] = S.O[r / RS][r % RS][at];
                else o[h] = (f[0] * S.O[0][r][at] + f[2] * S.O[2][r][at]) + (f[1] * S.O[1][r][at] + f[3] * S.O[3][r][at]);
            }
            const int lr = row0 + r;
            const int64_t gr = row_index(P, b, lr / P.grp, hk * P.grp + lr % P.grp);
            *(double2*)(P.pN + (pbase + gr) * dv + 2 * p) = make_double2(o[0], o[1]);
        }
        if (w == 3 && lane < nrow) {
            const int r = lane;
            double f[4], lost = 0.0;
            const int Rm = sums_at(r, f);
            int fl = Rm == INT_MIN, fo = 0;
            double Z = 0.0;
            if constexpr (WR > 1) {
                fl |= S.wf[r / RS][r % RS];
                fo = S.wn[r / RS];
                lost = S.we[r / RS][r % RS];
                Z = S.wZ[r / RS][r % RS];
            } else {
                for (int ww = 0; ww < 4; ++ww) {
                    fl |= S.wf[ww][r];
                    fo += S.wn[ww];
                    lost += f[ww] * S.we[ww][r];
                }
                Z = (f[0] * S.wZ[0][r] + f[2] * S.wZ[2][r]) + (f[1] * S.wZ[1][r] + f[3] * S.wZ[3][r]);
            }
            // keys of the piece up to the row's last visible one: at least the keys summed
            const uint64_t tm = S.tmk[r];
            const int ke = min(tm ? max(S.kvl[r], tb + 64 - (int)__clzll(tm)) : S.kvl[r], k1);
            const int nk = Rm == F4_NONE ? 0 : ke - kA;
            // The depth that the combine multiplies by u Z max|v|. P.V: int32 sums are exact, a fold adds 4 numbers up, a pair of the
            // exact path one (8 each), 16 for the joins. Z: one sum for every 64 keys in a lane at most, 16 for the joins. What the
            // weights lost, at most 12 units of 2^(base + G) for each of theirs, which the combine takes for max|v|: lost / Z, in
            // units of u
            const double depth = (double)(nk >> 6) + 40.0 + 8.0 * (double)fo + (lost / Z) * (0x1p53 * (1.0 + 0x1p-20)) + 1.0;
            int most = nk;
            if (nk > 0) {
                if (!(depth < 0x1p28)) fl = 1;
                most = fl ? nk : (int)depth * (MOD ? 4 : 1);  // the modified steps' combine counts a quarter
            }
            const int lr = row0 + r;
            const int64_t o = pbase + row_index(P, b, lr / P.grp, hk * P.grp + lr % P.grp);
            P.pR[o] = Rm == F4_NONE ? INT_MIN : Rm;
            P.pZ[o] = Z;
            P.pn[o] = fl ? -1 : most;
        } else if (w == 2) {
            for (int ch = lane; ch < dv; ch += 64) {
                const int l = ch >> 5;
                const uint32_t top = max(max(S.wv[0][l], S.wv[1][l]), max(S.wv[2][l], S.wv[3][l]));
                P.pV[(((int64_t)split * P.nseg + seg) * P.nrb + rbk) * dv + ch] = kv4_bound(top);
            }
        }
        if (P.stats && lane == 0) {
            if (n5) atomicAdd((unsigned long long*)&P.stats[5], (unsigned long long)n5);
            if (n6) atomicAdd((unsigned long long*)&P.stats[6], (unsigned long long)n6);
            if (n8) atomicAdd((unsigned long long*)&P.stats[8], (unsigned long long)n8);
        }
    };

    // One piece per block on uniform splits; on the equal-share plan (Params::dq_*) one per unit its share reaches, read as the
    // decode kernel reads it. A segment's row blocks go to one XCD (ea_decode.hip has both placements and their reasons).
    int u, start, end, share = 1, gb = 0;
    const int32_t* Su = P.dq_plan + 2;
    if (P.dq_stream) {
        gb = (int)blockIdx.x;
        if (P.nrb > 1 && (P.dq_blocks & 7) == 0 && (int64_t)P.dq_units * 8 > P.dq_blocks)
            gb = (gb & 7) * (P.dq_blocks >> 3) + (gb >> 3);
        const int4 rec = ((const int4*)(P.dq_plan + P.dq_rec_off))[gb];
        u = rec.x;
        share = rec.w;
        if (u >= P.dq_units || share <= 0) return;  // past the last share: no tile
        start = gb * share;
        end = min(start + share, P.dq_plan[0]);
    } else {
        u = (int)blockIdx.x;
        if (P.nrb > 1 && (P.nseg & 7) == 0) {
            const int lo = u & 7, hi = u >> 3;
            u = ((hi / P.nrb) * 8 + lo) * P.nrb + hi % P.nrb;
        }
        start = (int)blockIdx.y * (P.split_len >> 6);
        end = start + (P.split_len >> 6);
        if (MOD && blockIdx.y == gridDim.y - 1) end = 1 << 23;  // keys are below 2^29
    }
    for (bool first = true;; first = false) {
        int t0 = start, te = end, slot = (int)blockIdx.y;
        if (P.dq_stream) {
            if (start >= end || u >= P.dq_units) break;
            const int su = Su[u], eu = Su[u + 1];
            if (eu <= start) {
                ++u;
                continue;
            }
            slot = gb - su / share;
            t0 = start - su;
            te = min(end, eu) - su;
            start = min(end, eu);
            if (slot >= P.nsplit) break;  // share >= dq_min_share keeps every unit within nsplit slots
        }
        if (!first) __syncthreads();  // the previous piece's LDS reads are done
        piece(u, slot, t0 * 64, te * 64);
        if (!P.dq_stream) break;
        ++u;
    }
}

// Which drafted tokens stand, from the target's probabilities and given uniform numbers, and the token after them
// (gfx950; the definition is in exactattn_hip.h). No reference counterpart.
//
// A node's test reads one probability of its parent's row (and one of the draft's), so of a sequence's num_drafts + 1 rows only
// the one behind the last node that stands is read whole, with the draft's row at a rejection. What bounds it is latency: one launch,
// gridDim.x blocks a sequence. Each of them walks the nodes by itself (one wave, a lane a node), sums the weights of its part of the
// vocabulary and leaves the sum; the last one to do so finds the part that holds the new token, and the token in it.
// A chain of 4 over 32000 tokens 7.4 us, 64 chains of 8 over 128000 22 (65 MB, 13 at the copy rate), 16 trees of 16 over 50021 9.
// Weights are whole numbers of 2^-44, so their sums are exact in any order and the token does not depend on the split.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/exactattn_hip.h"

namespace {

int herr(hipError_t e) { return e == hipSuccess ? 0 : -100 - (int)e; }

constexpr int DC_THREADS = 256;
constexpr int DC_MAX_PARTS = 64;
constexpr int DC_WORK = DC_MAX_PARTS + 1;  // of the workspace, a sequence: a sum for each part, and their count
constexpr int DC_MAX_NODES = 64;
constexpr int DC_MAX_VOCAB = 1 << 19;
// a part is whole tiles, 8 at most: a thread's sums of 32 whole numbers up to 2^44 are exact in fp64
constexpr int DC_TILE = DC_THREADS * 4;

__device__ __forceinline__ double clip(float p) { return p > 0.0f ? (double)fminf(p, 1.0f) : 0.0; }  // NaN: 0

__device__ __forceinline__ uint64_t shfl_up64(uint64_t x, int o) {
    return (uint64_t)__shfl_up((unsigned long long)x, o, 64);
}
// inclusive over the wave
__device__ __forceinline__ uint64_t wave_scan64(uint64_t x, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint64_t y = shfl_up64(x, o);
        if (lane >= o) x += y;
    }
    return x;
}

struct Choice {
    int row, qrow;  // of probs, and of draft_probs (-1: none)
};

// 4 tokens' probabilities from token i on, zeros past the vocabulary
__device__ __forceinline__ float4 load4(const float* p, int i, int V, bool wide) {
    if (wide && i + 3 < V) return *(const float4*)(p + i);
    float4 x;
    x.x = i < V ? p[i] : 0.0f;
    x.y = i + 1 < V ? p[i + 1] : 0.0f;
    x.z = i + 2 < V ? p[i + 2] : 0.0f;
    x.w = i + 3 < V ? p[i + 3] : 0.0f;
    return x;
}

__global__ void __launch_bounds__(DC_THREADS) ea_draft_check_kernel(ea_draft_check A, int part) {
    __shared__ Choice s_at;
    __shared__ int s_len, s_out, s_last, s_pick;
    __shared__ int s_gone[DC_MAX_NODES], s_ngone;  // tokens that p has lost
    __shared__ uint32_t s_bits[DC_MAX_VOCAB / DC_MAX_PARTS / 32 + 1];
    __shared__ uint64_t s_sum[DC_THREADS / 64], s_part[DC_MAX_PARTS];
    __shared__ uint64_t s_goal;
    __shared__ int s_whole;
    const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
    const int b = (int)blockIdx.y, N = A.num_drafts, V = A.vocab, parts = (int)gridDim.x;
    const float* const P = A.probs + b * A.p_seq_stride;
    const float* const Q = A.draft_probs ? A.draft_probs + b * A.q_seq_stride : nullptr;
    const float* const U = A.uniforms + (int64_t)b * (N + 1);
    if (w == 0) {
        const int n = A.counts ? min(max(A.counts[b], 0), N) : N;
        int x = -1, par = -2;
        float p = 0.0f, q = 0.0f, u = 2.0f;
        if (lane < n) {
            x = A.drafted[(int64_t)b * N + lane];
            par = A.parents ? A.parents[(int64_t)b * N + lane] : lane - 1;
            u = U[lane];
            if (x < 0 || x >= V || par < -1 || par >= lane) par = -2;  // nobody's child
            else p = P[(par + 1) * A.p_row_stride + x];
            if (par != -2 && Q) q = Q[lane * A.q_row_stride + x];
        }
        const double pc = clip(p);
        const bool ok = Q && (double)u * clip(q) < pc;
        int cur = -1, len = 0, mine = -1;  // mine: the node at place `lane` of the path
        double gone = 0.0;
        uint64_t out = 0;  // the children of cur that did not stand
        for (uint64_t todo = __ballot(par == -1); todo;) {
            const int i = __builtin_ctzll(todo);
            todo &= todo - 1;
            bool take;
            if (Q) {
                take = (__ballot(ok) >> i) & 1;
            } else {
                const int xi = __shfl(x, i, 64);
                const bool twice = (__ballot(x == xi) & out) != 0;
                const double pi = __shfl(pc, i, 64);
                take = !twice && (double)__shfl(u, i, 64) * (1.0 - gone) < pi;
                if (!take && !twice) gone += pi;
            }
            if (take) {
                if (lane == len) mine = i;
                ++len;
                cur = i;
                gone = 0.0;
                out = 0;
                todo = __ballot(par == i);
            } else {
                out |= 1ull << i;
                if (Q) break;  // a chain ends
            }
        }
        // the tokens p has lost: those of the last node's children
        if (!Q && ((out >> lane) & 1)) s_gone[__popcll(out & ((1ull << lane) - 1))] = x;
        const int tok = __shfl(x, max(mine, 0), 64);
        if (lane == 0) {
            s_ngone = Q ? 0 : (int)__popcll(out);
            s_at.row = cur + 1;
            s_at.qrow = Q && len < n ? len : -1;
            s_len = len;
        }
        if (blockIdx.x == 0) {
            if (lane == 0) A.accepted[b] = len;
            if (lane < N) A.path[(int64_t)b * N + lane] = lane < len ? mine : -1;
            // the new token's place (len) is the last block's
            if (lane < len) A.tokens[(int64_t)b * (N + 1) + lane] = tok;
            if (lane > len && lane <= N) A.tokens[(int64_t)b * (N + 1) + lane] = -1;
            if (lane == 0 && N == 64 && len < 64) A.tokens[(int64_t)b * 65 + 64] = -1;
        }
    }
    __syncthreads();
    const float* const pr = P + s_at.row * A.p_row_stride;
    const float* const qr = s_at.qrow >= 0 ? Q + s_at.qrow * A.q_row_stride : nullptr;
    const bool wide = !(((uintptr_t)pr | (qr ? (uintptr_t)qr : 0)) & 15);
    // which tokens of part k are out, a bit each
    auto mark = [&](int k) {
        const int lo = k * part;
        for (int i = tid; i <= part / 32; i += DC_THREADS) s_bits[i] = 0;
        __syncthreads();
        if (tid < s_ngone) {
            const int i = s_gone[tid] - lo;
            if (i >= 0 && i < part) atomicOr(&s_bits[i >> 5], 1u << (i & 31));
        }
        __syncthreads();
    };
    // the weights of tokens i .. i + 3 of the part from lo; all: p itself
    auto weights = [&](int lo, int i, float4 p, float4 q, bool all, double (&x)[4]) __attribute__((always_inline)) {
        const uint32_t out = all ? 0 : s_bits[(i - lo) >> 5] >> ((i - lo) & 31);
        const float pe[4] = {p.x, p.y, p.z, p.w}, qe[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const double a = clip(pe[j]);
            x[j] = trunc(fmax(all ? a : a - clip(qe[j]), 0.0) * 0x1p44);
            if ((out >> j) & 1) x[j] = 0.0;
        }
    };
    const float4 none = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    // the block's sum over part k, in thread 0; all: of p itself
    auto part_sum = [&](int k, bool all) -> uint64_t {
        const int lo = k * part, hi = min(lo + part, V);
        double s = 0.0;
        for (int i = lo + 4 * tid; i < hi; i += 2 * DC_TILE) {  // two tiles' loads at once
            const bool more = i + DC_TILE < hi;
            const float4 p[2] = {load4(pr, i, V, wide), more ? load4(pr, i + DC_TILE, V, wide) : none};
            const float4 q[2] = {qr && !all ? load4(qr, i, V, wide) : none, qr && !all && more ? load4(qr, i + DC_TILE, V, wide) : none};
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                if (e && !more) break;
                double x[4];
                weights(lo, i + e * DC_TILE, p[e], q[e], all, x);
                s += (x[0] + x[1]) + (x[2] + x[3]);
            }
        }
        uint64_t t = (uint64_t)s;
        for (int o = 32; o > 0; o >>= 1) t += (uint64_t)__shfl_xor((unsigned long long)t, o, 64);
        if (lane == 0) s_sum[w] = t;
        __syncthreads();
        t = 0;
        for (int e = 0; e < DC_THREADS / 64; ++e) t += s_sum[e];
        return t;
    };
    mark((int)blockIdx.x);
    const uint64_t own = part_sum((int)blockIdx.x, false);
    uint64_t* const sums = A.work + (int64_t)b * DC_WORK;
    uint64_t* const count = sums + DC_MAX_PARTS;
    if (tid == 0) {
        // An exchange happens where all dies meet, and one that has returned has happened: the count moves after the sum without a
        // release, which writes back a die's second-level cache for every block (64 sequences of 8 drafts over 128000 tokens, 1024
        // blocks: 50 us with it, 27 without, and 2048 blocks 75 and 24)
        const uint64_t was = __hip_atomic_exchange(&sums[blockIdx.x], own, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        asm volatile("" ::"v"(was) : "memory");
        s_last = __hip_atomic_fetch_add(count, (uint64_t)1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint64_t)(parts - 1);
    }
    __syncthreads();
    if (!s_last) return;
    if (w == 0) {
        const uint64_t t = lane < parts ? __hip_atomic_load(&sums[lane], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) : 0;
        s_part[lane] = t;
        const bool any = __ballot(t != 0) != 0;
        if (lane == 0) s_whole = !any;  // nothing left of p: p itself
    }
    __syncthreads();
    if (s_whole)
        for (int k = 0; k < parts; ++k) {  // as good as never
            const uint64_t t = part_sum(k, true);
            if (tid == 0) s_part[k] = t;
            __syncthreads();
        }
    if (w == 0) {
        const uint64_t t = s_part[lane];
        const uint64_t upto = wave_scan64(t, lane);
        const uint64_t total = (uint64_t)__shfl((unsigned long long)upto, 63, 64);
        const double u = (double)U[N];
        const double g = u > 0.0 ? u * (double)total : 0.0;  // NaN: 0
        uint64_t goal = g < (double)total ? (uint64_t)g : total;
        if (goal >= total) goal = total - 1;  // a number of 1 or more takes the last token that has a weight
        const uint64_t m = __ballot(lane < parts && upto > goal);
        if (lane == 0) {
            __hip_atomic_store(count, (uint64_t)0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            s_pick = total == 0 ? -1 : __builtin_ctzll(m);
            s_out = -1;
        }
        if (total && lane == __builtin_ctzll(m)) s_goal = goal - (upto - t);
    }
    __syncthreads();
    const int k = s_pick;
    if (k >= 0) {
        const bool all = s_whole;
        const uint64_t goal = s_goal;
        const int lo = k * part, hi = min(lo + part, V);
        mark(k);
        uint64_t before = 0;
        for (int at = lo; at < hi; at += DC_TILE) {
            const int i = at + 4 * tid;
            double x[4] = {0.0, 0.0, 0.0, 0.0};
            if (i < hi) weights(lo, i, load4(pr, i, V, wide), qr && !all ? load4(qr, i, V, wide) : none, all, x);
            const uint64_t own = (uint64_t)((x[0] + x[1]) + (x[2] + x[3]));
            const uint64_t upto = wave_scan64(own, lane);
            if (lane == 63) s_sum[w] = upto;
            __syncthreads();
            uint64_t base = before, all4 = 0;
            for (int j = 0; j < DC_THREADS / 64; ++j) {
                if (j < w) base += s_sum[j];
                all4 += s_sum[j];
            }
            base += upto - own;
            if (base <= goal && goal < base + own) {
                uint64_t r = goal - base;
                int j = 0;
                while (j < 3 && r >= (uint64_t)x[j]) r -= (uint64_t)x[j++];
                s_out = i + j;
            }
            before += all4;
            __syncthreads();
            if (before > goal) break;  // the same in every thread
        }
    }
    if (tid == 0) A.tokens[(int64_t)b * (N + 1) + s_len] = s_out;
}

// parts of the vocabulary: blocks enough for the device, on whole tiles. A tile a part where there are few: 16 trees over 50021 tokens
// 12.3 us a call with parts of 4 tiles, 9.4 of 1
int parts_of(int B, int V, int* part) {
    const int tiles = (V + DC_TILE - 1) / DC_TILE;
    int n = std::max(1, std::min({DC_MAX_PARTS, tiles, std::max(1, 2048 / std::max(B, 1))}));
    // at most 8192 tokens a part, which its bits have room for
    n = std::max(n, (tiles + 7) / 8);
    const int per = (tiles + n - 1) / n;
    *part = per * DC_TILE;
    return (tiles + per - 1) / per;
}

}  // namespace

extern "C" {

size_t ea_hip_draft_check_size(const ea_draft_check* a) {
    return a && a->num_seqs > 0 ? (size_t)a->num_seqs * DC_WORK * 8 : 0;
}

int ea_hip_draft_check(const ea_draft_check* a, ea_stream_t stream) {
    if (!a || a->num_seqs < 0 || a->num_seqs > 65535 || a->num_drafts < 0 || a->num_drafts > DC_MAX_NODES) return -1;
    if (a->vocab <= 0 || a->vocab > DC_MAX_VOCAB) return -1;
    if (a->num_seqs == 0) return 0;
    if (!a->probs || !a->uniforms || !a->accepted || !a->tokens || !a->work) return -1;
    if (a->num_drafts > 0 && (!a->drafted || !a->path)) return -1;
    if (a->draft_probs && a->parents) return -1;  // trees are of given tokens
    int part = 0;
    const int parts = parts_of(a->num_seqs, a->vocab, &part);
    hipLaunchKernelGGL(ea_draft_check_kernel, dim3((unsigned)parts, (unsigned)a->num_seqs), dim3(DC_THREADS), 0, (hipStream_t)stream,
                       *a, part);
    return herr(hipGetLastError());
}

}  // extern "C"

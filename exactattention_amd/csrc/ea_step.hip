// What a serving step does before its attention call (gfx950): the step plan (block-table growth,
// slots, positions and visible lengths from the requests' lengths) and the rotary positions of q and k
// with the write into the paged cache. No reference counterpart: the reference's demo leaves its cache
// and its positions to transformers (scripts/spec_decode_demo.py:116-125).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "../../include/exactattn_hip.h"
#include "ea_params.h"

namespace {

int herr(hipError_t e) { return e == hipSuccess ? 0 : -100 - (int)e; }

// ------------------------------------------------------------------------------------------------
// Step plan. Sequence b holds L_b keys in held_b = ceil(L_b / P) pages and takes c_b more:
//   cu_b = sum of c before b, need_b = ceil((L_b + c_b) / P) - held_b, np_b = sum of need before b
//   page i of the new ones of b is free[num_free - 1 - np_b - i] (a stack, its top first)
//   token j of b, at flat index cu_b + j: position L_b + j, its page from the table when it has one
//   there already, else from the stack; its pool row is page P + position % P
// What bounds it is latency: 24 bytes a token leave it, and a step of 125,000 tokens writes 5 MB. So it
// is one launch of a short chain: every block reads the sequences (12 bytes each), sums them up in LDS by
// itself, and takes its share of the padded rows (b, j), whose sequence is a division away, without a
// search (with searches 5.6, 8.3 and 9.0 us for 33 sequences of 1 token, 256 of up to 300 and 1000 of up to 500;
// 3.1, 5.0 and 6.3 so). A row with a token writes all that belongs to it, and the table entry too where it opens a
// page. No block reads what another one writes (new pages come from the stack, not from the table), so
// none waits for another. Every input is checked by each block alike: a step that does not fit leaves
// the table alone and reports why.
// ------------------------------------------------------------------------------------------------
constexpr int SP_THREADS = 1024;
constexpr int SP_MAX_SEQS = 8192;
constexpr int SP_MAX_ROWS = 65536;

__global__ void __launch_bounds__(SP_THREADS) ea_step_plan_kernel(ea_step_plan A, int pshift) {
    extern __shared__ __align__(16) int smem[];
    __shared__ int part[2][SP_THREADS / 64];
    __shared__ int s_status, s_pages;
    const int tid = threadIdx.x, B = A.num_seqs, P = A.page_size, T = A.pad_tokens;
    int* const cu = smem;          // B + 1
    int* const np = cu + B + 1;    // B: counts until the sums are known
    int* const len = np + B;       // B
    int* const row = len + B;      // B
    uint32_t* const seen = (uint32_t*)(row + B);  // a bit per table row
    const int words = (A.table_rows + 31) / 32;
    const int nf = *A.num_free;
    for (int i = tid; i < words; i += SP_THREADS) seen[i] = 0;
    if (tid == 0) s_status = 0;
    __syncthreads();
    const int64_t room = min((int64_t)A.table_width << pshift, (int64_t)A.max_seq_len);
    const int per = (B + SP_THREADS - 1) / SP_THREADS;
    const int b0 = min(tid * per, B), b1 = min(b0 + per, B);
    auto need_of = [&](int64_t L, int64_t c) { return (int)(((L + c + P - 1) >> pshift) - ((L + P - 1) >> pshift)); };
    int bad = 0, st = 0, sp = 0;
    for (int b = b0; b < b1; ++b) {
        const int64_t L = A.seq_len[b], c = A.counts[b];
        const int s = A.slots ? A.slots[b] : b;
        np[b] = 0;
        len[b] = (int)L;
        row[b] = s;
        if (L < 0 || c < 0 || s < 0 || s >= A.table_rows) {
            bad |= EA_PLAN_BAD_INPUT;
            continue;
        }
        if (atomicOr(&seen[s >> 5], 1u << (s & 31)) >> (s & 31) & 1) bad |= EA_PLAN_BAD_INPUT;
        if (L + c > room) bad |= EA_PLAN_TOO_LONG;
        if (c > T) {
            bad |= EA_PLAN_TOO_MANY;
            continue;
        }
        // at most B T tokens, below 2^31, and no more pages than tokens
        np[b] = (int)c;
        st += (int)c;
        sp += need_of(L, c);
    }
    int at = ea::wave_scan_dpp(st), ap = ea::wave_scan_dpp(sp);
    if ((tid & 63) == 63) {
        part[0][tid >> 6] = at;
        part[1][tid >> 6] = ap;
    }
    __syncthreads();
    for (int i = 0; i < tid >> 6; ++i) {
        at += part[0][i];
        ap += part[1][i];
    }
    if (tid == SP_THREADS - 1) {
        if (at > A.max_tokens) bad |= EA_PLAN_TOO_MANY;
        if (nf < 0 || nf > A.free_capacity) bad |= EA_PLAN_BAD_INPUT;
        else if (ap > nf) bad |= EA_PLAN_NO_PAGES;
        cu[B] = at;
        s_pages = ap;
    }
    if (bad) atomicOr(&s_status, bad);
    at -= st;
    ap -= sp;
    for (int b = b0; b < b1; ++b) {
        const int c = np[b], n = need_of(len[b], c);
        cu[b] = at;
        np[b] = ap;
        at += c;
        ap += n;
    }
    __syncthreads();
    const int status = s_status;
    const int total = status ? 0 : cu[B];
    const int64_t g0 = (int64_t)blockIdx.x * SP_THREADS + tid, gs = (int64_t)gridDim.x * SP_THREADS;
    if (g0 == 0) {
        *A.status = status;
        *A.new_num_free = nf - (status ? 0 : s_pages);
    }
    for (int64_t b = g0; b < B; b += gs) A.new_seq_len[b] = len[b] + (status ? 0 : cu[b + 1] - cu[b]);
    const int64_t rows = (int64_t)B * T;
    for (int64_t i = g0; i < rows; i += gs) {
        const int b = (int)((uint32_t)i / (uint32_t)T), j = (int)i - b * T;
        const bool live = !status && j < cu[b + 1] - cu[b];
        const int pos = len[b] + j;
        if (A.kv_len) A.kv_len[i] = live ? pos + 1 : 0;
        if (!live) continue;
        const int held = (int)(((int64_t)len[b] + P - 1) >> pshift), idx = pos >> pshift;
        int32_t* const entry = A.block_table + (int64_t)row[b] * A.table_width + idx;
        int page;
        if (idx < held) {
            page = *entry;
        } else {
            page = A.free_pages[nf - 1 - (np[b] + idx - held)];
            if ((pos & (P - 1)) == 0) *entry = page;
        }
        const int t = cu[b] + j;
        A.dst_rows[t] = ((int64_t)page << pshift) + (pos & (P - 1));
        if (A.positions) A.positions[t] = pos;
        if (A.seq_of) A.seq_of[t] = b;
        if (A.q_rows) A.q_rows[t] = i;
    }
    for (int64_t t = total + g0; t < A.max_tokens; t += gs) {
        A.dst_rows[t] = -1;
        if (A.positions) A.positions[t] = -1;
        if (A.seq_of) A.seq_of[t] = -1;
        if (A.q_rows) A.q_rows[t] = -1;
    }
}

// ------------------------------------------------------------------------------------------------
// Rotary positions. Pair i of a head, (x, y) = elements (i, i + R/2) or (2i, 2i + 1), turns by the angle
// theta = (position on axis(i)) * w_i:  (x cos - y sin, y cos + x sin) * scale, by -theta when inverse,
// which is the transposed rotation and so the gradient's. Elements past R pass unchanged.
// The angle is taken in half turns in fp64 (a position of 2^20 at frequency 1 still has an error below
// 2^-32 of a turn) and the rotation in fp64 too, rounded once to the output type: 8 fp64 operations a pair cost
// less than the pair's 8 bytes of traffic, so the exact form is free here.
// What bounds it is memory: every element is read once and written once. A block takes whole tokens, so
// the sines of a token are computed once for all its heads (LDS), and q, k and v of a token go in one
// launch, k and v straight to their pool rows. 16,384 tokens of 32 q, 8 k and 8 v heads of 128 dims: 88 us, 4.6
// TB/s of the 4.78 that a large copy reaches; 33 tokens 4.2 us, of which a launch alone is about 2 (of a graph of
// 24 launches each).
// ------------------------------------------------------------------------------------------------
constexpr int RT_THREADS = 256;
constexpr int RT_MAX_PAIRS = 128;  // rot_dim at most 256

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

// V = 8: 16-byte accesses throughout (the host has checked strides and alignment); V = 1 (pairs of
// halves) or 2 (adjacent pairs): any stride. A unit is V elements, of a pair's both halves where those
// are apart: unit u of a token is in turn those of its q heads, k heads and v heads. gridDim.y cuts a
// token's units where there are few tokens. The first unit of a thread is loaded ahead of the sines.
template <int V, bool IN32, bool OUT32, bool ADJ>
__global__ void __launch_bounds__(RT_THREADS) ea_rotary_kernel(ea_rotary A, int tpb) {
    extern __shared__ __align__(16) double2 cs[];  // tpb x pairs of (cos, sin) * scale
    const int h = A.rot_dim / 2, d = A.head_dim, tid = threadIdx.x;
    const int64_t t0 = (int64_t)blockIdx.x * tpb;
    const int nt = (int)min((int64_t)tpb, A.num_tokens - t0);
    const int pu = ADJ ? A.rot_dim / V : h / V;  // units of a head that turn, and its other ones
    const int uh = pu + (d - A.rot_dim) / V, uv = d / V;
    const int uq = A.num_q_heads * uh, uk = A.num_kv_heads * uh, ua = uq + uk + (A.v ? A.num_kv_heads * uv : 0);
    struct Unit {
        bool live, turn;
        int c, tk;
        const void* src;
        void* dst;
        int64_t s, o;
        Chunk<V, IN32> a, b;
    };
    auto fetch = [&](int u, Unit& x) __attribute__((always_inline)) {
        x.tk = u / ua;
        int r = u - x.tk * ua;
        const int64_t t = t0 + x.tk;
        const int64_t drow = r >= uq ? (A.dst_rows ? A.dst_rows[t] : t) : (A.q_rows ? A.q_rows[t] : t);
        x.live = drow >= 0 && drow < (r >= uq ? A.pool_rows : A.q_out_rows);
        x.turn = false;
        if (r >= uq + uk) {
            r -= uq + uk;
            const int hd = r / uv;
            x.src = A.v;
            x.dst = A.v_out;
            x.s = t * A.v_tok_stride + hd * A.v_head_stride + (r - hd * uv) * V;
            x.o = drow * A.vo_tok_stride + hd * A.vo_head_stride + (r - hd * uv) * V;
        } else {
            const bool isk = r >= uq;
            if (isk) r -= uq;
            const int hd = r / uh, c = r - hd * uh;
            x.turn = c < pu;
            x.c = c * V;
            const int e = x.turn ? c * V : A.rot_dim + (c - pu) * V;
            x.src = isk ? A.k : A.q;
            x.dst = isk ? A.k_out : A.q_out;
            x.s = (isk ? t * A.k_tok_stride + hd * A.k_head_stride : t * A.q_tok_stride + hd * A.q_head_stride) + e;
            x.o = (isk ? drow * A.ko_tok_stride + hd * A.ko_head_stride : drow * A.qo_tok_stride + hd * A.qo_head_stride) + e;
        }
        if (!x.live) return;
        x.a.load(x.src, x.s);
        if (!ADJ && x.turn) x.b.load(x.src, x.s + h);
    };
    auto finish = [&](Unit& x) __attribute__((always_inline)) {
        if (!x.live) return;
        if (!x.turn) {
            store_as<V, IN32, OUT32>(x.a, x.dst, x.o);
            return;
        }
        const double2* z = cs + x.tk * h;
        Chunk<V, OUT32> y0, y1;
        if constexpr (ADJ) {
#pragma unroll
            for (int i = 0; i < V; i += 2) {
                const double2 q = z[(x.c + i) >> 1];
                const double u0 = x.a.get(i), u1 = x.a.get(i + 1);
                y0.put(i, __fma_rn(u0, q.x, -(u1 * q.y)));
                y0.put(i + 1, __fma_rn(u1, q.x, u0 * q.y));
            }
            y0.store(x.dst, x.o);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const double2 q = z[x.c + i];
                const double u0 = x.a.get(i), u1 = x.b.get(i);
                y0.put(i, __fma_rn(u0, q.x, -(u1 * q.y)));
                y1.put(i, __fma_rn(u1, q.x, u0 * q.y));
            }
            y0.store(x.dst, x.o);
            y1.store(x.dst, x.o + h);
        }
    };
    const int us = gridDim.y * RT_THREADS, u1 = nt * ua;
    int u = blockIdx.y * RT_THREADS + tid;
    Unit x;
    if (u < u1) fetch(u, x);
    for (int i = tid; i < nt * h; i += RT_THREADS) {
        const int tk = i / h, p = i - tk * h;
        const int axis = A.axis_of_pair ? A.axis_of_pair[p] : 0;
        const double pos = (double)((int64_t)A.positions[axis * A.pos_axis_stride + t0 + tk] + A.pos_offset);
        const double w = A.half_turns[p];
        // pos w mod 2 half turns: the product's rounding error comes back by the FMA
        const double y = pos * w, e = __fma_rn(pos, w, -y);
        double sn, cn;
        sincospi((y - 2.0 * rint(0.5 * y)) + e, &sn, &cn);
        cs[i] = make_double2(cn * (double)A.scale, (A.inverse ? -sn : sn) * (double)A.scale);
    }
    __syncthreads();
    if (u < u1) finish(x);
    for (u += us; u < u1; u += us) {
        fetch(u, x);
        finish(x);
    }
}

// Whether an array that the plan writes lies in another of its arrays: its blocks read the inputs while others
// write, and no block waits for another
bool plan_shares_memory(const ea_step_plan& p) {
    struct Range {
        const void* at;
        int64_t bytes;
    };
    const int64_t B = p.num_seqs, N = p.max_tokens, table = (int64_t)p.table_rows * p.table_width;
    const Range r[] = {{p.block_table, 4 * table},  {p.dst_rows, 8 * N},    {p.positions, 4 * N},    {p.seq_of, 4 * N},
                       {p.q_rows, 8 * N},           {p.kv_len, 4 * B * p.pad_tokens}, {p.new_seq_len, 4 * B}, {p.new_num_free, 4},
                       {p.status, 4},  // written up to here
                       {p.seq_len, 4 * B},          {p.counts, 4 * B},      {p.slots, 4 * B},
                       {p.free_pages, 4 * (int64_t)p.free_capacity},        {p.num_free, 4}};
    constexpr int n = sizeof(r) / sizeof(r[0]), written = 9;
    for (int i = 0; i < written; ++i)
        for (int j = i + 1; j < n; ++j) {
            const uintptr_t a = (uintptr_t)r[i].at, b = (uintptr_t)r[j].at;
            if (a && b && r[i].bytes > 0 && r[j].bytes > 0 && a < b + r[j].bytes && b < a + r[i].bytes) return true;
        }
    return false;
}

template <int V, bool ADJ>
void rotary_launch(const ea_rotary& A, dim3 grid, size_t lds, int tpb, hipStream_t st) {
    if (!A.in_fp32) hipLaunchKernelGGL((ea_rotary_kernel<V, false, false, ADJ>), grid, dim3(RT_THREADS), lds, st, A, tpb);
    else if (A.out_fp32)
        hipLaunchKernelGGL((ea_rotary_kernel<V, true, true, ADJ>), grid, dim3(RT_THREADS), lds, st, A, tpb);
    else hipLaunchKernelGGL((ea_rotary_kernel<V, true, false, ADJ>), grid, dim3(RT_THREADS), lds, st, A, tpb);
}

}  // namespace

extern "C" {

int ea_hip_step_plan(const ea_step_plan* p, ea_stream_t stream) {
    if (!p || p->num_seqs < 0 || p->num_seqs > SP_MAX_SEQS || p->max_tokens < 0 || p->pad_tokens < 0) return -1;
    if (p->page_size <= 0 || (p->page_size & (p->page_size - 1))) return -1;
    if (p->table_rows < 0 || p->table_rows > SP_MAX_ROWS || p->table_width < 0 || p->max_seq_len < 0 || p->free_capacity < 0)
        return -1;
    if (!p->num_free || !p->new_num_free || !p->status) return -1;
    if (p->num_seqs > 0 && (!p->seq_len || !p->counts || !p->new_seq_len || !p->block_table)) return -1;
    if (p->max_tokens > 0 && !p->dst_rows) return -1;
    if (p->free_capacity > 0 && !p->free_pages) return -1;
    if (p->num_seqs > 0 && (p->pad_tokens == 0 || (int64_t)p->num_seqs * p->pad_tokens >= (int64_t)1 << 31)) return -1;
    if (plan_shares_memory(*p)) return -1;
    int ps = 0;
    while ((1 << ps) < p->page_size) ++ps;
    // two rows a thread, up to two blocks a CU
    const int64_t work = std::max<int64_t>({(int64_t)p->max_tokens, (int64_t)p->num_seqs * p->pad_tokens, 1});
    const unsigned grid = (unsigned)std::min<int64_t>((work + 2 * SP_THREADS - 1) / (2 * SP_THREADS), 512);
    const size_t lds = ((size_t)4 * p->num_seqs + 1 + (p->table_rows + 31) / 32) * 4;  // at most 136 KB
    if (lds > 60 * 1024) {  // beside the static part
        const hipError_t e = hipFuncSetAttribute((const void*)ea_step_plan_kernel, hipFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)lds);
        if (e != hipSuccess) return herr(e);
    }
    hipLaunchKernelGGL(ea_step_plan_kernel, dim3(grid), dim3(SP_THREADS), lds, (hipStream_t)stream, *p, ps);
    return herr(hipGetLastError());
}

int ea_hip_rotary(const ea_rotary* a, ea_stream_t stream) {
    if (!a || a->num_tokens < 0 || a->num_q_heads < 0 || a->num_kv_heads < 0) return -1;
    const int d = a->head_dim, R = a->rot_dim, h = R / 2;
    if (d <= 0 || d > 256 || R <= 0 || R > d || (R & 1) || h > RT_MAX_PAIRS) return -1;
    if ((a->in_fp32 | 1) != 1 || (a->out_fp32 | 1) != 1 || (a->out_fp32 && !a->in_fp32)) return -2;
    if (a->num_axes <= 0 || (a->num_axes > 1 && !a->axis_of_pair)) return -1;
    if (!(a->scale - a->scale == 0.0f)) return -2;
    if (a->num_tokens == 0 || a->num_q_heads + a->num_kv_heads == 0) return 0;
    if (!a->positions || !a->half_turns || a->pool_rows < 0 || a->q_out_rows < 0) return -1;
    if (a->num_q_heads > 0 && (!a->q || !a->q_out)) return -1;
    if (a->num_kv_heads > 0 && (!a->k || !a->k_out || (a->v && !a->v_out))) return -1;
    // 16-byte accesses: every row of every tensor starts on one
    const int64_t in = a->in_fp32 ? 4 : 8, out = a->out_fp32 ? 4 : 8;
    uintptr_t ptr = 0;
    int64_t si = 0, so = 0;
    if (a->num_q_heads > 0) {
        ptr |= (uintptr_t)a->q | (uintptr_t)a->q_out;
        si |= a->q_tok_stride | a->q_head_stride;
        so |= a->qo_tok_stride | a->qo_head_stride;
    }
    if (a->num_kv_heads > 0) {
        ptr |= (uintptr_t)a->k | (uintptr_t)a->k_out;
        si |= a->k_tok_stride | a->k_head_stride;
        so |= a->ko_tok_stride | a->ko_head_stride;
        if (a->v) {
            ptr |= (uintptr_t)a->v | (uintptr_t)a->v_out;
            si |= a->v_tok_stride | a->v_head_stride;
            so |= a->vo_tok_stride | a->vo_head_stride;
        }
    }
    const bool wide = !(ptr & 15) && !(si & (in - 1)) && !(so & (out - 1)) && !(d & 7) && !((a->adjacent ? R : h) & 7);
    if (!wide && a->adjacent && (d & 1)) return -1;  // the narrow form of adjacent pairs takes two elements at a time
    // A unit is a thread's work, and a block takes whole tokens: where a token has fewer units than the block threads, it
    // takes as many tokens as fill them (1 -> 2 -> 4 a block: 40 units a token, 2000 tokens 6.7 -> 4.8 -> 5.2 us, 4096 10.7 ->
    // 7.4 -> 6.5; 88 units, 4096 tokens 14.3 -> 10.4 -> 11.8), from where there are blocks enough (1000 tokens 4.6 either
    // way). Many tokens take two at least, whose sines are then waited for once (8192 tokens of 256 units 28.5 -> 28.1
    // -> 29.4, 448 50.0 -> 49.3 -> 49.9, 704 75.5 -> 76.0 -> 82.3; 4096 of 448 29.3 -> 30.2), and very many of few units four
    // (16384 of 448 92.6 -> 89.1 -> 87.7, of 704 143.6 -> 141.7 -> 144.2). Few tokens of many units are cut into a block for
    // every 256 units (whole -> cut: 33 tokens of 448 5.8 -> 4.2, 500 7.7 -> 6.5, of 704 10.3 -> 8.7, of 2048 21.5 -> 16.2; but
    // 1000 of 448 10.0 -> 10.5, of 704 14.7 -> 14.4, of 2048 29.3 -> 29.2, and 4096 of 2048 88 -> 101). Times are those of 24
    // launches in a graph, over buffers past the caches' size where they are large.
    const int v = wide ? 8 : (a->adjacent ? 2 : 1);
    const int64_t units = (int64_t)(a->num_q_heads + a->num_kv_heads) * ((a->adjacent ? R : h) + d - R) / v +
                          (a->v ? (int64_t)a->num_kv_heads * d / v : 0);
    int tpb = 1;
    while (a->num_tokens >= 1536 && tpb < 4 && 2 * tpb * units <= RT_THREADS) tpb *= 2;
    if (a->num_tokens >= 8192) tpb = std::max(tpb, a->num_tokens >= 16384 && units <= 512 ? 4 : 2);
    if (units * tpb >= (int64_t)1 << 30) return -1;  // the kernel counts them in 32 bits
    const int64_t slices = a->num_tokens < 768 ? std::min<int64_t>((units + RT_THREADS - 1) / RT_THREADS, 64) : 1;
    const dim3 grid((unsigned)(((int64_t)a->num_tokens + tpb - 1) / tpb), (unsigned)slices);
    const size_t lds = (size_t)tpb * h * 16;
    const hipStream_t st = (hipStream_t)stream;
    if (a->adjacent) {
        if (wide) rotary_launch<8, true>(*a, grid, lds, tpb, st);
        else rotary_launch<2, true>(*a, grid, lds, tpb, st);
    } else {
        if (wide) rotary_launch<8, false>(*a, grid, lds, tpb, st);
        else rotary_launch<1, false>(*a, grid, lds, tpb, st);
    }
    return herr(hipGetLastError());
}

}  // extern "C"

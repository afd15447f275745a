// The multi-row split kernel (ea_mrow.h) on bf16 caches: its variants, and its host side, which the
// 4-bit caches' variants (ea_mrow4.hip) share.
#include <mutex>

#include "ea_mrow.h"

namespace {

// MOD: Params::mods, 0 the plain kernel
template <int RS, int MOD>
const void* mrow_fn(bool small) {
    return small ? (const void*)ea_mrow<RS, 2, 4, MOD> : (const void*)ea_mrow<RS, 4, 8, MOD>;
}
template <int RS>
const void* mrow_fn(bool small, int mod) {
    return mod == 3 ? mrow_fn<RS, 3>(small)
                    : (mod == 2 ? mrow_fn<RS, 2>(small) : (mod ? mrow_fn<RS, 1>(small) : mrow_fn<RS, 0>(small)));
}
template <int RS>
size_t mrow_lds(bool small, int mod) {
    if (mod) return small ? sizeof(MRowModSmem<RS, 2, 4>) : sizeof(MRowModSmem<RS, 4, 8>);
    return small ? sizeof(MRowSmem<RS, 2, 4>) : sizeof(MRowSmem<RS, 4, 8>);
}
// head sizes up to 64 take half the K chunks and 4 channels per lane
bool mrow_small(const Params& P) { return P.g.head_dim <= 64 && P.g.head_dim_v <= 64; }
const void* mrow_fn_for(const Params& P) {
    const bool s = mrow_small(P);
    if (P.ks) return ea_mrow_kv4_fn(P.rb, s, P.mods);
    return P.rb == 4 ? mrow_fn<4>(s, P.mods) : (P.rb == 8 ? mrow_fn<8>(s, P.mods) : mrow_fn<16>(s, P.mods));
}
size_t mrow_lds_for(const Params& P) {
    const bool s = mrow_small(P);
    return P.rb == 4 ? mrow_lds<4>(s, P.mods) : (P.rb == 8 ? mrow_lds<8>(s, P.mods) : mrow_lds<16>(s, P.mods));
}
hipError_t mrow_attrs() {
    static std::once_flag once;
    static hipError_t err = hipSuccess;
    std::call_once(once, [] {
        for (int mod = 0; mod < 4; ++mod)
            for (int small = 0; small < 2; ++small) {
                const void* fns[6] = {mrow_fn<4>(small, mod),           mrow_fn<8>(small, mod),
                                      mrow_fn<16>(small, mod),          ea_mrow_kv4_fn(4, small, mod),
                                      ea_mrow_kv4_fn(8, small, mod), ea_mrow_kv4_fn(16, small, mod)};
                for (const void* f : fns) {
                    hipError_t e =
                        hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(MRowModSmem<16, 4, 8>));
                    if (e != hipSuccess) err = e;
                }
            }
    });
    return err;
}
}  // namespace

int ea::ea_mrow_eligible(const Params& P) {
    const ea_geometry& g = P.g;
    if (P.bt && P.pshift < 4) return 0;  // one page lookup per 16 keys
    if (P.ks) {
        // rows of whole groups, 16 bytes of codes each: the cache's own condition (ea_hip.hip) covers the pointers
        const int64_t st[6] = {g.k_page_stride, g.k_slot_stride, g.k_head_stride, g.v_page_stride, g.v_slot_stride, g.v_head_stride};
        for (int64_t x : st)
            if (x & 31) return 0;
    }
    // 16-byte loads of K rows, loads of CPL channels (8 or 16 bytes) of V rows
    const int cpl = mrow_small(P) ? 4 : 8;
    if (((uintptr_t)P.k & 15) || ((g.k_page_stride | g.k_slot_stride | g.k_head_stride) & 7)) return 0;
    if (((uintptr_t)P.v & (2 * cpl - 1)) || ((g.v_page_stride | g.v_slot_stride | g.v_head_stride | g.head_dim_v) & (cpl - 1)))
        return 0;
    const int64_t lim = (int64_t)1 << 30;
    if (P.rows >= lim || (int64_t)g.max_seq_len + 256 >= lim) return 0;
    if (g.k_slot_stride < 0 || g.v_slot_stride < 0 || 32 * g.k_slot_stride + 256 >= lim || 32 * g.v_slot_stride + 256 >= lim)
        return 0;
    return 1;
}

int ea::ea_mrow_slots(const Params& P, int* slots) {
    // blocks resident on the current device at once, cached per device and kernel
    static std::mutex mu;
    static int cache[64][48] = {};
    hipError_t e = mrow_attrs();
    if (e != hipSuccess) return -100 - (int)e;
    int dev = 0;
    if ((e = hipGetDevice(&dev)) != hipSuccess) return -100 - (int)e;
    const int ki = (P.rb == 4 ? 0 : (P.rb == 8 ? 1 : 2)) + (mrow_small(P) ? 3 : 0) + 6 * P.mods + (P.ks ? 24 : 0);
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 0 || dev >= 64) return -1;
    if (!cache[dev][ki]) {
        int cus = 0, per = 0;
        if ((e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev)) != hipSuccess) return -100 - (int)e;
        if ((e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, mrow_fn_for(P), MR_THREADS, mrow_lds_for(P))) !=
            hipSuccess)
            return -100 - (int)e;
        cache[dev][ki] = (cus > 0 ? cus : 1) * (per > 0 ? per : 1);
    }
    *slots = cache[dev][ki];
    return 0;
}

int ea::ea_launch_mrow(const Params& P, hipStream_t st) {
    hipError_t e = mrow_attrs();
    if (e != hipSuccess) return -100 - (int)e;
    Params Pc = P;
    void* args[] = {&Pc};
    const dim3 grid = P.dq_stream ? dim3((unsigned)P.dq_blocks) : dim3((unsigned)(P.nseg * P.nrb), (unsigned)P.nsplit);
    e = hipLaunchKernel(mrow_fn_for(P), grid, dim3(MR_BX, MR_THREADS / MR_BX), args, mrow_lds_for(P), st);
    return e == hipSuccess ? 0 : -100 - (int)e;
}

// The split kernel of 4-bit caches: its variants and its host side.
#include <mutex>

#include "ea_four.h"

namespace {

// MOD: Params::mods, 0 the plain kernel; 4 groups of channels a lane's loads, or 2 where V has no more
template <int RS, int MOD>
const void* four_fn(bool small) {
    return small ? (const void*)ea_four<RS, 2, MOD> : (const void*)ea_four<RS, 4, MOD>;
}
template <int RS>
const void* four_fn(bool small, int mod) {
    return mod == 3 ? four_fn<RS, 3>(small) : (mod == 2 ? four_fn<RS, 2>(small) : (mod ? four_fn<RS, 1>(small) : four_fn<RS, 0>(small)));
}
bool four_small(const Params& P) { return P.g.head_dim_v <= 64; }
const void* four_fn_for(const Params& P) {
    return P.rb == 4 ? four_fn<4>(four_small(P), P.mods) : four_fn<8>(four_small(P), P.mods);
}
size_t four_lds(const Params& P) {
    const bool s = four_small(P);
    return P.rb == 4 ? (s ? sizeof(FourSmem<4, 2>) : sizeof(FourSmem<4, 4>)) : (s ? sizeof(FourSmem<8, 2>) : sizeof(FourSmem<8, 4>));
}
hipError_t four_attrs() {
    static std::once_flag once;
    static hipError_t err = hipSuccess;
    std::call_once(once, [] {
        for (int mod = 0; mod < 4; ++mod)
            for (int small = 0; small < 2; ++small)
                for (const void* f : {four_fn<4>(small, mod), four_fn<8>(small, mod)}) {
                    const hipError_t e =
                        hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(FourSmem<8, 4>));
                    if (e != hipSuccess) err = e;
                }
    });
    return err;
}

}  // namespace

int ea::ea_four_eligible(const Params& P) {
    const ea_geometry& g = P.g;
    const int64_t lim = (int64_t)1 << 29;  // a waiting pair keeps its key in 29 bits
    if (P.rows >= lim || (int64_t)g.max_seq_len + 256 >= lim) return 0;
    return g.k_slot_stride >= 0 && 32 * g.k_slot_stride + 256 < lim;
}

int ea::ea_four_slots(const Params& P, int* slots) {
    // blocks resident on the current device at once, cached per device and kernel
    static std::mutex mu;
    static int cache[64][16] = {};
    hipError_t e = four_attrs();
    if (e != hipSuccess) return -100 - (int)e;
    int dev = 0;
    if ((e = hipGetDevice(&dev)) != hipSuccess) return -100 - (int)e;
    const int ki = (P.rb == 4 ? 0 : 1) + (four_small(P) ? 2 : 0) + 4 * P.mods;
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 0 || dev >= 64) return -1;
    if (!cache[dev][ki]) {
        int cus = 0, per = 0;
        if ((e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev)) != hipSuccess) return -100 - (int)e;
        if ((e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, four_fn_for(P), F4_THREADS, four_lds(P))) != hipSuccess)
            return -100 - (int)e;
        cache[dev][ki] = (cus > 0 ? cus : 1) * (per > 0 ? per : 1);
    }
    *slots = cache[dev][ki];
    return 0;
}

int ea::ea_launch_four(const Params& P, hipStream_t st) {
    hipError_t e = four_attrs();
    if (e != hipSuccess) return -100 - (int)e;
    Params Pc = P;
    void* args[] = {&Pc};
    const dim3 grid = P.dq_stream ? dim3((unsigned)P.dq_blocks) : dim3((unsigned)(P.nseg * P.nrb), (unsigned)P.nsplit);
    e = hipLaunchKernel(four_fn_for(P), grid, dim3(F4_THREADS), args, four_lds(P), st);
    return e == hipSuccess ? 0 : -100 - (int)e;
}

// The split kernel of 4-bit caches: its variants and its host side. Compiled without the machine-level hoisting of loop invariants, as
// ea_prefill_mod.hip: with it blocks of 4 rows spill 28 registers (10 without), those of 16 rows 20 (none). A step of 32 ragged
// sequences to 4096 keys 64.4 us with it, 60.5 without, 8 drafted tokens of 8 x 16K 123 and 114, a chunk of 1500 tokens 576 and 564; 8
// sequences of 30000 to 131072 keys, in blocks of 2 rows, 172.6 and 173.6.
#include <algorithm>
#include <mutex>

#include "ea_four.h"

namespace {

// MOD: Params::mods, 0 the plain kernel; NG: V's groups of 32 channels, 2 also for 1; WR: waves with rows of their own
struct Four {
    const void* fn;
    size_t lds;
};
template <int RS, int NG, int WR>
Four four_of(int mod) {
    const void* const fn[4] = {(const void*)ea_four<RS, NG, 0, WR>, (const void*)ea_four<RS, NG, 1, WR>, (const void*)ea_four<RS, NG, 2, WR>,
                               (const void*)ea_four<RS, NG, 3, WR>};
    return {fn[mod], sizeof(FourSmem<RS, NG, WR>)};
}
template <int RS, int WR>
Four four_of(int ng, int mod) {
    return ng == 4 ? four_of<RS, 4, WR>(mod) : (ng == 3 ? four_of<RS, 3, WR>(mod) : four_of<RS, 2, WR>(mod));
}
constexpr int FOUR_RB[3] = {2, 4, 16};  // row blocks
Four four_of(int rb, int ng, int mod) { return rb == 2 ? four_of<2, 1>(ng, mod) : (rb == 4 ? four_of<4, 1>(ng, mod) : four_of<4, 4>(ng, mod)); }
int four_ng(const Params& P) { return std::max(2, (P.g.head_dim_v + 31) >> 5); }
Four four_of(const Params& P) { return four_of(P.rb, four_ng(P), P.mods); }
hipError_t four_attrs() {
    static std::once_flag once;
    static hipError_t err = hipSuccess;
    std::call_once(once, [] {
        for (int rb : FOUR_RB)
            for (int ng = 2; ng <= 4; ++ng)
                for (int mod = 0; mod < 4; ++mod) {
                    const Four f = four_of(rb, ng, mod);
                    const hipError_t e = hipFuncSetAttribute(f.fn, hipFuncAttributeMaxDynamicSharedMemorySize, (int)f.lds);
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
    static int cache[64][36] = {};
    hipError_t e = four_attrs();
    if (e != hipSuccess) return -100 - (int)e;
    int dev = 0;
    if ((e = hipGetDevice(&dev)) != hipSuccess) return -100 - (int)e;
    const Four f = four_of(P);
    const int ki = (P.rb == 2 ? 0 : (P.rb == 4 ? 1 : 2)) + 3 * (four_ng(P) - 2) + 9 * P.mods;
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 0 || dev >= 64) return -1;
    if (!cache[dev][ki]) {
        int cus = 0, per = 0;
        if ((e = hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev)) != hipSuccess) return -100 - (int)e;
        if ((e = hipOccupancyMaxActiveBlocksPerMultiprocessor(&per, f.fn, F4_THREADS, f.lds)) != hipSuccess)
            return -100 - (int)e;
        cache[dev][ki] = (cus > 0 ? cus : 1) * (per > 0 ? per : 1);
    }
    *slots = cache[dev][ki];
    return 0;
}

int ea::ea_launch_four(const Params& P, hipStream_t st) {
    hipError_t e = four_attrs();
    if (e != hipSuccess) return -100 - (int)e;
    const Four f = four_of(P);
    Params Pc = P;
    void* args[] = {&Pc};
    const dim3 grid = P.dq_stream ? dim3((unsigned)P.dq_blocks) : dim3((unsigned)(P.nseg * P.nrb), (unsigned)P.nsplit);
    e = hipLaunchKernel(f.fn, grid, dim3(F4_THREADS), args, f.lds, st);
    return e == hipSuccess ? 0 : -100 - (int)e;
}

// The multi-row split kernel on caches held in 4 bits (ea_kv4.h): its variants.
#include "ea_mrow.h"

namespace {
template <int RS, int MOD>
const void* fn(bool small) {
    return small ? (const void*)ea_mrow<RS, 2, 4, MOD, true> : (const void*)ea_mrow<RS, 4, 8, MOD, true>;
}
template <int RS>
const void* fn(bool small, int mods) {
    return mods == 3 ? fn<RS, 3>(small) : (mods == 2 ? fn<RS, 2>(small) : (mods ? fn<RS, 1>(small) : fn<RS, 0>(small)));
}
}  // namespace

const void* ea::ea_mrow_kv4_fn(int rb, bool small, int mods) {
    return rb == 4 ? fn<4>(small, mods) : (rb == 8 ? fn<8>(small, mods) : fn<16>(small, mods));
}

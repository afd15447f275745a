// ea_pf_main's variants with score modifications. Compiled without the machine-level hoisting of loop invariants
// (build.py): with it the constants of the whole item leave its loop, and come back from scratch in the tile
// loop (30 registers spilled with a bias). 2500 capped causal tokens, 16/8 heads: 715 us a step with
// neither the item loop nor the flag, 682 with either alone, 670 with both; packed documents of 4096 tokens
// 388 -> 377.
#include "ea_pf_main.h"

const void* ea::ea_pf_mod_fn(int mods) {
    return mods == 3 ? (const void*)ea_pf_main<8, false, 3>
                     : (mods == 2 ? (const void*)ea_pf_main<8, false, 2> : (const void*)ea_pf_main<8, false, 1>);
}

// The keys a query token sees: one set, which every tier attends, on the device and on the host.
#pragma once
#include <limits.h>
#include <stdint.h>

#ifdef __HIPCC__
#include <hip/hip_runtime.h>
#define EA_KEYS_HD __host__ __device__
#else
#define EA_KEYS_HD
#endif

namespace ea {

// The visible keys of a query token, the set every tier attends: the prefix n < Lc with
// Lc = min(kv_len, seq_len) (0 when kv_len < 0), and the tree keys tree_base + i (bit i of the tree
// mask) at or past Lc and below seq_len, so a key in both counts once. vis_tree_bits keeps those
// tree bits; the prefix clip is the caller's. Host and device.
EA_KEYS_HD inline uint64_t vis_tree_bits(uint64_t mask, int64_t tb, int64_t Lc, int64_t slen) {
    int64_t lo = Lc - tb, hi = slen - tb;  // keep bits i with lo <= i < hi
    lo = lo < 0 ? 0 : (lo > 64 ? 64 : lo);
    hi = hi < 0 ? 0 : (hi > 64 ? 64 : hi);
    if (hi <= lo) return 0;
    const uint64_t below_hi = hi >= 64 ? ~0ull : ((1ull << hi) - 1);
    const uint64_t below_lo = lo >= 64 ? ~0ull : ((1ull << lo) - 1);
    return mask & below_hi & ~below_lo;
}
EA_KEYS_HD inline int64_t vis_prefix(int64_t kv_len, int64_t slen) {
    return kv_len < 0 ? 0 : (kv_len < slen ? kv_len : slen);
}

// A row's visible keys, listed: the prefix [begin, begin + npre), then the tree keys outside it in
// bit order. With MOD false begin is 0.
struct RowKeys {
    int64_t begin, npre, tb;
    uint64_t mask;
    EA_KEYS_HD int64_t count() const { return npre + __builtin_popcountll(mask); }
    EA_KEYS_HD int64_t key(int64_t j) const {
        if (j < npre) return begin + j;
        uint64_t m = mask;
        for (int64_t c = j - npre; c > 0; --c) m &= m - 1;
        return tb + __builtin_ctzll(m);
    }
};
// kv_begin: the row's first prefix key (vis_begin). Tree keys below it count as tree keys.
EA_KEYS_HD inline RowKeys row_keys(int64_t kv_begin, int64_t kv_len, int64_t slen, uint64_t mask, int64_t tb) {
    RowKeys r;
    const int64_t L = vis_prefix(kv_len, slen);
    r.begin = kv_begin < L ? kv_begin : L;
    r.npre = L - r.begin;
    r.tb = tb;
    r.mask = vis_tree_bits(mask, tb, r.begin == 0 || r.npre > 0 ? L : 0, slen);
    if (r.begin > 0 && r.npre > 0) {
        // the bits below the prefix too: those of keys under begin
        const int64_t hi = r.begin - tb;
        const uint64_t below = hi <= 0 ? 0ull : (hi >= 64 ? ~0ull : ((1ull << hi) - 1));
        r.mask |= vis_tree_bits(mask, tb, 0, slen) & below;
    }
    return r;
}

// The range [beg, end) from a row's first visible key to its last one, beg >= 0; (INT_MAX, 0) when it sees none.
// Tree bits of keys below 0 or at or past slen name no key: with one of them as its first key a kernel whose
// tiles start there would read before the sequence's pages, and weigh what it read.
struct KeySpan {
    int beg, end;
};
EA_KEYS_HD inline KeySpan key_span(int kv_begin, int kv_len, int slen, uint64_t mask, int tb) {
    KeySpan s = {INT_MAX, 0};
    const int e = kv_len < slen ? kv_len : slen;
    if (kv_begin < e) s = {kv_begin, e};
    const uint64_t m = mask ? vis_tree_bits(mask, tb, 0, slen) : 0ull;
    if (m) {
        const int lo = tb + __builtin_ctzll(m), hi = tb + (63 - __builtin_clzll(m)) + 1;
        s.beg = lo < s.beg ? lo : s.beg;
        s.end = hi > s.end ? hi : s.end;
    }
    return s;
}

}  // namespace ea

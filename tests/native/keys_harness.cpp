// Host build of the key sets (ea_keys.h), for tests/test_keys.py.
#include "../../exactattention_amd/csrc/ea_keys.h"

extern "C" {

void h_key_span(int kv_begin, int kv_len, int slen, uint64_t mask, int tb, int* out) {
    const ea::KeySpan s = ea::key_span(kv_begin, kv_len, slen, mask, tb);
    out[0] = s.beg;
    out[1] = s.end;
}

// the row's keys into out (room for cap of them); returns how many there are
int64_t h_row_keys(int64_t kv_begin, int64_t kv_len, int64_t slen, uint64_t mask, int64_t tb, int64_t* out, int64_t cap) {
    const ea::RowKeys r = ea::row_keys(kv_begin, kv_len, slen, mask, tb);
    for (int64_t j = 0; j < r.count() && j < cap; ++j) out[j] = r.key(j);
    return r.count();
}

}  // extern "C"

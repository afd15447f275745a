"""The keys a token sees (exactattention_amd/csrc/ea_keys.h), built for the host from the same header and
checked against the definition: begin <= n < kv_len plus tree_base + i for every set bit i, of 0 <= n <
seq_len. key_span gives the modified kernels their first tile and their last key, row_keys the list
that tier 2 and the host exact tier sum over."""

import ctypes
import os
import random
import subprocess
import tempfile

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))
I32 = (-(1 << 31), (1 << 31) - 1)


@pytest.fixture(scope="module")
def lib():
    out = os.path.join(tempfile.mkdtemp(prefix="ea_keys_"), "libkeys.so")
    subprocess.run(["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-o", out, os.path.join(HERE, "native", "keys_harness.cpp")],
                   check=True)
    L = ctypes.CDLL(out)
    L.h_key_span.argtypes = [ctypes.c_int] * 3 + [ctypes.c_uint64, ctypes.c_int, ctypes.POINTER(ctypes.c_int)]
    L.h_key_span.restype = None
    L.h_row_keys.argtypes = [ctypes.c_int64] * 3 + [ctypes.c_uint64, ctypes.c_int64, ctypes.POINTER(ctypes.c_int64), ctypes.c_int64]
    L.h_row_keys.restype = ctypes.c_int64
    return L


def _set(begin, kv_len, slen, mask, tb):
    return sorted(set(range(begin, min(kv_len, slen))) | {n for i in range(64) if mask >> i & 1 and 0 <= (n := tb + i) < slen})


def _check(L, begin, kv_len, slen, mask, tb):
    want = _set(begin, kv_len, slen, mask, tb)
    got = (ctypes.c_int64 * 512)()
    n = L.h_row_keys(begin, kv_len, slen, mask, tb, got, 512)
    assert n == len(want) and sorted(got[:n]) == want, (begin, kv_len, slen, hex(mask), tb)
    span = (ctypes.c_int * 2)()
    L.h_key_span(begin, kv_len, slen, mask, tb, span)
    assert list(span) == ([want[0], want[-1] + 1] if want else [I32[1], 0]), (begin, kv_len, slen, hex(mask), tb)


def test_random(lib):
    rng = random.Random(3)
    for _ in range(20000):
        slen = rng.choice([0, 1, rng.randrange(200)])
        mask = rng.choice([0, rng.getrandbits(64), 1 << rng.randrange(64), (1 << 64) - 1, rng.getrandbits(64) & rng.getrandbits(64)])
        _check(lib, rng.randrange(220), rng.randrange(-3, 220), slen, mask, rng.randrange(-80, 210))


@pytest.mark.parametrize("tb", [-1, -3, -63, -64, -65, I32[0], I32[0] + 1, I32[1], I32[1] - 63, I32[1] - 64, 99, 100, 36, 37])
@pytest.mark.parametrize("mask", [1, 5, 1 << 63, (1 << 64) - 1, 0xF0])
@pytest.mark.parametrize("begin, kv_len", [(0, 0), (0, 70), (40, 70), (80, 70), (0, -5)])
def test_bits_outside_the_sequence(lib, tb, mask, begin, kv_len):
    """Bits whose key is below 0 or past the sequence name none: the first key is never negative."""
    _check(lib, begin, kv_len, 100, mask, tb)

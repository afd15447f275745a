"""GPU: attention over a 4-bit cache at the edges of what its kernel sums exactly, and NaN and infinities in its pages."""

import numpy as np
import pytest

import kv4_format as f4
from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from gen import bf16
from test_gpu_kv4 import _check, _pool
from test_gpu_parity import _oracle

pytestmark = pytest.mark.gpu


def _bits(codes, scales, d):
    """A pool's values as bf16 bits, NaN as the quiet one."""
    with np.errstate(all="ignore"):
        x = f4.values(codes, scales, d)
        return np.where(np.isnan(x), 0x7FC0, f4.as_bf16(np.where(np.isnan(x), 0.0, x))).astype(np.uint16)


def _pair(q, arrays, bt, kv_len, seq_len):
    """(the problem over a 4-bit cache, the same one over the bf16 cache of its values), on one block table."""
    d = q.shape[-1]
    want = problem.paged(q, _bits(arrays[0], arrays[1], d), _bits(arrays[2], arrays[3], d), bt, kv_len, seq_len, "HND")
    pool = _pool(arrays, d)
    got = {**want, "kv4": pool, "geom": {**want["geom"], **pool.geometry()}}
    del got["k"], got["v"]
    return got, want


# tokens, heads: blocks of 2 rows, of 4, and (512 of them or more) of 16
SHAPES = [(2, 1, 2, 2), (1, 3, 2, 2), (16, 64, 4, 2)]


def _far_groups(rng, B, T, Hkv, grp, d, low, high, cancel=False):
    """Keys whose first groups have scale byte `high`, the last one `low`, and codes at the ends of the sums: 6, -6, both, in
    halves that cancel (`cancel`: all keys), or any. Queries are whole multiples of 2^-24 of their unit, 8 times it the largest, so that their six digits hold
    them whole: 1, which is the digit -16 and a carry, powers of two, and any 8 bits."""
    page, S = 16, 64 + T
    per = -(-S // page)
    pages = B * per
    arrays = f4.random_pool(rng, pages, Hkv, page, d, -2, 2)
    k = arrays[0]
    m = (d - 32) // 2  # bytes of the first groups
    kind = np.where(cancel, 2, rng.integers(0, 4, k.shape[:3]))
    k[..., :m][kind == 0] = 0x77
    k[..., :m][kind == 1] = 0xFF
    half = np.where(np.arange(m) < m // 2, 0x77, 0xFF).astype(np.uint8)
    k[..., :m][kind == 2] = half
    arrays[1][...] = high
    arrays[1][..., -1] = low
    sign = rng.choice([-1.0, 1.0], (B, T, Hkv * grp, d))
    q = np.where(rng.random(sign.shape) < 0.5, 1.0, np.exp2(rng.integers(-24, 1, sign.shape)))
    any8 = rng.integers(1, 256, sign.shape) * np.exp2(rng.integers(-24, -7, sign.shape))
    rows = rng.integers(0, 3, sign.shape[:3])[..., None]
    q = np.where(rows == 0, 1.0, np.where(rows == 1, q * sign, any8 * sign))
    q[..., 0] = 8.0
    q = np.ldexp(q, 126 - high)
    f = q.astype(np.float32)
    assert np.array_equal(f.astype(np.float64), q) and not np.any(f.view(np.uint32) & 0xFFFF)
    bt = rng.permutation(pages).reshape(B, per).astype(np.int32)
    kv = np.broadcast_to(S - T + 1 + np.arange(T), (B, T))
    return _pair((f.view(np.uint32) >> 16).astype(np.uint16), arrays, bt, kv, np.full(B, S))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,T,Hkv,grp", SHAPES)
@pytest.mark.parametrize("cancel", [False, True])
@pytest.mark.parametrize("low,high", [(120, 129), (100, 109), (40, 49), (221, 230)])
def test_scales_as_far_apart_as_sums_are_exact(gpu, B, T, Hkv, grp, d, low, high, cancel):
    """2^9 apart: a digit's sum reaches 3/4 of 2^24 of its smallest unit, and no pair takes the exact path."""
    rng = np.random.default_rng(1000 * d + 10 * low + T)
    st = _check(_far_groups(rng, B, T, Hkv, grp, d, low, high, cancel), "fp32")
    assert st["slow_path_scores"] == 0, st


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("B,T,Hkv,grp", SHAPES)
@pytest.mark.parametrize("low,high", [(120, 130), (119, 129), (99, 109), (39, 48), (222, 231)])
def test_scales_past_that(gpu, B, T, Hkv, grp, d, low, high):
    """2^10 apart, or scales where fp32's ends come near: pairs take the exact path."""
    rng = np.random.default_rng(1000 * d + 10 * low + T)
    pair = _far_groups(rng, B, T, Hkv, grp, d, low, high)
    if B * T > 64:  # as many rows as blocks of 16 take, and fewer of their pairs
        pair = tuple({**p, "kv_len": np.minimum(p["kv_len"], 9)} for p in pair)
    st = _check(pair, "fp32")
    assert st["slow_path_scores"] > B * T * Hkv * grp, st


@pytest.mark.parametrize("B,T,Hkv,grp", SHAPES + [(1, 70, 2, 2)])
@pytest.mark.parametrize("which,byte", [(1, 255), (3, 255), (1, 254), (3, 253)])
@pytest.mark.parametrize("where", ["among the tokens", "hidden", "past the end", "before the window"])
def test_numbers_that_are_none_in_a_page_that_is_read(gpu, B, T, Hkv, grp, which, byte, where):
    """A NaN scale, or values past the largest bf16, of one key, in K (which 1) or V (3): a domain error for the rows that see it and for
    no others, whose bits do not change; where rows end before it, in a slot past the sequence, and before a window, for none."""
    rng = np.random.default_rng(100 * T + 10 * which + byte)
    d, page, Hq = 128, 16, Hkv * grp
    S = T + 78  # no multiple of 16
    per = -(-(S + 1) // page)
    arrays = f4.random_pool(rng, B * per, Hkv, page, d, -2, 2)
    bt = rng.permutation(B * per).reshape(B, per).astype(np.int32)
    kv = np.broadcast_to(S - T + 1 + np.arange(T), (B, T)).copy()
    q = bf16(rng, (B, T, Hq, d), "normal", 1.0)
    b, head = B - 1, Hkv - 1
    pos = {"among the tokens": S - T + T // 2, "hidden": S - T - 1, "past the end": S, "before the window": 35}[where]
    if where == "hidden":
        kv = np.minimum(kv, pos)
    mods = hip.ScoreMods(window=40) if where == "before the window" else None
    bad = [a.copy() for a in arrays]
    at = (bt[b, pos // page], head, pos % page)
    bad[which][at + (2,)] = byte
    bad[which - 1][at] = 0x77
    assert not np.isfinite(f4.values(bad[which - 1][at], bad[which][at], d)).all()
    ab = default_alpha_bits(d)
    got, flags, _ = hip.attention_problem(_pair(q, bad, bt, kv, np.full(B, S))[0], None, alpha_bits=ab, fallback=False, device="cuda:0",
                                          mods=mods)
    sees = np.zeros((B, T, Hq), bool)
    if where == "among the tokens":
        sees[b, :, head * grp:(head + 1) * grp] = (kv[b] > pos)[:, None]
        assert sees.any()
    flags = flags.reshape(B, T, Hq)
    assert np.array_equal(flags, np.where(sees, 2, 0))
    clean = _pair(q, arrays, bt, kv, np.full(B, S))[1]
    if mods is None:
        want = _oracle(clean, ab, "bf16")[0]
    else:
        want, wf, _ = hip.attention_problem(clean, None, alpha_bits=ab, kernel="general", mods=mods, device="cuda:0")
        assert not wf.any()
    assert np.array_equal(got[~sees], want[~sees])

"""GPU: attention over a cache held in 4 bits. Its values are bf16 numbers, so the bar is equal bits: with the oracle on
those values, and with the bf16 kernels where score modifications are on."""

import ctypes

import numpy as np
import pytest

import kv4_format as f4
from exactattention_amd import hip, problem
from exactattention_amd.formats import ExactAttentionDomainError, default_alpha_bits
from exactattention_amd.kv4 import KV4Pool
from gen import bf16
from test_gpu_parity import _oracle

pytestmark = pytest.mark.gpu


def _pool(arrays, d):
    import torch
    return KV4Pool.of(*(torch.from_numpy(a).cuda() for a in arrays), head_dim=d)


def _problem(rng, B, T, Hq, Hkv, S, d, page=16, kind="normal", arrays=None, kv_len=None, lo=-3, hi=3, qscale=1.0, tree=None):
    """(the problem over a 4-bit cache, the same one over the bf16 cache of its values)."""
    per = -(-S // page)
    pages = B * per + 2
    arrays = f4.random_pool(rng, pages, Hkv, page, d, lo, hi) if arrays is None else arrays
    bt = rng.permutation(pages)[:B * per].reshape(B, per).astype(np.int32)
    q = bf16(rng, (B, T, Hq, d), kind, qscale)
    kv_len = np.broadcast_to(S - T + 1 + np.arange(T), (B, T)) if kv_len is None else kv_len
    kw = {} if tree is None else dict(tree_mask=tree[0], tree_base=tree[1])
    with np.errstate(all="ignore"):
        k, v = (f4.values(arrays[i], arrays[i + 1], d) for i in (0, 2))
        bits = [np.where(np.isnan(x), 0x7FC0, f4.as_bf16(np.where(np.isnan(x), 0.0, x))).astype(np.uint16) for x in (k, v)]
    want = problem.paged(q, *bits, bt, kv_len, np.full(B, S), "HND", **kw)
    pool = _pool(arrays, d)
    got = {**want, "kv4": pool, "geom": {**want["geom"], **pool.geometry()}}
    del got["k"], got["v"]
    return got, want


def _check(pair, out="bf16", splits=0, **kw):
    ab = default_alpha_bits(pair[1]["geom"]["head_dim"])
    want, wflags = _oracle(pair[1], ab, out)
    got, flags, st = hip.attention_problem(pair[0], None, out, splits, alpha_bits=ab, device="cuda:0", **kw)
    assert not flags.any() and not np.any(wflags)
    assert np.array_equal(got, want), st
    return st


def test_every_value(gpu):
    """Each element under each scale byte, against the table; pad columns are not returned."""
    import torch
    c = np.broadcast_to(np.arange(256, dtype=np.uint8), (256, 1, 16, 256)).reshape(256, 1, 16, 256)[..., :32].copy()
    c[:, 0, :, :16] = np.arange(256, dtype=np.uint8).reshape(16, 16)
    s = np.broadcast_to(np.arange(256, dtype=np.uint8)[:, None, None, None], (256, 1, 16, 2)).copy()
    pool = _pool((c, s, c.copy(), s.copy()), 40)
    k, v = pool.values()
    assert k.shape == (256, 1, 16, 40) and k.dtype == torch.bfloat16
    want = f4.values(c, s, 40)
    for x in (k, v):
        got = x.cpu().double().numpy()
        assert np.array_equal(got, want, equal_nan=True)
        assert np.array_equal(np.signbit(got[~np.isnan(want)]), np.signbit(want[~np.isnan(want)]))


@pytest.mark.parametrize("T,grp", [(1, 1), (1, 2), (1, 4), (3, 2), (1, 8), (5, 1), (9, 2), (1, 16)])
@pytest.mark.parametrize("d", [8, 32, 64, 72, 96, 128])
def test_rows_and_head_sizes(gpu, T, grp, d):
    """1 to 18 rows a segment, heads that fill their groups in part, keys at the edges of steps, tiles and pages."""
    rng = np.random.default_rng(1000 * T + 10 * grp + d)
    for S, page, splits in ((T, 16, 0), (15 + T, 16, 0), (17 + T, 64, 0), (63 + T, 16, 0), (64 + T, 32, 0), (777, 64, 3)):
        st = _check(_problem(rng, 2, T, 2 * grp, 2, max(S, T), d, page), "fp32" if S & 2 else "bf16", splits)
        assert st["mrow_kernel_rows"] == 2 * T * 2 * grp


@pytest.mark.parametrize("B,T,grp", [(70, 1, 8), (70, 9, 1), (40, 17, 1), (300, 1, 2)])
@pytest.mark.parametrize("d", [64, 128])
def test_wide_blocks_and_many_units(gpu, B, T, grp, d):
    """Segments of 8 to 17 rows, and grids past one round of blocks."""
    rng = np.random.default_rng(B + T + d)
    for S in (T, 65 + T, 200):
        _check(_problem(rng, B, T, 2 * grp, 2, S, d), "fp32" if S & 1 else "bf16")


@pytest.mark.parametrize("T,d", [(64, 128), (100, 128), (33, 128), (70, 64), (40, 96)])
def test_prompt_chunks(gpu, T, d):
    """Prompt chunks behind a prefix."""
    rng = np.random.default_rng(T + d)
    for S in (T, T + 100):
        _check(_problem(rng, 2, T, 4, 2, S, d))


@pytest.mark.parametrize("B,T,Hkv,grp", [(32, 64, 8, 4), (64, 13, 8, 1), (130, 31, 4, 1)])
@pytest.mark.parametrize("d", [64, 96, 128])
def test_waves_with_rows_of_their_own(gpu, B, T, Hkv, grp, d):
    """Blocks of 16 rows: full ones, ones of 13 rows whose last wave has one, a second one of 15; keys that end inside tiles, and
    sequences that end inside the prompt."""
    rng = np.random.default_rng(B + T + d)
    S = T + 90
    kv = np.minimum(np.broadcast_to(S - T + 1 + np.arange(T), (B, T)), rng.integers(0, S + 1, (B, 1)))
    _check(_problem(rng, B, T, Hkv * grp, Hkv, S, d, 32, kv_len=kv))


@pytest.mark.parametrize("T", [2, 64])
def test_scales_far_apart(gpu, T):
    """Groups 2^60 apart, beyond what the sums hold exactly, subnormal values, and groups of zeros."""
    rng = np.random.default_rng(T)
    for lo, hi in ((-30, 30), (-126, -100), (-127, -126)):
        pair = _problem(rng, 1, T, 4, 2, 130, 128, lo=lo, hi=hi, qscale=0.25 if hi > 0 else 1.0)
        if hi < 0:
            _check(pair)
            continue
        # logits past the oracle's domain (weights more than 2^20 binades apart): what the bf16 cache of the values gives
        got, want = (hip.attention_problem(p, None, alpha_bits=default_alpha_bits(128), device="cuda:0", fallback=False) for p in pair)
        assert np.array_equal(got[1], want[1]) and np.array_equal(got[0], want[0])
    _check(_problem(rng, 1, T, 4, 2, 130, 128, lo=-40, hi=2))
    arrays = f4.random_pool(rng, 20, 2, 16, 128, -2, 2)
    for i in (0, 2):
        arrays[i][:, :, ::3] = 0
    _check(_problem(rng, 1, T, 4, 2, 130, 128, arrays=arrays))


@pytest.mark.parametrize("kind", ["wide", "outlier", "dupes", "subnormal"])
@pytest.mark.parametrize("T", [1, 5, 70])
def test_query_kinds(gpu, kind, T):
    rng = np.random.default_rng(T)
    _check(_problem(rng, 2, T, 4, 2, 300, 128, kind=kind))


@pytest.mark.parametrize("T", [1, 4, 64])
def test_lengths_and_rows_without_keys(gpu, T):
    """Rows that see nothing, one key, and sequences of length 0 and 1, in one batch."""
    rng = np.random.default_rng(T)
    S = 200
    kv = rng.integers(0, S + 1, (4, T))
    kv[0], kv[1], kv[2, 0] = 0, 1, 0
    pair = _problem(rng, 4, T, 4, 2, S, 128, kv_len=kv)
    for p in pair:
        p["seq_len"] = np.array([0, 1, S, 77], np.int32)
    _check(pair)


@pytest.mark.parametrize("T", [1, 2, 70])
def test_numbers_that_are_none(gpu, T):
    """A NaN scale, and values past the largest bf16, in keys that rows see are domain errors for those rows alone; the same in keys
    that no row sees, in K or in V, change nothing."""
    rng = np.random.default_rng(T)
    S = 140
    for which, byte in ((1, 255), (3, 255), (1, 254), (3, 253)):
        arrays = f4.random_pool(rng, 11, 2, 16, 128, -2, 2)
        pair = _problem(rng, 1, T, 4, 2, S, 128, arrays=arrays)
        key = S - T - 1  # the last key before the tokens' own
        page = int(pair[1]["block_table"][0, key // 16])
        arrays[which][page, 1, key % 16, 2] = byte
        arrays[which - 1][page, 1, key % 16] = 0x77
        pair = _problem(rng, 1, T, 4, 2, S, 128, arrays=arrays)
        for p in pair:
            p["block_table"] = pair[1]["block_table"]
        pos = int(np.flatnonzero(pair[1]["block_table"][0] == page)[0]) * 16 + key % 16 if page in pair[1]["block_table"][0] else None
        if pos is None or pos >= S:
            continue
        got, flags, _ = hip.attention_problem(pair[0], None, alpha_bits=default_alpha_bits(128), fallback=False, device="cuda:0")
        fl = flags.reshape(1, T, 4)
        sees = pos < pair[1]["kv_len"].reshape(1, T)
        assert np.array_equal(fl[..., 2:] == 2, np.broadcast_to(sees[..., None], (1, T, 2)))
        assert not fl[..., :2].any()
        if sees.any():
            with pytest.raises(ExactAttentionDomainError):
                hip.attention_problem(pair[0], None, alpha_bits=default_alpha_bits(128), device="cuda:0")
        # hidden: the rows end before it
        kv = np.minimum(pair[1]["kv_len"], pos)
        a, b = ({**p, "kv_len": kv} for p in pair)
        clean = {**b, "k": b["k"].copy(), "v": b["v"].copy()}
        clean["k" if which == 1 else "v"][page, 1, key % 16] = 0
        want, _ = _oracle(clean, default_alpha_bits(128), "bf16")
        got, flags, _ = hip.attention_problem(a, None, alpha_bits=default_alpha_bits(128), device="cuda:0")
        assert not flags.any() and np.array_equal(got, want)


def test_tree_masks(gpu):
    rng = np.random.default_rng(5)
    B, T, L = 2, 16, 100
    parents = [[-1] + [int(rng.integers(-1, i)) for i in range(1, T)] for _ in range(B)]
    mask = np.zeros((B, T), np.uint64)
    for b in range(B):
        for i in range(T):
            j = i
            while j >= 0:
                mask[b, i] |= np.uint64(1 << j)
                j = parents[b][j]
    for Hq in (2, 4):
        _check(_problem(rng, B, T, Hq, 2, L + T, 128, kv_len=np.full((B, T), L), tree=(mask, np.full(B, L, np.int32))))


MODS = {"window": dict(window=70), "cap": dict(softcap=12.0), "bias": dict(slopes=True), "all": dict(softcap=20.0, slopes=True, window=90)}


@pytest.mark.parametrize("name", list(MODS))
@pytest.mark.parametrize("T,d", [(1, 128), (6, 64), (80, 128), (70, 96)])
def test_score_modifications(gpu, name, T, d):
    rng = np.random.default_rng(T + d)
    m = dict(MODS[name])
    if m.get("slopes"):
        m["slopes"] = (1.4426950408889634 * 2.0 ** (-2.0 * (np.arange(4) + 1))).astype(np.float32)
    a, b = _problem(rng, 2, T, 4, 2, 240, d, qscale=2.0)
    ab = default_alpha_bits(d)
    want, wf, _ = hip.attention_problem(b, None, alpha_bits=ab, kernel="general", mods=hip.ScoreMods(**m), device="cuda:0")
    got, flags, _ = hip.attention_problem(a, None, alpha_bits=ab, mods=hip.ScoreMods(**m), device="cuda:0")
    assert not flags.any() and not wf.any() and np.array_equal(got, want)


@pytest.mark.parametrize("name", sorted(MODS))
@pytest.mark.parametrize("B,T,Hkv,grp,d", [(16, 64, 4, 2, 128), (80, 14, 8, 1, 64), (6, 90, 6, 4, 96)])
def test_score_modifications_in_wide_blocks(gpu, name, B, T, Hkv, grp, d):
    """Blocks of 16 rows, whose key range counts from their first visible key."""
    rng = np.random.default_rng(B + T + d)
    m = dict(MODS[name])
    if m.get("slopes"):
        m["slopes"] = (1.4426950408889634 * 2.0 ** (-2.0 * (np.arange(Hkv * grp) % 4 + 1))).astype(np.float32)
    a, b = _problem(rng, B, T, Hkv * grp, Hkv, T + 170, d, qscale=2.0)
    ab = default_alpha_bits(d)
    want, wf, _ = hip.attention_problem(b, None, alpha_bits=ab, kernel="general", mods=hip.ScoreMods(**m), device="cuda:0")
    got, flags, _ = hip.attention_problem(a, None, alpha_bits=ab, mods=hip.ScoreMods(**m), device="cuda:0")
    assert not flags.any() and not wf.any() and np.array_equal(got, want)


@pytest.mark.parametrize("T,d", [(1, 128), (4, 72), (64, 128)])
def test_the_other_tiers(gpu, T, d):
    """Every row through the device's second tier, and through the host's exact one."""
    import torch
    rng = np.random.default_rng(T)
    pair = _problem(rng, 1, T, 2, 2, 150, d)
    _check(pair, force_tier2=True)
    _check(pair, "fp32", force_tier2=True)
    ab = default_alpha_bits(d)
    dp = hip.DeviceProblem(pair[0], device="cuda:0")
    hip.launch_hip(dp, ab)
    torch.cuda.synchronize()
    dp.flags.fill_(1)
    dp.out.fill_(0)
    hip.exact_rows(dp, ab)
    assert not bool(dp.flags.any())
    assert np.array_equal(dp.out.cpu().numpy().view(np.uint16), _oracle(pair[1], ab, "bf16")[0])


def test_slot_major_and_contiguous_caches(gpu):
    """The C entry point on other strides than KV4Pool's: K's slots of all heads together, and no block table."""
    import torch
    rng = np.random.default_rng(8)
    lib = hip.load()
    for paged in (True, False):
        B, T, Hq, Hkv, S, d, P = 2, 3, 4, 2, 96, 72, 16
        pair = _problem(rng, B, T, Hq, Hkv, S, d, P)
        pool = pair[0]["kv4"]
        arr = [x.cpu().numpy() for x in (pool.k, pool.k_scales, pool.v, pool.v_scales)]
        w = f4.width(d)
        g = dict(pair[1]["geom"], **pool.geometry())
        slots = P
        if not paged:  # a sequence's pages one after another
            bt = pair[1]["block_table"]
            arr = [np.swapaxes(a[bt], 1, 2).reshape((B, Hkv, -1) + a.shape[3:]) for a in arr]
            slots = arr[0].shape[2]
            g.update(page_size=1, block_table_stride=0, v_page_stride=Hkv * slots * w, v_head_stride=slots * w)
        arr[:2] = [a.transpose(0, 2, 1, 3) for a in arr[:2]]
        g.update(k_page_stride=slots * Hkv * w, k_slot_stride=Hkv * w, k_head_stride=w)
        t = [torch.from_numpy(np.ascontiguousarray(a)).cuda() for a in arr]
        dp = hip.DeviceProblem(pair[0], device="cuda:0")
        gc, o = hip.geometry(g), hip.options(dp, default_alpha_bits(d))
        b = dp.buffers()
        b.k, b.v = t[0].data_ptr(), t[2].data_ptr()
        if not paged:
            b.block_table = None
        x = hip.KV4Args(t[1].data_ptr(), t[3].data_ptr())
        n, ns = ctypes.c_size_t(0), ctypes.c_int32(0)
        assert lib.ea_hip_kv4_workspace_size(ctypes.byref(gc), ctypes.byref(o), None, ctypes.byref(n), ctypes.byref(ns)) == 0
        ws = torch.empty(max(n.value, 256), dtype=torch.uint8, device="cuda")
        rc = lib.ea_hip_attention_kv4(ctypes.byref(gc), ctypes.byref(b), ctypes.byref(o), None, ctypes.byref(x), ws.data_ptr(), n.value,
                                      hip._stream_ptr(torch))
        torch.cuda.synchronize()
        assert rc == 0 and not bool(dp.flags.any())
        assert np.array_equal(dp.out.cpu().numpy().view(np.uint16), _oracle(pair[1], default_alpha_bits(d), "bf16")[0])


@pytest.mark.parametrize("T", [1, 64])
def test_offsets_past_32_bits(gpu, T):
    """Pages past 2^32 elements (and past 2^32 bytes of values) of a large pool."""
    import torch
    rng = np.random.default_rng(3)
    Hkv, P, d, S = 8, 64, 128, 150
    pages = (1 << 33) // (Hkv * P * d) + 40
    small = f4.random_pool(rng, 3, Hkv, P, d, -2, 2)
    pool = KV4Pool(pages, P, Hkv, d, "cuda:0")
    at = [pages - 1, 5, pages - 30]
    few = _pool(small, d)
    for t, a in zip((pool.k, pool.k_scales, pool.v, pool.v_scales), (few.k, few.k_scales, few.v, few.v_scales)):
        t[torch.tensor(at, device="cuda")] = a
    pair = _problem(rng, 1, T, 16, Hkv, S, d, P, arrays=small)
    bt = np.array([[0, 1, 2]], np.int32)
    a = {**pair[0], "kv4": pool, "block_table": np.array([at], np.int32)}
    _check((a, {**pair[1], "block_table": bt}))


def test_captured_and_on_another_stream(gpu):
    """A captured step, replayed on new codes between eager work, and two steps in flight on two streams."""
    import torch
    rng = np.random.default_rng(4)
    ab = default_alpha_bits(128)
    pair = _problem(rng, 2, 3, 4, 2, 500, 128)
    dp = hip.DeviceProblem(pair[0], device="cuda:0")
    other = hip.DeviceProblem(pair[0], device="cuda:0")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        hip.launch_hip(dp, ab)
    hip.launch_hip(other, ab)
    torch.cuda.synchronize()
    want = _oracle(pair[1], ab, "bf16")[0]
    for x in (dp, other):
        assert np.array_equal(x.out.cpu().numpy().view(np.uint16), want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        hip.launch_hip(dp, ab)
    pool = pair[0]["kv4"]
    for i in range(4):
        pool.k.copy_(torch.randint(0, 256, pool.k.shape, dtype=torch.uint8, generator=torch.Generator().manual_seed(i)))
        dp.out.fill_(-1)
        graph.replay()
        hip.launch_hip(other, ab)
        torch.cuda.synchronize()
        assert torch.equal(dp.out, other.out) and not bool(dp.flags.any())
    assert not np.array_equal(dp.out.cpu().numpy().view(np.uint16), want)


def test_the_splits_do_not_change_a_bit(gpu):
    rng = np.random.default_rng(6)
    pair = _problem(rng, 2, 1, 8, 2, 3000, 128)
    want = None
    for splits in (1, 2, 7, 0):
        got, flags, _ = hip.attention_problem(pair[0], None, "fp32", splits, alpha_bits=default_alpha_bits(128), device="cuda:0")
        assert not flags.any() and (want is None or np.array_equal(got, want))
        want = got


@pytest.mark.parametrize("T,grp", [(1, 2), (1, 4), (12, 2)])
def test_logits_on_a_tie(gpu, T, grp):
    """Scores of few bits: products with alpha that lie halfway between two fp32 numbers round to even, and no pair of them takes the
    exact path."""
    rng = np.random.default_rng(T + grp)
    arrays = f4.random_pool(rng, 82, 2, 16, 128, 0, 0)
    pair = _problem(rng, 2, T, 2 * grp, 2, 640, 128, arrays=arrays)
    q = (rng.integers(-6, 7, pair[1]["q"].shape) / 4.0).astype(np.float32)
    bits = (q.view(np.uint32) >> 16).astype(np.uint16)
    for p in pair:
        p["q"] = bits
    ab = default_alpha_bits(128)
    alpha = float(np.array([ab], np.uint32).view(np.float32)[0])
    k = f4.values(arrays[0], arrays[1], 128)  # (pages, heads, slots, d)
    s = np.einsum("bthd,phsd->bthps", q.reshape(2, T, 2, grp, 128)[:, :, :, 0], k)
    p = alpha * s  # exact: 24 and 15 bits
    f = p.astype(np.float32)
    other = np.nextafter(f, np.where(p > f, np.inf, -np.inf).astype(np.float32))
    ties = (p != f) & (p == (f.astype(np.float64) + other.astype(np.float64)) / 2)
    assert ties.sum() > 50
    st = _check(pair)
    assert st["slow_path_scores"] == 0, st

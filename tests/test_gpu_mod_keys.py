"""GPU: score modifications with draft trees, on every kernel: tree bits that name no key (below 0, past the
sequence), and trees together with intervals on the int8 prefill kernel."""

import numpy as np
import pytest

from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from gen import bf16
import mod_oracle as mo

pytestmark = pytest.mark.gpu


def _prob(seed, B, T, Hq, Hkv, d, S, page=0):
    """T tokens a sequence at the end of its keys, S - 9 b of them."""
    rng = np.random.default_rng(seed)
    seq = S - 9 * np.arange(B)
    kv = np.maximum(seq[:, None] - T + 1 + np.arange(T), 0)
    p = problem.contiguous(bf16(rng, (B, T, Hq, d), "normal", 2.0), bf16(rng, (B, Hkv, S, d)), bf16(rng, (B, Hkv, S, d)), kv,
                           seq_len=seq)
    return rng, problem.to_paged(p, page, np.random.default_rng(7), "NHD") if page else p


def _run(p, mods, kernel="auto", force=False, out="bf16"):
    import torch
    ab = default_alpha_bits(p["geom"]["head_dim"])
    dp = hip.DeviceProblem(p, out, 0, "cuda:0", kernel, mods=hip.ScoreMods(**mods))
    dp.out.fill_(-1)
    dp.flags.fill_(9)
    hip.launch_hip(dp, ab, force_tier2=force)
    torch.cuda.synchronize()
    return dp, dp.out.cpu().numpy().view(np.uint32 if out == "fp32" else np.uint16), dp.flags.cpu().numpy()


def _stats(dp):
    return dict(zip(hip.STATS, dp.stats.cpu().numpy().tolist()))


def _want(p, mods, r, out="bf16"):
    """The oracle's row, the bits that name no key taken out of the masks first."""
    g = p["geom"]
    tok = np.arange(len(p["tree_mask"]))
    base = np.asarray(p["tree_base"])[tok // g["num_tokens"]]
    sl = np.asarray(p["seq_len"])[tok // g["num_tokens"]]
    mask = [sum(1 << i for i in range(64) if int(m) >> i & 1 and 0 <= int(b) + i < s) for m, b, s in zip(p["tree_mask"], base, sl)]
    return mo.row(dict(p, tree_mask=np.array(mask, np.uint64)), default_alpha_bits(g["head_dim"]), r, out, mods.get("kv_begin"),
                  mods.get("window", 0), mods.get("slopes"), mods.get("q_pos"), mods.get("softcap", 0.0))


@pytest.mark.parametrize("mods", ["docs", "window", "bias", "cap"])
@pytest.mark.parametrize("T, Hq, Hkv, d, page, kernels", [
    (1, 4, 2, 128, 16, ("auto", "general")), (6, 4, 2, 64, 16, ("auto", "general")), (5, 4, 1, 128, 8, ("auto",)),
    (34, 2, 1, 128, 32, ("prefill", "auto", "general")), (33, 2, 2, 96, 0, ("prefill", "auto")),
])
def test_bits_that_name_no_key(gpu, T, Hq, Hkv, d, page, kernels, mods):
    """Tree bases below 0 and near a sequence's end, with low and high bits set: the set is that of the keys
    there are, in every tier, beside prefixes that are empty, short or start late."""
    import torch
    B, S = 3, 140
    rng, p = _prob(T, B, T, Hq, Hkv, d, S, page)
    p["tree_base"] = np.array([-3, -61, S - 18 - 20], np.int32)
    p["tree_mask"] = rng.integers(0, 1 << 63, B * T, dtype=np.int64).astype(np.uint64) | np.uint64(0x7)
    p["tree_mask"][::5] = 7  # bases -3 and -61: keys below 0 alone
    kv = np.asarray(p["kv_len"]).reshape(B, T).copy()
    kv[:, ::2] = rng.integers(0, 4, kv[:, ::2].shape)
    p["kv_len"] = kv.astype(np.int32).reshape(-1)
    sl = (2.0 ** -np.arange(1, Hq + 1)).astype(np.float32)
    m = {"docs": dict(kv_begin=rng.integers(0, S, (B, T)).astype(np.int32)), "window": dict(window=3),
         "bias": dict(slopes=sl, q_pos=kv + 3, window=70), "cap": dict(softcap=5.0, kv_begin=kv // 2)}[mods]
    rows = B * T * Hq
    some = range(rows) if rows <= 40 else sorted(rng.permutation(rows)[:24].tolist())
    want = {r: _want(p, m, r) for r in some}
    for kernel in kernels:
        for force in (False, True):
            dp, res, fl = _run(p, m, kernel, force)
            assert (fl == 0).all(), (kernel, force)
            if kernel == "prefill":
                assert _stats(dp)["prefill_kernel_rows"] == rows
            for r in some:
                assert np.array_equal(res.reshape(rows, d)[r], want[r]), (kernel, force, r)
    dp.out.fill_(-1)
    dp.flags.fill_(1)  # and the host tier
    hip.exact_rows(dp, default_alpha_bits(d))
    torch.cuda.synchronize()
    assert not bool(dp.flags.any()) and np.array_equal(dp.out.cpu().numpy().view(np.uint16), res)


def test_bits_that_name_no_key_in_shares(gpu):
    """The same on the multi-row kernel's equal-share plan, which counts a unit's tiles from its first key."""
    B, T, Hq, Hkv, d, S = 40, 1, 16, 8, 128, 3000
    rng, p = _prob(2, B, T, Hq, Hkv, d, S, 16)
    p["tree_base"] = rng.integers(-63, -1, B).astype(np.int32)
    p["tree_mask"] = rng.integers(1, 1 << 62, B, dtype=np.int64).astype(np.uint64) | np.uint64(1)
    m = dict(kv_begin=rng.integers(0, 2900, (B, 1)).astype(np.int32), softcap=20.0)
    dp, res, fl = _run(p, m)
    st = _stats(dp)
    assert (fl == 0).all() and st["mrow_kernel_rows"] == B * Hq and st["decode_equal_share_steps"] == 1
    _, other, fl = _run(p, m, "general")
    assert (fl == 0).all() and np.array_equal(res, other)
    for r in (0, B * Hq - 1):
        assert np.array_equal(res.reshape(-1, d)[r], _want(p, m, r))


@pytest.mark.parametrize("d", [128, 72])
def test_trees_and_intervals_on_the_prefill_kernel(gpu, d):
    """Tree keys past the interval, inside it and before its first key, on the int8 kernel, against the definition."""
    B, T, Hq, Hkv, S = 2, 34, 2, 1, 330
    rng, p = _prob(9, B, T, Hq, Hkv, d, S, 16)
    kv = rng.integers(0, S, (B, T)).astype(np.int32)
    begin = np.maximum(kv - rng.integers(0, 150, (B, T)), 0).astype(np.int32)
    begin[:, ::7] = S  # no prefix key: the tree's alone
    p["kv_len"] = kv.reshape(-1)
    p["tree_mask"] = rng.integers(1, 1 << 62, B * T, dtype=np.int64).astype(np.uint64)
    p["tree_mask"][::6] = 0
    p["tree_base"] = np.array([70, 250], np.int32)
    m = dict(kv_begin=begin, slopes=np.array([0.5, 0.02], np.float32), q_pos=kv + 3, softcap=12.0)
    for out in ("bf16", "fp32"):
        dp, res, fl = _run(p, m, "prefill", out=out)
        assert (fl == 0).all() and _stats(dp)["prefill_kernel_rows"] == B * T * Hq
        for r in rng.permutation(B * T * Hq)[:30].tolist() + [0, 1, B * T * Hq - 1]:
            assert np.array_equal(res.reshape(-1, d)[r], _want(p, m, r, out)), (out, r)


@pytest.mark.parametrize("base", [3, 700, 1180])
def test_tiles_between_a_tree_and_the_intervals(gpu, base):
    """One token's tree far before, or past, the intervals of the others: its tiles count as seen, the slicing
    leaves out those before every token's first key and no others."""
    B, T, Hq, Hkv, d, S = 2, 200, 4, 2, 128, 1300
    rng, p = _prob(base, B, T, Hq, Hkv, d, S, 16)
    kv = np.asarray(p["kv_len"]).reshape(B, T)
    p["tree_mask"] = np.zeros(B * T, np.uint64)
    p["tree_mask"][[5, T + 199]] = np.array([1 << 63 | 1, 1 << 40], np.uint64)
    p["tree_base"] = np.full(B, base, np.int32)
    m = dict(kv_begin=np.maximum(kv - 90, 0).astype(np.int32), softcap=9.0)
    dp, res, fl = _run(p, m, "prefill")
    assert (fl == 0).all() and _stats(dp)["prefill_kernel_rows"] == B * T * Hq
    for kernel in ("general", "decode"):
        _, other, f2 = _run(p, m, kernel)
        assert (f2 == 0).all() and np.array_equal(res, other), kernel
    for r in (5 * Hq, 6 * Hq, B * T * Hq - 1):
        assert np.array_equal(res.reshape(-1, d)[r], _want(p, m, r))

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

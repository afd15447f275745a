"""GPU: score modifications through ExactAttentionBackend with the cache's digit tiles."""

import numpy as np
import pytest

from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache
from gen import bf16

pytestmark = pytest.mark.gpu


def _cuda(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x).view(np.int16)).cuda()


def _slopes(Hq):
    return (1.4426950408889634 * 2.0 ** (-8.0 * (np.arange(Hq) + 1) / Hq)).astype(np.float32)


def _general(q, k, v, kv_len, mods, out="bf16", **more):
    """The general kernel's bits on one sequence: q (T, Hq, d), k and v (S, Hkv, d)."""
    import torch
    p = problem.contiguous(q[None], k.transpose(1, 0, 2)[None], v.transpose(1, 0, 2)[None], np.asarray(kv_len)[None])
    p.update(more)
    dp = hip.DeviceProblem(p, out, 0, "cuda:0", "general", mods=hip.ScoreMods(**mods))
    hip.launch_hip(dp, default_alpha_bits(q.shape[-1]))
    torch.cuda.synchronize()
    assert not bool(dp.flags.any())
    return dp.out.cpu().numpy().view(np.uint32 if out == "fp32" else np.uint16)[0]


def test_tiles_are_sliced_for_the_steps_that_read_them(gpu):
    """fp32 outputs under a bias run on the multi-row kernel: a prompt chunk leaves the stale tiles as they are."""
    rng = np.random.default_rng(1)
    Hq, Hkv, d, S = 4, 2, 128, 300
    ab = default_alpha_bits(d)
    c = PagedKVCache(num_pages=40, page_size=16, num_kv_heads=Hkv, head_dim=d, max_seqs=2, max_seq_len=S)
    s = c.add_sequence()
    q, k, v = (bf16(rng, (S, h, d)) for h in (Hq, Hkv, Hkv))
    mods = dict(slopes=_slopes(Hq))
    be = ExactAttentionBackend(c, Hq, None, "fp32", alpha_bits=ab, mods=hip.ScoreMods(**mods))
    out, fl = be.forward(_cuda(q), _cuda(k), _cuda(v), [s], [S])
    be.check_flags(fl)
    assert c.stale[s] == 0
    assert np.array_equal(out.cpu().numpy().view(np.uint32), _general(q, k, v, 1 + np.arange(S), mods, "fp32"))


def test_problem_with_a_digit_cache_and_modifications(gpu):
    """A problem whose launch with a digit cache takes the int8 kernel and without one the multi-row kernel:
    both run, and the bits are the same."""
    import torch
    rng = np.random.default_rng(2)
    B, T, Hq, Hkv, d, S = 2, 96, 16, 8, 128, 2000
    ab = default_alpha_bits(d)
    p = problem.contiguous(bf16(rng, (B, T, Hq, d), "normal", 2.0), bf16(rng, (B, Hkv, S, d)), bf16(rng, (B, Hkv, S, d)),
                           np.broadcast_to(S - T + 1 + np.arange(T), (B, T)))
    dp = hip.DeviceProblem(p, mods=hip.ScoreMods(softcap=20.0))
    dig = hip.KVDigits(dp, (S + 63) // 64)
    at = [torch.full((B,), n, dtype=torch.int32, device="cuda") for n in (0, S)]
    dig.update(dp, *at, S)
    got = []
    for kw in ({}, {"kv_digits": dig}):
        dp.out.fill_(-1)
        dp.stats.zero_()
        hip.launch_hip(dp, ab, **kw)
        torch.cuda.synchronize()
        got.append((dp.out.cpu().numpy(), dict(zip(hip.STATS, dp.stats.tolist()))))
        assert not bool(dp.flags.any())
    assert got[0][1]["mrow_kernel_rows"] == got[1][1]["prefill_kernel_rows"] == B * T * Hq
    assert np.array_equal(got[0][0], got[1][0])

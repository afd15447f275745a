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


MODS = {"window": dict(window=500), "cap": dict(softcap=15.0), "bias": dict(slopes=_slopes(16)),
        "all": dict(softcap=25.0, slopes=_slopes(16), window=700)}


def _reads(be):
    """Whether the backend's latest launch read the cache's digit tiles."""
    import ctypes
    gc, _, o = be._last["args"]
    r = ctypes.c_int32(0)
    assert hip.load().ea_hip_mods_reads_kv_digits(ctypes.byref(gc), ctypes.byref(o), ctypes.byref(be._last["mods"]), ctypes.byref(r)) == 0
    return r.value


@pytest.mark.parametrize("name", list(MODS))
@pytest.mark.parametrize("page", [16, 64])
def test_prompt_chunks_read_the_cached_tiles(gpu, name, page):
    """Prompts in chunks with decode tokens between them, two sequences, one alone, in runs and padded together: the
    int8 kernel on the cache's tiles, those that the appends made stale sliced again, gives the bits of the
    general kernel on the keys themselves."""
    rng = np.random.default_rng(page)
    Hq, Hkv, d = 16, 8, 128
    mods = MODS[name]
    c = PagedKVCache(num_pages=4000 // page, page_size=page, num_kv_heads=Hkv, head_dim=d, max_seqs=3, max_seq_len=2000)
    be = ExactAttentionBackend(c, Hq, None, alpha_bits=default_alpha_bits(d), mods=hip.ScoreMods(**mods))
    c.add_sequence()  # the slots used are 1 and 2
    slots = [c.add_sequence(), c.add_sequence()]
    c.drop_sequence(0)
    hist = {s: [np.zeros((0, Hkv, d), np.uint16)] * 2 for s in slots}
    read = []
    for seqs, counts in ((slots[:1], [900]), (slots[1:], [700]), (slots, [1, 1]), (slots, [400, 400]), (slots, [1, 1]),
                         (slots[::-1], [500, 450]), (slots, [1, 90])):
        n = sum(counts)
        q, k, v = (bf16(rng, (n, h, d), "normal", w) for h, w in ((Hq, 2.0), (Hkv, 1.0), (Hkv, 1.0)))
        out, fl = be.forward(_cuda(q), _cuda(k), _cuda(v), seqs, counts)
        be.check_flags(fl)
        assert not bool(fl.any())
        read.append(_reads(be))
        out, at = out.cpu().numpy().view(np.uint16), 0
        for s, m in zip(seqs, counts):
            hist[s] = [np.concatenate([h, x[at:at + m]]) for h, x in zip(hist[s], (k, v))]
            S = len(hist[s][0])
            want = _general(q[at:at + m], *hist[s], S - m + 1 + np.arange(m), mods)
            assert np.array_equal(out[at:at + m], want), (seqs, counts, s)
            at += m
    assert read[0] == read[1] == read[3] == read[5] == 1 and read[2] == read[4] == 0, read


@pytest.mark.parametrize("window", [0, 2000])
def test_draft_tree_reads_the_cached_tiles(gpu, window):
    """64 draft nodes on a long prefix, capped, with and without a window: trees and intervals on the int8
    kernel and the cache's tiles."""
    rng = np.random.default_rng(window)
    Hq, Hkv, d, L, N = 64, 8, 128, 2940, 64
    c = PagedKVCache(num_pages=200, page_size=16, num_kv_heads=Hkv, head_dim=d, max_seqs=1, max_seq_len=3100)
    be = ExactAttentionBackend(c, Hq, None, alpha_bits=default_alpha_bits(d), mods=hip.ScoreMods(softcap=15.0, window=window))
    s = c.add_sequence()
    k, v = bf16(rng, (L + N, Hkv, d)), bf16(rng, (L + N, Hkv, d))
    c.append(s, k[:L], v[:L])
    q = bf16(rng, (N, Hq, d), "normal", 2.0)
    parents = [-1] + [int(rng.integers(-1 if i % 9 == 0 else max(0, i - 4), i)) for i in range(1, N)]
    out, fl = be.verify_tree(s, q, k[L:], v[L:], parents)
    assert _reads(be) == 1 and (fl == 0).all()
    depth, mask = np.zeros(N, np.int64), np.zeros(N, np.uint64)
    for i, p in enumerate(parents):
        depth[i] = depth[p] + 1 if p >= 0 else 0
        mask[i] = (int(mask[p]) if p >= 0 else 0) | 1 << i
    more = dict(tree_mask=mask, tree_base=np.array([L], np.int32))
    m = dict(softcap=15.0)
    if window:
        m["kv_begin"] = np.clip(L + depth + 1 - window, 0, L)
    assert np.array_equal(out, _general(q, k, v, np.full(N, L), m, **more))

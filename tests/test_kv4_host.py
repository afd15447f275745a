"""The 4-bit cache's refusals and sizes: no GPU."""

import ctypes

import numpy as np
import pytest

import kv4_format as f4
from exactattention_amd import hip
from exactattention_amd.kv4 import KV4Pool
from exactattention_amd.serving import PagedKVCache


def test_format_of_every_bf16_scale():
    """The quantizer restated for the tests: no element is off by more than half a step, and scales are the smallest."""
    rng = np.random.default_rng(0)
    x = rng.standard_normal((200, 64)) * np.exp2(rng.integers(-20, 20, (200, 1)))
    c, s = f4.quantize(x)
    y = f4.values(c, s, 64)
    unit = np.repeat(np.ldexp(1.0, s.astype(int) - 127), 32, -1)
    step = np.where(np.abs(x) < 2 * unit, 0.5, np.where(np.abs(x) < 4 * unit, 1.0, 2.0)) * unit
    assert np.all(np.abs(x - y) <= step / 2)
    top = np.abs(x).reshape(200, 2, 32).max(-1)
    assert np.all(top < 7 * np.ldexp(1.0, s.astype(int) - 127)) and np.all(top >= 3.5 * np.ldexp(1.0, s.astype(int) - 127))


def _cpu(pages=3, heads=2, P=16, d=40):
    import torch
    w = f4.width(d)
    return [torch.zeros((pages, heads, P, n), dtype=torch.uint8) for n in (w // 2, w // 32)] + \
        [torch.zeros((pages, heads, P // 16, n, 16), dtype=torch.uint8) for n in (w // 2, w // 32)]


def test_pool_refusals():
    import torch
    ok = _cpu()
    pool = KV4Pool.of(*ok, head_dim=40)
    assert pool.width == 64 and pool.geometry()["k_head_stride"] == 16 * 64
    for i in range(4):
        for bad in (ok[i][:2], ok[i].int(), ok[i].transpose(1, 2), ok[i][..., :-1]):
            with pytest.raises(ValueError):
                KV4Pool.of(*(bad if j == i else t for j, t in enumerate(ok)), head_dim=40)
    with pytest.raises(ValueError, match="share"):
        KV4Pool.of(ok[0], ok[1], ok[0].view(ok[2].shape), ok[3], head_dim=40)
    with pytest.raises(ValueError, match="multiple of 8"):
        KV4Pool.of(*ok, head_dim=36)
    for P in (8, 24):
        with pytest.raises(ValueError, match="page_size"):
            KV4Pool.of(*_cpu(P=P), head_dim=40)
    for kw in (dict(num_pages=-1), dict(num_kv_heads=0), dict(head_dim=0)):
        with pytest.raises(ValueError):
            KV4Pool(**{**dict(num_pages=1, page_size=16, num_kv_heads=1, head_dim=64, device="cpu"), **kw})
    with pytest.raises(ValueError):
        PagedKVCache(4, 16, 2, 64, 1, 64, device="cpu", bits=4)
    with pytest.raises(ValueError):
        PagedKVCache(4, 16, 2, 64, 1, 64, device="cpu", bits=8)
    assert torch.equal(ok[0], torch.zeros_like(ok[0]))


def _call(geom=None, opt=None, mods=None, ptr=None, scales=(1 << 20, 1 << 20), null=False):
    lib = hip.load()
    d, w, P = 72, 96, 32
    g = dict(num_seqs=1, num_tokens=1, num_q_heads=2, num_kv_heads=1, head_dim=d, head_dim_v=d, q_seq_stride=2 * d, q_tok_stride=2 * d,
             q_head_stride=d, o_seq_stride=2 * d, o_tok_stride=2 * d, o_head_stride=d, k_page_stride=P * w, k_slot_stride=w,
             k_head_stride=P * w, v_page_stride=P * w, v_slot_stride=w, v_head_stride=P * w, page_size=P, block_table_stride=4,
             max_seq_len=64)
    g.update(geom or {})
    o = hip.Options(alpha_bits=0x3F800000, tier2=1, **(opt or {}))
    names = ("q", "k", "v", "seq_len", "kv_len", "block_table", "out", "flags")
    b = hip.Buffers(**{**{n: 1 << 20 for n in names}, **(ptr or {})})
    x = hip.KV4Args(*scales)
    n, ns = ctypes.c_size_t(0), ctypes.c_int32(0)
    rc = lib.ea_hip_kv4_workspace_size(ctypes.byref(hip.geometry(g)), ctypes.byref(o), mods, ctypes.byref(n), ctypes.byref(ns))
    # a workspace too small ends a good call before anything is enqueued
    rc2 = lib.ea_hip_attention_kv4(ctypes.byref(hip.geometry(g)), ctypes.byref(b), ctypes.byref(o), mods, None if null else ctypes.byref(x),
                                   None, 0, None)
    return rc, rc2


def test_c_refusals():
    assert _call() == (0, -2)
    assert _call(null=True)[1] == -1
    for n in ("k_page_stride", "k_slot_stride", "k_head_stride", "v_page_stride", "v_slot_stride", "v_head_stride"):
        assert _call({n: 96 + 16}) == (-1, -1), n
    for n in ("v_page_stride", "v_head_stride"):
        assert _call({n: 96}) == (-1, -1), n
    assert _call(dict(v_slot_stride=192)) == (-1, -1)
    assert _call(dict(k_slot_stride=1 << 24))[1] == -2 and _call(dict(k_slot_stride=1 << 20))[1] == -2
    assert _call(dict(head_dim_v=68)) == (-1, -1)
    assert _call(dict(head_dim=136)) == (-1, -1)
    for opt in (*(dict(kernel=hip.KERNELS[x]) for x in ("prefill", "decode", "general")), dict(timers=1 << 20),
                dict(kv_digits=1 << 20, kv_digits_tiles=1)):
        assert _call(opt=opt) == (-2, -2), opt
    assert _call(dict(page_size=8))[1] == -1
    assert _call(ptr=dict(k=(1 << 20) + 8))[1] == -1
    assert _call(ptr=dict(v=(1 << 20) + 4))[1] == -1
    assert _call(scales=(1 << 20, (1 << 20) + 2))[1] == -1
    assert _call(scales=(None, 1 << 20))[1] == -1 and _call(scales=(1 << 20, None))[1] == -1
    for n in ("q", "k", "v", "seq_len", "kv_len", "out", "flags"):
        assert _call(ptr={n: None})[1] == -1, n
    lib = hip.load()
    assert lib.ea_hip_kv4_values(-1, 64, 0, None, None, None, None) == -1
    assert lib.ea_hip_kv4_values(1, 36, 0, 1 << 20, 1 << 20, 1 << 20, None) == -1
    assert lib.ea_hip_kv4_values(1, 64, 0, None, 1 << 20, 1 << 20, None) == -1
    assert lib.ea_hip_kv4_values(1, 64, 0, 1 << 20, 1 << 20, (1 << 20) + 8, None) == -1
    assert lib.ea_hip_kv4_values(8, 64, 1, 1 << 20, 1 << 20, 1 << 20, None) == -1
    assert lib.ea_hip_kv4_values(0, 64, 0, None, None, None, None) == 0


def test_workspace_is_the_modified_steps():
    """A 4-bit decode step's partials are those of a step with modifications: neither takes the bf16 decode kernel."""
    g = dict(num_seqs=32, num_tokens=1, num_q_heads=16, num_kv_heads=8, head_dim=128, head_dim_v=128, k_page_stride=16 * 8 * 128,
             k_slot_stride=128, k_head_stride=2048, v_page_stride=16 * 8 * 128, v_slot_stride=128, v_head_stride=2048, page_size=16,
             block_table_stride=256, max_seq_len=4096)
    nb, ns = hip.workspace_size(g, kv4=True)
    assert (nb, ns) == hip.workspace_size(g, mods=hip.ScoreModsArgs()) and ns > 0

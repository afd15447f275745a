"""Score modifications without a GPU: what the entry points refuse, how the workspace follows the span,
and the restated cap against tanh in decimal arithmetic."""

import ctypes
from decimal import Decimal

import numpy as np
import pytest

from exactattention_amd import hip
import mod_oracle as mo

GEOM = dict(num_seqs=2, num_tokens=1, num_q_heads=4, num_kv_heads=2, head_dim=128, head_dim_v=128, q_seq_stride=512,
            q_tok_stride=512, q_head_stride=128, o_seq_stride=512, o_tok_stride=512, o_head_stride=128, k_page_stride=4096,
            k_slot_stride=256, k_head_stride=128, v_page_stride=4096, v_slot_stride=256, v_head_stride=128, page_size=16,
            block_table_stride=8192, max_seq_len=131072)


def _size(mods, **opt):
    o = hip.Options(tier2=1, **opt)
    nb, ns = ctypes.c_size_t(0), ctypes.c_int32(0)
    rc = hip.load().ea_hip_mods_workspace_size(ctypes.byref(hip.geometry(GEOM)), ctypes.byref(o), ctypes.byref(mods),
                                               ctypes.byref(nb), ctypes.byref(ns))
    return rc, nb.value, ns.value


@pytest.mark.parametrize("kw", [dict(window=-1), dict(max_span=-1), dict(softcap_bits=0x80000000), dict(softcap_bits=0xBF800000),
                                dict(softcap_bits=0x7F800000), dict(softcap_bits=0x7FC00000), dict(softcap_bits=1)])
def test_refused(kw):
    m = hip.ScoreModsArgs(**kw)
    assert _size(m)[0] == -2
    o = hip.Options(tier2=1)
    p = 1 << 20
    b = hip.Buffers(q=p, k=p, v=p, seq_len=p, kv_len=p, out=p, flags=p)
    assert hip.load().ea_hip_attention_mods(ctypes.byref(hip.geometry(GEOM)), ctypes.byref(b), ctypes.byref(o), ctypes.byref(m),
                                            p, 1 << 30, None) == -2
    assert hip.load().ea_hip_exact_rows_mods(ctypes.byref(hip.geometry(GEOM)), ctypes.byref(b), ctypes.byref(o),
                                             ctypes.byref(m), None) == -2


def test_refused_with_timers():
    assert _size(hip.ScoreModsArgs(), timers=1 << 20)[0] == -2
    assert _size(hip.ScoreModsArgs())[0] == 0


@pytest.mark.parametrize("kw", [dict(softcap=-1.0), dict(softcap=float("inf")), dict(softcap=float("nan")), dict(softcap=1e-40),
                                dict(window=-1), dict(max_span=-2), dict(window=1 << 31)])
def test_spec_refused(kw):
    with pytest.raises(ValueError):
        hip.ScoreMods(**kw)


@pytest.mark.parametrize("kw", [dict(kv_begin=np.zeros(3, np.int32)), dict(q_pos=np.zeros(1, np.int32)),
                                dict(slopes=np.zeros(2, np.float32)), dict(slopes=np.zeros(4, np.int32)),
                                dict(kv_begin=np.zeros(2, np.float32)), dict(q_pos=np.zeros(2, bool)),
                                dict(kv_begin=np.array([0, 1 << 31])), dict(q_pos=np.array([0, -(1 << 31) + 131072]))])
def test_arrays_refused(kw):
    with pytest.raises(ValueError):
        hip.ScoreMods(**kw).bind(GEOM, "cpu")


def test_arrays_bound():
    a, keep = hip.ScoreMods(kv_begin=np.array([3, 4]), slopes=np.ones(4), window=7, softcap=2.0).bind(GEOM, "cpu")
    assert a.kv_begin == keep[0].data_ptr() and a.q_pos is None and a.window == 7 and a.softcap_bits == 0x40000000
    assert keep[0].dtype.itemsize == 4 and keep[2].dtype.is_floating_point


def test_farthest_positions():
    """Positions whose distance to every key still fits 32 bits."""
    hip.ScoreMods(q_pos=np.array([(1 << 31) - 1, -(1 << 31) + 131073])).bind(GEOM, "cpu")


def test_window_sizes_the_grid():
    """A window far below the sequence length takes the splits of a cache of its size, not the cache's."""
    plain = _size(hip.ScoreModsArgs())
    win = _size(hip.ScoreModsArgs(window=1024))
    span = _size(hip.ScoreModsArgs(max_span=1024))
    assert plain[0] == win[0] == span[0] == 0
    assert win[1:] == span[1:] and win[2] <= 17 and plain[2] > 32


@pytest.mark.parametrize("c", [1.0, 43.28085, 72.13475, 0.01, 3.0e30])
def test_cap_is_tanh(c):
    """The cap's sequence is RN32 of c tanh(t / c), or its neighbour within 2^-14 of a step of a midpoint."""
    c = float(np.float32(c))
    rng = np.random.default_rng(4)
    ts = np.concatenate([c * rng.standard_normal(150) * 2, c * 2.0 ** rng.uniform(-40, 6, 150), [0.0, c, -c, c * 2.0 ** -11, 1e38, -1e38]])
    for t in ts.astype(np.float32).tolist():
        got, want = mo.cap32(t, c), mo.tanh_exact(t, c)
        step = float(np.spacing(np.float32(abs(got)))) if got else 2.0 ** -149
        assert abs(Decimal(got) - want) <= Decimal(step) * (Decimal("0.5") + Decimal(2) ** -14), t
        assert abs(got) <= abs(t) and abs(got) <= c


def test_bias_is_one_rounding():
    assert mo.bias32(1.0, 2.0 ** -24, 1) == float(np.float32(1.0 - 2.0 ** -24))
    assert mo.bias32(0.0, 0.1, 7) == float(np.float32(-np.float64(np.float32(0.1)) * 7))
    assert mo.bias32(-3.5, 0.0, 1 << 30) == -3.5
    # |n - p| past 24 bits rounds first
    assert mo.bias32(0.0, 1.0, (1 << 24) + 1) == -float(1 << 24)

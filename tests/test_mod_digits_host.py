"""Which steps with score modifications read a digit-tile cache, and the workspace they need, without a GPU
(host logic of the library alone)."""

import ctypes

import numpy as np
import pytest

from exactattention_amd import hip

FAKE = 4096  # stands for device memory: only the host's plan is made


def _geom(T, S, B=1, Hq=16, Hkv=8, d=128):
    return dict(num_seqs=B, num_tokens=T, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=d, head_dim_v=d, q_seq_stride=T * Hq * d,
                q_tok_stride=Hq * d, q_head_stride=d, o_seq_stride=T * Hq * d, o_tok_stride=Hq * d, o_head_stride=d,
                k_page_stride=16 * Hkv * d, k_slot_stride=Hkv * d, k_head_stride=d, v_page_stride=16 * Hkv * d,
                v_slot_stride=Hkv * d, v_head_stride=d, page_size=16, block_table_stride=S // 16 + 1, max_seq_len=S)


def _reads(g, m, digits=True, **opt):
    o = hip.Options(tier2=1, kv_digits=FAKE if digits else None, kv_digits_tiles=(g["max_seq_len"] + 63) // 64 if digits else 0, **opt)
    r = ctypes.c_int32(-7)
    rc = hip.load().ea_hip_mods_reads_kv_digits(ctypes.byref(hip.geometry(g)), ctypes.byref(o),
                                                None if m is None else ctypes.byref(m), ctypes.byref(r))
    return rc, r.value


def _plain(g, **opt):
    o = hip.Options(tier2=1, kv_digits=FAKE, kv_digits_tiles=(g["max_seq_len"] + 63) // 64, **opt)
    r = ctypes.c_int32(-7)
    rc = hip.load().ea_hip_reads_kv_digits(ctypes.byref(hip.geometry(g)), ctypes.byref(o), ctypes.byref(r))
    return rc, r.value


def test_reads_follow_the_modified_kernel_choice():
    """A modified step that runs on the multi-row kernel reads no tile, though the plain step of its shape does."""
    slopes = hip.ScoreModsArgs(slopes=FAKE)
    small, large = _geom(64, 64), _geom(700, 4000)
    assert _plain(small) == _plain(large) == _plain(large, out_fp32=1) == (0, 1)
    assert _reads(large, hip.ScoreModsArgs(window=1024)) == _reads(large, slopes) == (0, 1)
    assert _reads(large, slopes, out_fp32=1) == (0, 0)   # fp32 outputs under a bias: the fp64 sums
    assert _reads(small, hip.ScoreModsArgs(softcap_bits=0x41A00000)) == (0, 0)
    assert _reads(small, slopes, kernel=1) == (0, 1)
    assert _reads(large, slopes, digits=False) == (0, 0)  # no cache given


def test_reads_without_modifications():
    for T in (1, 8, 64, 300):
        for S in (64, 1000, 9000):
            g = _geom(T, max(S, T))
            assert _reads(g, None) == _plain(g)
    assert _reads(_geom(64, 64, d=100), None)[0] == -1


def test_reads_refused():
    assert _reads(_geom(64, 64), hip.ScoreModsArgs(window=-1))[0] == -2
    assert _reads(_geom(64, 64), hip.ScoreModsArgs(), splits=-1)[0] == -2


@pytest.mark.parametrize("geom", [(96, 2000, 2, 16, 8), (33, 16000, 2, 16, 8)])
def test_workspace_holds_a_step_with_digits(geom):
    """The estimate that picks the kernel leaves slicing out where a digit cache is given: a problem's workspace
    is enough for its launches with one and without."""
    T, S, B, Hq, Hkv = geom
    g = _geom(T, S, B, Hq, Hkv)
    spec = hip.ScoreMods(softcap=20.0)
    a, _ = spec.bind(g, "cpu")
    without, with_ = (hip.workspace_size(g, mods=a, kv_digits=x)[0] for x in (False, True))
    assert _reads(g, a) == (0, 1) and with_ > without  # the choice differs here
    prob = dict(geom=g, out_shape=(B, T, Hq, 128), q=np.zeros((B, T, Hq, 128), np.uint16))
    dp = hip.DeviceProblem(prob, device="cpu", mods=spec)
    assert dp.ws_bytes >= max(without, with_) and dp.workspace.numel() >= dp.ws_bytes
    assert hip.DeviceProblem(prob, device="cpu").ws_bytes == hip.workspace_size(g)[0]


def test_modified_prompts_keep_no_epoch_sums():
    """A plain int8 step keeps 128 KB of epoch sums per row block and key split; a modified one keeps its own in
    registers and asks for that much less."""
    for T, S, B in ((4096, 4096, 1), (2500, 2500, 1), (700, 700, 3)):
        g = _geom(T, S, B)
        m = hip.ScoreModsArgs(softcap_bits=0x41A00000)
        assert _reads(g, m) == (0, 1)
        plain, splits = hip.workspace_size(g)
        mods, other = hip.workspace_size(g, mods=m)
        blocks = B * 8 * ((2 * T + 31) // 32)
        assert splits == other and plain - mods >= blocks * splits * 512 * 32 * 8

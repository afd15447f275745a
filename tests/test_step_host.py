"""The step plan and the rotary positions: what they refuse, without a GPU (the C entry points check
their arguments before any device call)."""

import ctypes

import numpy as np
import pytest

from exactattention_amd import hip
from exactattention_amd.step import Rotary, StepPlan, _deal

PTR = 1 << 20  # stands for device memory: a refused call touches none


def _plan(**kw):
    a = dict(num_seqs=2, page_size=16, table_rows=4, table_width=8, max_tokens=4, pad_tokens=2, max_seq_len=100,
             free_capacity=3, seq_len=PTR, counts=PTR, free_pages=PTR, num_free=PTR, block_table=PTR, dst_rows=PTR,
             kv_len=PTR, new_seq_len=2 * PTR, new_num_free=2 * PTR, status=PTR)
    a.update(kw)
    return hip.load().ea_hip_step_plan(ctypes.byref(hip.StepPlanArgs(**a)), None)


@pytest.mark.parametrize("kw", [
    dict(num_seqs=-1), dict(num_seqs=8193), dict(page_size=0), dict(page_size=24), dict(table_rows=65537), dict(table_width=-1),
    dict(max_tokens=-1), dict(pad_tokens=-1), dict(pad_tokens=0), dict(free_capacity=-1), dict(max_seq_len=-1),
    dict(seq_len=None), dict(counts=None), dict(free_pages=None), dict(num_free=None), dict(block_table=None),
    dict(dst_rows=None), dict(new_seq_len=None), dict(new_num_free=None), dict(status=None),
    dict(new_seq_len=PTR), dict(new_num_free=PTR),  # an output that is the input it is computed from
])
def test_step_plan_refuses(kw):
    assert _plan(**kw) == -1


def test_step_plan_null():
    assert hip.load().ea_hip_step_plan(None, None) == -1
    assert hip.load().ea_hip_rotary(None, None) == -1


def _rotary(**kw):
    a = dict(num_tokens=3, num_q_heads=2, num_kv_heads=1, head_dim=64, rot_dim=64, num_axes=1, scale=1.0, q_tok_stride=128,
             q_head_stride=64, k_tok_stride=64, k_head_stride=64, v_tok_stride=64, v_head_stride=64, q_out_rows=3,
             pool_rows=3, q=PTR, k=PTR, v=PTR, positions=PTR, half_turns=PTR, axis_of_pair=PTR, q_out=PTR, k_out=PTR, v_out=PTR)
    a.update(kw)
    return hip.load().ea_hip_rotary(ctypes.byref(hip.RotaryArgs(**a)), None)


@pytest.mark.parametrize("rc, kw", [
    (-1, dict(num_tokens=-1)), (-1, dict(num_q_heads=-1)), (-1, dict(num_kv_heads=-2)), (-1, dict(head_dim=0)),
    (-1, dict(head_dim=260)), (-1, dict(rot_dim=0)), (-1, dict(rot_dim=66)), (-1, dict(rot_dim=63)), (-1, dict(num_axes=0)),
    (-1, dict(num_axes=2, axis_of_pair=None)), (-2, dict(in_fp32=2)), (-2, dict(out_fp32=1)), (-2, dict(scale=float("nan"))),
    (-2, dict(scale=float("inf"))), (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(q_out=None)), (-1, dict(k_out=None)),
    (-1, dict(v_out=None)), (-1, dict(positions=None)), (-1, dict(half_turns=None)), (-1, dict(pool_rows=-1)),
    (-1, dict(head_dim=63, rot_dim=62, adjacent=1)), (-1, dict(num_q_heads=1 << 28)),
])
def test_rotary_refuses(rc, kw):
    assert _rotary(**kw) == rc


def test_rotary_without_tokens():
    assert _rotary(num_tokens=0, q=None, k=None, v=None, positions=None, q_out=None, k_out=None, v_out=None) == 0


@pytest.mark.parametrize("kw", [
    dict(head_dim=0), dict(head_dim=300), dict(head_dim=64, rot_dim=66), dict(head_dim=64, rot_dim=7),
    dict(head_dim=64, inv_freq=[1.0, 2.0]), dict(head_dim=4, inv_freq=[1.0, float("inf")]), dict(head_dim=64, sections=[8, 8]),
    dict(head_dim=64, sections=[40, -8]), dict(head_dim=64, sections=[32], axis_of_pair=[0] * 32),
    dict(head_dim=64, axis_of_pair=[0] * 31), dict(head_dim=4, axis_of_pair=[0, -1]), dict(head_dim=4, axis_of_pair=[0, 256]),
    dict(head_dim=64, scale=float("nan")), dict(head_dim=64, device="cpu"),
])
def test_rotary_spec_refuses(kw):
    with pytest.raises(ValueError):
        Rotary(**dict(dict(device="cpu"), **kw))


@pytest.mark.parametrize("args", [(-1, 4, 2), (2, -1, 2), (2, 4, 0), (8193, 4, 2), (2, 4, 2)])
def test_plan_spec_refuses(args):
    with pytest.raises(ValueError):
        StepPlan(*args, device="cpu")


def test_sections():
    assert _deal([2, 3, 3], 8, False) == [0, 0, 1, 1, 1, 2, 2, 2]
    assert _deal([2, 3, 3], 8, True) == [0, 1, 2, 0, 1, 2, 1, 2]
    assert _deal([0, 2], 2, True) == [1, 1]
    assert np.bincount(_deal([16, 24, 24], 64, True)).tolist() == [16, 24, 24]

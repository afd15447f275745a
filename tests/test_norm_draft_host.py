"""Head norms with rotary positions, and the check of drafted tokens: what their C entry points refuse, without a GPU."""

import ctypes

import pytest

from exactattention_amd import hip

PTR = 1 << 20  # stands for device memory: a refused call touches none
NAN = float("nan")


def _rotary(**kw):
    a = dict(num_tokens=3, num_q_heads=2, num_kv_heads=1, head_dim=64, rot_dim=64, num_axes=1, scale=1.0, q_tok_stride=128,
             q_head_stride=64, k_tok_stride=64, k_head_stride=64, v_tok_stride=64, v_head_stride=64, qo_tok_stride=128, qo_head_stride=64,
             ko_tok_stride=64, ko_head_stride=64, vo_tok_stride=64, vo_head_stride=64, q_out_rows=3, pool_rows=3, q=PTR, k=PTR, v=PTR,
             positions=PTR, half_turns=PTR, axis_of_pair=PTR, q_out=2 * PTR, k_out=3 * PTR, v_out=4 * PTR)
    a.update(kw)
    return hip.RotaryArgs(**a)


def _fwd(r=None, **kw):
    a = dict(q_weight=PTR, k_weight=PTR, eps=1e-6)
    a.update(kw)
    return hip.load().ea_hip_norm_rotary(ctypes.byref(hip.NormRotaryArgs(r=_rotary(**(r or {})), **a)), None)


ROTARY = [(-1, dict(num_tokens=-1)), (-1, dict(num_q_heads=-1)), (-1, dict(num_kv_heads=-2)), (-1, dict(head_dim=0)),
          (-1, dict(head_dim=260)), (-1, dict(rot_dim=66)), (-1, dict(rot_dim=63)), (-1, dict(rot_dim=-2)), (-1, dict(num_axes=0)),
          (-1, dict(num_axes=2, axis_of_pair=None)), (-2, dict(in_fp32=2)), (-2, dict(out_fp32=1)), (-2, dict(scale=NAN)),
          (-2, dict(scale=float("inf"))), (-1, dict(q=None)), (-1, dict(k=None)), (-1, dict(q_out=None)), (-1, dict(k_out=None)),
          (-1, dict(positions=None)), (-1, dict(half_turns=None)), (-1, dict(head_dim=63, rot_dim=62, adjacent=1)),
          (-1, dict(head_dim=253, rot_dim=64)), (-1, dict(head_dim=254, rot_dim=6))]


@pytest.mark.parametrize("rc, r", ROTARY + [(-1, dict(v_out=None)), (-1, dict(pool_rows=-1)), (-1, dict(q_out_rows=-1)),
                                            (-2, dict(inverse=1)), (-1, dict(num_q_heads=1 << 30))])
def test_forward_refuses(rc, r):
    assert _fwd(r) == rc


@pytest.mark.parametrize("rc, kw", [(-1, dict(q_weight=None)), (-1, dict(k_weight=None)), (-2, dict(eps=-1.0)), (-2, dict(eps=NAN)),
                                    (-2, dict(eps=float("inf"))), (-2, dict(weights_fp32=2)), (-1, dict(k_scales=PTR, page_size=16)),
                                    (-1, dict(v_scales=PTR, page_size=16)), (-1, dict(k_scales=PTR, v_scales=PTR))])
def test_norm_refuses(rc, kw):
    assert _fwd(**kw) == rc


FOUR = dict(k_scales=PTR, v_scales=PTR, page_size=16, k_page_stride=1024, v_page_stride=1024)


@pytest.mark.parametrize("r, kw", [(dict(head_dim=60, rot_dim=60), {}), (dict(rot_dim=62), {}), (dict(ko_tok_stride=80), {}),
                                   (dict(vo_head_stride=16), {}), ({}, dict(k_page_stride=1000)), (dict(k_out=PTR + 2), {}),
                                   (dict(in_fp32=1, out_fp32=1), {}), ({}, dict(page_size=0)), ({}, dict(page_size=-16))])
def test_four_bits_refuse(r, kw):
    assert _fwd(r, **{**FOUR, **kw}) == -1


def test_nothing_to_do():
    none = dict(q=None, k=None, v=None, positions=None, q_out=None, k_out=None, v_out=None)
    assert _fwd(dict(num_tokens=0, **none)) == 0
    assert _fwd(dict(num_q_heads=0, num_kv_heads=0, **none)) == 0
    assert hip.load().ea_hip_norm_rotary(None, None) == hip.load().ea_hip_norm_rotary_grad(None, None) == -1
    assert hip.load().ea_hip_norm_rotary_grad_size(None) == 0


def _grad(r=None, **kw):
    a = dict(gq=PTR, gk=PTR, gq_tok_stride=128, gq_head_stride=64, gk_tok_stride=64, gk_head_stride=64, q_weight=PTR, k_weight=PTR,
             dq_weight=PTR, dk_weight=PTR, partial=PTR, eps=1e-6)
    a.update(kw)
    return hip.load().ea_hip_norm_rotary_grad(ctypes.byref(hip.NormRotaryGradArgs(r=_rotary(v=None, **(r or {})), **a)), None)


@pytest.mark.parametrize("rc, r", [x for x in ROTARY if x[1] != dict(out_fp32=1)] +
                         [(-2, dict(in_fp32=1)), (-2, dict(inverse=1)), (-1, dict(q_out=PTR)), (-1, dict(k_out=PTR))])
def test_gradient_refuses(rc, r):
    assert _grad(r) == rc


@pytest.mark.parametrize("rc, kw", [(-1, dict(gq=None)), (-1, dict(gk=None)), (-1, dict(q_weight=None)), (-1, dict(k_weight=None)),
                                    (-1, dict(partial=None)), (-2, dict(eps=NAN)), (-2, dict(weights_fp32=-1))])
def test_gradient_arguments(rc, kw):
    assert _grad(**kw) == rc


def _draft(**kw):
    a = dict(num_seqs=2, num_drafts=3, vocab=10, p_seq_stride=40, p_row_stride=10, q_seq_stride=30, q_row_stride=10, probs=PTR,
             drafted=PTR, uniforms=PTR, accepted=PTR, path=PTR, tokens=PTR, work=PTR)
    a.update(kw)
    return hip.load().ea_hip_draft_check(ctypes.byref(hip.DraftCheckArgs(**a)), None)


@pytest.mark.parametrize("kw", [dict(num_seqs=-1), dict(num_seqs=65536), dict(num_drafts=-1), dict(num_drafts=65), dict(vocab=0),
                                dict(vocab=(1 << 19) + 1), dict(probs=None), dict(drafted=None), dict(uniforms=None), dict(accepted=None),
                                dict(path=None), dict(tokens=None), dict(work=None), dict(draft_probs=PTR, parents=PTR)])
def test_draft_check_refuses(kw):
    assert _draft(**kw) == -1


def test_draft_check_sizes():
    lib = hip.load()
    assert lib.ea_hip_draft_check(None, None) == -1 and lib.ea_hip_draft_check_size(None) == 0
    assert _draft(num_seqs=0, probs=None) == 0
    assert lib.ea_hip_draft_check_size(hip.DraftCheckArgs(num_seqs=3)) == 3 * lib.ea_hip_draft_check_size(hip.DraftCheckArgs(num_seqs=1)) > 0

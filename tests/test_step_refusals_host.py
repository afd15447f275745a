"""What the step's operators refuse of their tensors, without a GPU: tensors on the host stand for the device's, no call reaches it."""

import pytest
import torch

from exactattention_amd import hip, step


@pytest.fixture
def calls(monkeypatch):
    made = []
    monkeypatch.setattr(step, "_call", lambda fn, args, index, what: made.append(what))
    return made


def _check(B, N, V):
    """A DraftCheck whose device is the host (index -1)."""
    c = step.DraftCheck.__new__(step.DraftCheck)
    c.num_seqs, c.num_drafts, c.vocab, c.dev, c._at, c._fn = B, N, V, torch.device("cpu"), -1, None
    c._i32, c._f32, c._out = torch.int32, torch.float32, (0,) * 4
    c.accepted, c.path, c.tokens = (torch.empty(s, dtype=torch.int32) for s in ((B,), (B, N), (B, N + 1)))
    return c


def test_drafts_of_another_layout(calls):
    """Tensors of as many entries laid out otherwise, which would give tokens and random numbers to the wrong sequences."""
    B, N, V = 2, 3, 50
    c = _check(B, N, V)
    ok = dict(probs=torch.zeros((B, N + 1, V)), drafted=torch.zeros((B, N), dtype=torch.int32), uniforms=torch.zeros((B, N + 1)))
    ints = ok["drafted"].t().contiguous()
    for bad in (dict(drafted=ints), dict(drafted=ints.view(-1)), dict(parents=ints), dict(parents=ints.view(-1)),
                dict(uniforms=ok["uniforms"].t().contiguous()), dict(uniforms=ok["uniforms"].view(-1)),
                dict(counts=torch.zeros((B, 1), dtype=torch.int32)), dict(counts=torch.zeros((1, B), dtype=torch.int32))):
        with pytest.raises(ValueError, match="must be"):
            c.verify(**{**ok, **bad})
    assert not calls
    c.verify(**ok)
    c.verify(**ok, parents=ok["drafted"].clone(), counts=torch.zeros(B, dtype=torch.int32))
    assert len(calls) == 2


def test_append_without_a_pool_for_v(calls, monkeypatch):
    """A bf16 pool for k alone is an argument that is missing, not an attribute of None."""
    r = step.Rotary.__new__(step.Rotary)
    r.dev, r._at, r.head_dim, r._i64, r._bits = torch.device("cpu"), -1, 64, torch.int64, (torch.bfloat16, torch.int16)
    monkeypatch.setattr(step.Rotary, "_args", lambda *a: (2, 1, 1, False, (64, 64) * 3, 0))
    x, at = torch.zeros((2, 1, 64), dtype=torch.bfloat16), torch.zeros(2, dtype=torch.int64)
    for v_pool in ((), (None,)):
        with pytest.raises(ValueError, match="v_pool"):
            r.append(x, x, x, at.int(), at, torch.zeros((1, 16, 1, 64), dtype=torch.bfloat16), *v_pool)
    assert not calls


def test_forward_mode_tangents(calls, monkeypatch):
    """A tangent of q, k or a weight is refused, whether or not anything needs a gradient: the kernels would drop it."""
    import torch.autograd.forward_ad as fwd
    monkeypatch.setattr(step, "_C", torch._C)
    monkeypatch.setattr(step, "_FORWARD", fwd, raising=False)
    r = step.Rotary.__new__(step.Rotary)
    r.dev, r._at, r.head_dim, r._fn, r._norm_fn, r._half, r._axis = torch.device("cpu"), -1, 8, None, None, 0, 0
    r.rot_dim, r.axes, r.adjacent, r.scale = 8, 1, False, 1.0
    r._f32, r._i32, r._bits = torch.float32, torch.int32, (torch.bfloat16, torch.int16)
    q, k, w, pos = torch.ones((2, 3, 8)), torch.ones((2, 1, 8)), torch.ones(8), torch.zeros(2, dtype=torch.int32)
    with fwd.dual_level():
        r.rotate(q, k, pos)
        r.rotate(q, k, pos, norm=step.HeadNorm(w, w))
        assert len(calls) == 2
        for args, norm in (((fwd.make_dual(q, q), k), None), ((q, fwd.make_dual(k, k)), None),
                           ((q, fwd.make_dual(k, k)), step.HeadNorm(w, w)), ((q, k), step.HeadNorm(fwd.make_dual(w, w), w)),
                           ((q, k), step.HeadNorm(w, fwd.make_dual(w, w))), ((fwd.make_dual(q.clone().requires_grad_(), q), k), None)):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                r.rotate(*args, pos, norm=norm)
    r.rotate(q, k, pos)
    assert len(calls) == 3


@pytest.mark.parametrize("eps", [3.5e38, 1e300, -1e-9, float("inf"), float("nan")])
def test_eps_that_is_no_fp32(eps):
    """Refused where the norm is made, not while a step's arguments are packed, its tokens already counted in the cache."""
    w = torch.ones(8)
    with pytest.raises(ValueError, match="eps"):
        step.HeadNorm(w, w, eps)
    assert step.HeadNorm(w, w, 3e38).eps == 3e38 and step.HeadNorm(w, w, 0.0).eps == 0.0


def test_draft_check_workspace():
    """A sum for each of 64 parts of the vocabulary and their count, for each sequence."""
    size = hip.load().ea_hip_draft_check_size
    assert [size(hip.DraftCheckArgs(num_seqs=n)) for n in (0, 1, 7)] == [0, 65 * 8, 7 * 65 * 8]

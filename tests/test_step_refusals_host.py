"""What the step's operators refuse of their tensors, without a GPU: tensors on the host stand for the device's, no call reaches it."""

import pytest
import torch

from exactattention_amd import step


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

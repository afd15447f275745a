"""GPU: gradients through the rotary positions, against the formula's in 64 bits and against differences."""

import numpy as np
import pytest

from exactattention_amd.step import Rotary

pytestmark = pytest.mark.gpu


def _turned(rot, x, positions, sign):
    """R(sign theta) x times the scale, in 64 bits on the host."""
    x = x.double().cpu().numpy()
    n, h, d = x.shape
    half = rot.rot_dim // 2
    pos = positions.cpu().numpy().reshape(-1, n) if positions.dim() == 2 else positions.cpu().numpy()[None]
    ax = rot.axis_of_pair.cpu().numpy()
    theta = sign * np.pi * rot.half_turns.cpu().numpy()[None] * pos[ax].T.astype(np.float64)  # (n, half)
    c, s = np.cos(theta)[:, None] * rot.scale, np.sin(theta)[:, None] * rot.scale
    y = x.copy()
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if rot.adjacent else (slice(0, half), slice(half, 2 * half))
    y[..., i], y[..., j] = x[..., i] * c - x[..., j] * s, x[..., j] * c + x[..., i] * s
    return y


def _near(got, want, bits, size):
    """One rounding of half a step, 2^-bits of the value, and the angles': the kernel's and this file's are within
    2^-38 each of the exact ones (positions below 2^12, frequencies up to 1), which moves a pair by that of its size."""
    got = got.double().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -bits * np.abs(want) + 2.0 ** -37 * size + 1e-44).all()


CASES = [
    # tokens, Hq, Hkv, d, keyword arguments of Rotary
    (5, 3, 1, 64, dict()),
    (1, 2, 2, 128, dict(adjacent=True, scale=0.75)),
    (33, 4, 2, 40, dict(rot_dim=24)),
    (7, 2, 1, 10, dict(adjacent=True)),          # accesses of single elements
    (900, 2, 1, 64, dict(sections=[8, 12, 12], interleaved=True)),
]


def _inputs(case, dtype, seed):
    import torch
    n, hq, hk, d, kw = case
    g = torch.Generator().manual_seed(seed)
    rot = Rotary(d, device="cuda:0", **kw)
    q, k, gq, gk = (torch.randn((n, h, d), generator=g).to(dtype).cuda() for h in (hq, hk, hq, hk))
    pos = torch.randint(0, 4096, (rot.axes, n) if rot.axes > 1 else (n,), generator=g, dtype=torch.int32).cuda()
    return rot, q.requires_grad_(), k.requires_grad_(), gq, gk, pos


@pytest.mark.parametrize("dtype, bits", [("float32", 24), ("bfloat16", 8)])
@pytest.mark.parametrize("inverse", [False, True])
@pytest.mark.parametrize("case", CASES)
def test_gradient_is_the_formula(gpu, case, inverse, dtype, bits):
    import torch
    rot, q, k, gq, gk, pos = _inputs(case, getattr(torch, dtype), 3)
    yq, yk = rot.rotate(q, k, pos, inverse=inverse)
    with torch.no_grad():
        pq, pk = rot.rotate(q, k, pos, inverse=inverse)
    assert torch.equal(yq, pq) and torch.equal(yk, pk) and pq.grad_fn is None
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    sign = 1 if inverse else -1
    for got, g in ((dq, gq), (dk, gk)):
        assert got.dtype == g.dtype
        _near(got, _turned(rot, g, pos, sign), bits, float(g.abs().max()) * rot.scale * 2)


def test_gradient_is_the_difference(gpu):
    """f(x) = sum y g, linear in x: a step of 1 moves two elements of y, each rounded within 2^-24 of itself,
    on both sides, so the quotient is within 2 x 2 x 2^-24 / 2 of the largest |y| |g|."""
    import torch
    rot, q, k, gq, gk, pos = _inputs(CASES[2], torch.float32, 4)
    yq, yk = rot.rotate(q, k, pos)
    dq, dk = torch.autograd.grad((yq, yk), (q, k), (gq, gk))
    f = lambda a, b: sum((y.double() * g).sum().item() for y, g in zip(rot.rotate(a, b, pos), (gq, gk)))
    rng = np.random.default_rng(1)
    with torch.no_grad():
        for which, x, g, dx in ((0, q, gq, dq), (1, k, gk, dk)):
            for _ in range(12):
                at = tuple(int(rng.integers(0, m)) for m in x.shape)
                side = []
                for h in (1.0, -1.0):
                    z = x.clone()
                    z[at] += h
                    # z[at] is rounded: count the step that was taken
                    side.append((f(z, k) if which == 0 else f(q, z), z[at].item()))
                diff = (side[0][0] - side[1][0]) / (side[0][1] - side[1][1])
                big = (float(x.abs().max()) + 1) * 2 * float(g.abs().max())
                # the sums of 64-bit products add 2^-52 of each term, far below
                assert abs(diff - dx[at].item()) <= 2.0 ** -23 * big + 2.0 ** -24 * abs(dx[at].item()) + 1e-9


def test_one_of_them_alone(gpu):
    """Only q, only k, a gradient of a sum (strides of 0), of one output, and none asked for."""
    import torch
    rot, q, k, gq, gk, pos = _inputs(CASES[0], torch.float32, 5)
    yq, yk = rot.rotate(q, k.detach(), pos)
    assert yq.requires_grad and not yk.requires_grad
    dq, = torch.autograd.grad(yq.sum(), q)
    _near(dq, _turned(rot, torch.ones_like(q), pos, -1), 24, 2.0)
    yq, yk = rot.rotate(q.detach(), k, pos)
    assert yk.requires_grad and not yq.requires_grad
    dk, = torch.autograd.grad(yk, k, gk)
    _near(dk, _turned(rot, gk, pos, -1), 24, 2 * float(gk.abs().max()))
    yq, yk = rot.rotate(q, k, pos)  # both, one output used
    dq, dk = torch.autograd.grad(yk, (q, k), gk.transpose(1, 2).contiguous().transpose(1, 2), allow_unused=True)
    assert dq is None
    _near(dk, _turned(rot, gk, pos, -1), 24, 2 * float(gk.abs().max()))


def test_gradient_of_the_gradient(gpu):
    """The rotation keeps lengths: the gradient of |y|^2 / 2 is x, and its own gradient the identity."""
    import torch
    rot, q, k, gq, gk, pos = _inputs(CASES[0], torch.float32, 6)
    yq, yk = rot.rotate(q, k, pos)
    dq, = torch.autograd.grad((yq * yq).sum() / 2, q, create_graph=True)
    big = float(q.detach().abs().max()) * 2
    # y and dq round once each, and so do both passes of the second gradient
    assert float((dq.detach() - q.detach()).abs().max()) <= 4 * 2.0 ** -24 * big
    d2, = torch.autograd.grad((dq * gq).sum(), q)
    assert float((d2 - gq).abs().max()) <= 4 * 2.0 ** -24 * 2 * float(gq.abs().max())


def test_through_a_projection_and_inputs_of_a_layer(gpu):
    """Leaves behind a product, views of one tensor, backward called as a training step does."""
    import torch
    g = torch.Generator().manual_seed(7)
    n, hq, hk, d, width = 40, 4, 2, 32, 24
    rot = Rotary(d, device="cuda:0")
    w = torch.randn((width, (hq + hk) * d), generator=g).cuda().requires_grad_()
    x = torch.randn((n, width), generator=g).cuda()
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    grads = []
    for _ in range(3):
        w.grad = None
        qk = (x @ w).view(n, hq + hk, d)
        yq, yk = rot.rotate(qk[:, :hq], qk[:, hq:], pos)
        (yq.pow(2).sum() + yk.pow(3).sum()).backward()
        grads.append(w.grad.clone())
    assert torch.equal(grads[0], grads[1]) and torch.equal(grads[0], grads[2])
    with torch.no_grad():
        qk = (x @ w).view(n, hq + hk, d)
        yq, yk = rot.rotate(qk[:, :hq], qk[:, hq:], pos)
        dq, dk = rot.rotate(2 * yq, 3 * yk.pow(2), pos, inverse=True)
        each = torch.cat([dq, dk], 1).view(n, -1)
        want, size = x.t() @ each, x.t().abs() @ each.abs()
    # the same n products in sums of any order, each within n 2^-24 of their sizes, of numbers that a power and its
    # factor round in up to 8 places
    assert bool(((grads[0] - want).abs() <= 2 * (n + 8) * 2.0 ** -24 * size).all())


def test_outputs_given_are_refused(gpu):
    import torch
    rot, q, k, gq, gk, pos = _inputs(CASES[0], torch.float32, 8)
    for kw in (dict(q_out=torch.empty_like(q)), dict(k_out=k.detach().clone()), dict(q_out=q, k_out=k)):
        with pytest.raises(ValueError, match="gradients"):
            rot.rotate(q, k, pos, **kw)
    with torch.no_grad():
        rot.rotate(q, k, pos, q_out=torch.empty_like(q))
    rot.rotate(q.detach(), k.detach(), pos, q_out=torch.empty_like(q), k_out=torch.empty_like(k))


def test_on_a_stream_and_in_a_graph(gpu):
    """Forward and backward on another stream than the default, and captured and replayed on new values."""
    import torch
    rot, q, k, gq, gk, pos = _inputs((50, 4, 2, 64, {}), torch.float32, 9)
    st = torch.cuda.Stream()
    torch.cuda.synchronize()

    def step():
        yq, yk = rot.rotate(q, k, pos)
        return (yq, yk, *torch.autograd.grad((yq, yk), (q, k), (gq, gk)))

    def want():
        with torch.no_grad():
            return (*rot.rotate(q, k, pos), *rot.rotate(gq, gk, pos, inverse=True))

    with torch.cuda.stream(st):
        for _ in range(3):
            got = step()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want()))
    del got  # no eager graph of these leaves lives while the capture runs
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = step()
    for i in range(4):
        with torch.no_grad():
            for x in (q, k, gq, gk):
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want())), i

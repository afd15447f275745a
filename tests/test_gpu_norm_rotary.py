"""GPU: head norms with rotary positions in one pass, forward, into both kinds of cache, and backward, against the formulas
in 64 bits."""

import numpy as np
import pytest

import kv4_format as f4
from exactattention_amd.kv4 import KV4Pool
from exactattention_amd.step import HeadNorm, Rotary

pytestmark = pytest.mark.gpu

# tokens, Hq, Hkv, d, keyword arguments of Rotary; the last ones have heads or halves that no run of 8 fits
CASES = [
    (5, 3, 1, 64, dict()),
    (1, 2, 2, 128, dict(adjacent=True, scale=0.75)),
    (33, 4, 2, 96, dict(rot_dim=48)),
    (7, 16, 8, 128, dict(rot_dim=32)),
    (900, 2, 1, 64, dict(sections=[8, 12, 12], interleaved=True)),
    (3, 5, 1, 256, dict()),
    (2000, 3, 2, 80, dict(base=1000.0)),
    (9, 2, 2, 248, dict(rot_dim=16)),
    (33, 4, 2, 40, dict(rot_dim=20)),
    (7, 2, 1, 10, dict(adjacent=True)),
    (6, 2, 1, 7, dict(rot_dim=6)),
    (4, 1, 1, 250, dict(rot_dim=100)),
    (3, 2, 1, 8, dict()),
]
FOUR = [c for c in CASES if c[3] % 8 == 0 and c[4].get("rot_dim", c[3]) % 4 == 0]


def _norm64(x, w, eps):
    x = x.double().cpu().numpy()
    y = x / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    return y if w is None else y * w.double().cpu().numpy()


def _turned(rot, y, positions, sign=1.0):
    n = y.shape[0]
    half = rot.rot_dim // 2
    pos = positions.cpu().numpy().reshape(-1, n)
    theta = sign * np.pi * rot.half_turns.cpu().numpy()[None] * pos[rot.axis_of_pair.cpu().numpy()].T.astype(np.float64)
    c, s = np.cos(theta)[:, None] * rot.scale, np.sin(theta)[:, None] * rot.scale
    z = y.copy()
    i, j = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if rot.adjacent else (slice(0, half), slice(half, 2 * half))
    z[..., i], z[..., j] = y[..., i] * c - y[..., j] * s, y[..., j] * c + y[..., i] * s
    return z


def _inputs(case, dtype, seed, wdtype=None):
    import torch
    n, hq, hk, d, kw = case
    g = torch.Generator().manual_seed(seed)
    rot = Rotary(d, device="cuda:0", **kw)
    q, k, v, gq, gk = (torch.randn((n, h, d), generator=g).mul(2.0).to(dtype).cuda() for h in (hq, hk, hk, hq, hk))
    wd = wdtype or dtype
    qw, kw_ = ((1 + 0.3 * torch.randn(d, generator=g)).to(wd).cuda() for _ in range(2))
    pos = torch.randint(0, 4096, (rot.axes, n) if rot.axes > 1 else (n,), generator=g, dtype=torch.int32).cuda()
    return rot, q, k, v, gq, gk, HeadNorm(qw, kw_, 1e-5), pos


def _near(got, want, bits, size):
    """One rounding of half a step, 2^-bits of the value, and the angles': the kernel's and this file's are within 2^-38 each of the
    exact ones (positions below 2^12, frequencies up to 1), which moves a pair by that of its size; fp64 sums of up to 256 terms
    are far below."""
    got = got.double().cpu().numpy()
    assert (np.abs(got - want) <= 2.0 ** -bits * np.abs(want) + 2.0 ** -37 * size + 1e-44).all()


@pytest.mark.parametrize("dtype, bits", [("float32", 24), ("bfloat16", 8)])
@pytest.mark.parametrize("case", CASES)
def test_forward(gpu, case, dtype, bits):
    import torch
    rot, q, k, _, _, _, norm, pos = _inputs(case, getattr(torch, dtype), 1)
    yq, yk = rot.rotate(q, k, pos, norm=norm)
    for got, x, w in ((yq, q, norm.q_weight), (yk, k, norm.k_weight)):
        y = _norm64(x, w, norm.eps)
        assert got.dtype == x.dtype
        _near(got, _turned(rot, y, pos), bits, np.abs(y).max() * max(rot.scale, 1.0) * 2)
    # in place, and from views with other strides
    n, hq, hk, d, _ = case
    fused = torch.cat([q, k], 1).reshape(n, -1)
    fq, fk = fused[:, :hq * d].view(n, hq, d), fused[:, hq * d:].view(n, hk, d)
    assert all(torch.equal(a, b) for a, b in zip(rot.rotate(fq, fk, pos, norm=norm), (yq, yk)))
    rot.rotate(fq, fk, pos, norm=norm, q_out=fq, k_out=fk)
    assert torch.equal(fq, yq) and torch.equal(fk, yk)
    # rows that start anywhere
    loose = torch.empty(n * hq * d + 1, dtype=q.dtype, device="cuda")[1:].view(n, hq, d)
    loose.copy_(q)
    assert torch.equal(rot.rotate(loose, k, pos, norm=norm)[0], yq)


@pytest.mark.parametrize("value", [0.0, 1e-30, 3e38, float("inf"), float("nan")])
def test_heads_of_zeros_and_of_no_numbers(gpu, value):
    """A head of zeros stays zero; 64 bits hold the squares of the smallest and largest values; NaN and infinity stay in their head."""
    import torch
    rot, q, k, _, _, _, norm, pos = _inputs((4, 2, 1, 64, {}), torch.float32, 2)
    q[1, 1] = value
    y = rot.rotate(q, k, pos, norm=norm)[0]
    if np.isfinite(value):
        z = _norm64(q, norm.q_weight, norm.eps)
        _near(y, _turned(rot, z, pos), 24, np.abs(z).max() * 2)
    else:
        assert bool(y[1, 1].isnan().all())
        y[1, 1] = 0
    assert bool(y.isfinite().all())


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("case", CASES)
def test_append_bf16(gpu, case, dtype):
    """The same bits as the rotation alone gives, rounded to bf16 once; rows that no token names stay as they were."""
    import torch
    rot, q, k, v, _, _, norm, pos = _inputs(case, getattr(torch, dtype), 3)
    n, hq, hk, d, _ = case
    P, pages = 4, n // 4 + 2
    r = np.random.default_rng(n)
    dst = r.permutation(P * pages)[:n].astype(np.int64)
    dst[n // 2] = -1
    kp, vp = (torch.full((pages, P, hk, d), -3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    got = rot.append(q, k, v, pos, torch.from_numpy(dst).cuda(), kp, vp, norm=norm)
    assert got.dtype == torch.bfloat16
    for x, w, y in ((q, norm.q_weight, got), (k, norm.k_weight, None)):
        z = _norm64(x, w, norm.eps)
        rows = y if y is not None else kp.view(-1, hk, d)[torch.from_numpy(dst[dst >= 0]).cuda()]
        want = _turned(rot, z, pos)
        _near(rows, want if y is not None else want[dst >= 0], 8, np.abs(z).max() * max(rot.scale, 1.0) * 2)
    keep = np.setdiff1d(np.arange(P * pages), dst[dst >= 0])
    live = torch.from_numpy(dst[dst >= 0]).cuda()
    assert torch.equal(vp.view(-1, hk, d)[live], v[torch.from_numpy(dst >= 0).cuda()].to(torch.bfloat16))
    for p in (kp, vp):
        assert bool((p.view(-1, hk, d)[torch.from_numpy(keep).cuda()] == -3.0).all())


def _codes_match(got, gs, want64, slack):
    """Codes and scales of want64 (float64), but where a value lies within its slack (d,) of a border between two codes, or a group's
    largest of the border between two scales."""
    d = want64.shape[-1]
    x = np.concatenate([want64, np.zeros(want64.shape[:-1] + (f4.width(d) - d,))], -1).reshape(want64.shape[:-1] + (-1, 32))
    each = np.concatenate([slack, np.zeros(f4.width(d) - d)]).reshape(-1, 32)
    slack = each.max(-1)
    s = f4.scales_of(x)
    unit = np.ldexp(1.0, s.astype(int) - 127)
    top = np.abs(x).max(-1) / unit
    near = (np.abs(top - 7.0) < slack / unit) | (np.abs(top - 3.5) < slack / unit)
    assert np.all((gs == s) | near) and np.mean(near) < 0.01
    c = np.stack([got & 15, got >> 4], -1).reshape(x.shape)
    t = f4.steps(x, s)
    want = f4.codes_of(t)
    borders = np.array([0.0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    close = np.abs(np.abs(t)[..., None] - borders).min(-1) < each / unit[..., None]
    ok = (c == want) | close | near[..., None]
    inside = np.arange(x.shape[-2] * 32).reshape(x.shape[-2:]) < d
    assert np.all(ok | ~inside) and np.mean(close & inside) < 0.01


@pytest.mark.parametrize("normed", [True, False])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("case", FOUR)
def test_append_in_4_bits(gpu, case, dtype, normed):
    import torch
    rot, q, k, v, _, _, norm, pos = _inputs(case, getattr(torch, dtype), 4)
    n, hq, hk, d, _ = case
    P, pages = 16, n // 16 + 2
    r = np.random.default_rng(n)
    before = f4.random_pool(r, pages, hk, P, d)
    pool = KV4Pool.of(*(torch.from_numpy(a).cuda() for a in before), head_dim=d)
    dst = r.permutation(P * pages)[:n].astype(np.int64)
    if n > 2:
        dst[n // 2], dst[0] = -1, P * pages + 5
    norm = norm if normed else None
    q2 = rot.append(q, k, v, pos, torch.from_numpy(dst).cuda(), pool, norm=norm)
    live = (dst >= 0) & (dst < P * pages)
    page, slot = dst[live] // P, dst[live] % P
    y = _norm64(k, norm.k_weight, norm.eps) if normed else k.double().cpu().numpy()
    k64 = _turned(rot, y, pos)[live]
    arrays = [a.cpu().numpy() for a in pool.rows()]
    # elements that neither the norm nor the rotation changes are exact, ties among them
    slack = np.where(normed | (np.arange(d) < rot.rot_dim), 2.0 ** -36 * np.abs(y).max(), 0.0)
    _codes_match(arrays[0][page, :, slot], arrays[1][page, :, slot], k64, slack)
    c, s = f4.quantize(v.double().cpu().numpy()[live])  # v as it is: to the bit, pad columns left alone
    m = d // 2
    assert np.array_equal(arrays[2][page, :, slot][..., :m], c[..., :m])
    assert np.array_equal(arrays[2][page, :, slot][..., m:], before[2][page, :, slot][..., m:])
    assert np.array_equal(arrays[3][page, :, slot], s)
    for a, b in zip(arrays, before):  # rows of no token
        a, b = a.copy(), b.copy()
        a[page, :, slot] = b[page, :, slot] = 0
        assert np.array_equal(a, b)
    # q as into a bf16 cache
    kp, vp = (torch.empty((n + 1, 1, hk, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = torch.arange(n, device="cuda")
    assert torch.equal(q2, rot.append(q, k, v, pos, at, kp, vp, norm=norm))


@pytest.mark.parametrize("d", [8, 64, 80, 128, 256])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_pool_append(gpu, d, dtype):
    """Keys and values without norm or rotation: the codes to the bit, over all scales, ties, zeros, and no numbers."""
    import torch
    r = np.random.default_rng(d)
    n, H, P = 70, 3, 16
    x = []
    for _ in range(2):
        a = r.standard_normal((n, H, d)) * np.exp2(r.integers(-130, 120, (n, H, 1)))
        a[:20] = r.choice([0, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5, 6, 7, -0.25, -2.5, 3.4999, 7.001], (20, H, d))
        a[20] = 0.0
        a[21, 0, 0], a[22, 1, d - 1], a[23, 2, 3] = np.inf, np.nan, 3.3e38
        x.append(torch.from_numpy(a.astype(np.float32)).to(getattr(torch, dtype)).cuda())
    pool = KV4Pool(7, P, H, d, "cuda:0")
    dst = r.permutation(7 * P)[:n].astype(np.int64)
    pool.append(x[0].transpose(0, 1).contiguous().transpose(0, 1), x[1], torch.from_numpy(dst).cuda())
    page, slot = dst // P, dst % P
    rows = pool.rows()
    for t, codes, scales in ((x[0], *rows[:2]), (x[1], *rows[2:])):
        c, s = f4.quantize(t.double().cpu().numpy())
        bad = np.repeat(s == 255, 16, -1)
        got = codes.cpu().numpy()[page, :, slot]
        assert np.array_equal(scales.cpu().numpy()[page, :, slot], s)
        m = d // 2
        assert np.array_equal(np.where(bad, 0, got)[..., :m], np.where(bad, 0, c)[..., :m])


def _grads64(rot, x, w, g, eps, pos):
    x, g = x.double().cpu().numpy(), _turned_back(rot, g, pos)
    w = w.double().cpu().numpy()
    r = 1.0 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    xh, gw = x * r, g * w
    dx = r * (gw - xh * (gw * xh).mean(-1, keepdims=True))
    return dx, (g * xh).sum((0, 1)), np.abs(r * gw).max() + np.abs(r * xh).max() * np.abs(gw * xh).mean(-1).max(), \
        (np.abs(g) * np.abs(xh)).sum((0, 1)).max()


def _turned_back(rot, g, pos):
    return _turned(rot, g.double().cpu().numpy(), pos, -1.0)


@pytest.mark.parametrize("dtype, wdtype", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("case", CASES)
def test_gradients_are_the_formulas(gpu, case, dtype, wdtype):
    import torch
    rot, q, k, _, gq, gk, norm, pos = _inputs(case, getattr(torch, dtype), 5, getattr(torch, wdtype))
    leaves = [x.requires_grad_() for x in (q, k, norm.q_weight, norm.k_weight)]
    y = rot.rotate(q, k, pos, norm=norm)
    with torch.no_grad():
        plain = rot.rotate(q, k, pos, norm=norm)
    assert all(torch.equal(a, b) for a, b in zip(y, plain))
    got = torch.autograd.grad(y, leaves, (gq, gk))
    bits, wbits = (24 if t == "float32" else 8 for t in (dtype, wdtype))
    for x, w, g, dx, dw in ((q, norm.q_weight, gq, got[0], got[2]), (k, norm.k_weight, gk, got[1], got[3])):
        assert dx.dtype == x.dtype and dw.dtype == w.dtype
        wx, ww, size, wsize = _grads64(rot, x.detach(), w.detach(), g, norm.eps, pos)
        _near(dx, wx, bits, 4 * size * max(rot.scale, 1.0))
        _near(dw, ww, wbits, 4 * wsize * max(rot.scale, 1.0))
    again = torch.autograd.grad(rot.rotate(q, k, pos, norm=norm), leaves, (gq, gk))
    assert all(torch.equal(a, b) for a, b in zip(got, again))


def test_gradients_are_the_differences(gpu):
    """f = sum of y g along a direction: central differences of a step 2^-8 in fp32 inputs. The third derivative of a norm of
    numbers about 1 stays below 2^6 of the sizes, so they are within 2^-16 2^6 / 6 of them, and y's rounding, 2^-24 of it over a step of
    2^-8, within 2^-16 of the sum of |y g| each."""
    import torch
    rot, q, k, _, gq, gk, norm, pos = _inputs((6, 2, 1, 32, {}), torch.float32, 6)
    leaves = [x.requires_grad_() for x in (q, k, norm.q_weight, norm.k_weight)]
    got = torch.autograd.grad(rot.rotate(q, k, pos, norm=norm), leaves, (gq, gk))
    gen = torch.Generator().manual_seed(1)

    def f(args):
        with torch.no_grad():
            y = rot.rotate(args[0], args[1], pos, norm=HeadNorm(args[2], args[3], norm.eps))
        return sum((a.double() * g.double()).sum().item() for a, g in zip(y, (gq, gk))), \
            sum((a.double() * g.double()).abs().sum().item() for a, g in zip(y, (gq, gk)))

    for i, x in enumerate(leaves):
        for _ in range(4):
            v = torch.randn(x.shape, generator=gen).cuda()
            v /= v.norm()
            base = [t.detach() for t in leaves]
            side = []
            for h in (2.0 ** -8, -2.0 ** -8):
                moved = list(base)
                moved[i] = (base[i] + h * v)
                side.append((moved[i].double(), *f(moved)))
            step = (side[0][0] - side[1][0])
            # along the step that fp32 took
            want = (got[i].double() * step).sum().item()
            size = side[0][2]
            assert abs((side[0][1] - side[1][1]) - want) <= (2.0 ** -8) * 2.0 ** -16 * 2.0 ** 6 * size + 2 * 2.0 ** -24 * size


def test_some_of_them_alone(gpu):
    """Only weights, only q, one output used, strides of 0 from a sum, and no tokens or heads."""
    import torch
    rot, q, k, _, gq, gk, norm, pos = _inputs(CASES[0], torch.float32, 7)
    full = [x.clone().requires_grad_() for x in (q, k, norm.q_weight, norm.k_weight)]
    want = torch.autograd.grad(rot.rotate(full[0], full[1], pos, norm=HeadNorm(full[2], full[3], norm.eps)), full, (gq, gk))
    w = norm.k_weight.clone().requires_grad_()
    yq, yk = rot.rotate(q, k, pos, norm=HeadNorm(norm.q_weight, w, norm.eps))
    assert yk.requires_grad and not yq.requires_grad
    assert torch.equal(torch.autograd.grad(yk, w, gk)[0], want[3])
    yq, yk = rot.rotate(full[0], k, pos, norm=norm)
    assert yq.requires_grad and not yk.requires_grad
    assert torch.equal(torch.autograd.grad(yq, full[0], gq)[0], want[0])
    yq, yk = rot.rotate(full[0], full[1], pos, norm=HeadNorm(full[2], full[3], norm.eps))
    got = torch.autograd.grad(yk, full, gk.transpose(1, 2).contiguous().transpose(1, 2), allow_unused=True)
    assert got[0] is None and got[2] is None and torch.equal(got[1], want[1]) and torch.equal(got[3], want[3])
    yq, yk = rot.rotate(full[0], full[1], pos, norm=HeadNorm(full[2], full[3], norm.eps))
    dq, = torch.autograd.grad(yq.sum(), full[0])
    ones = torch.ones_like(q)
    assert torch.equal(dq, torch.autograd.grad(rot.rotate(full[0], k, pos, norm=norm)[0], full[0], ones)[0])
    none = torch.empty((0, 3, 64), device="cuda").requires_grad_()
    yq, yk = rot.rotate(none, torch.empty((0, 1, 64), device="cuda"), pos[:0], norm=HeadNorm(full[2], full[3]))
    dw, = torch.autograd.grad(yq.sum() + yk.sum(), full[2])
    assert bool((dw == 0).all())
    yq, yk = rot.rotate(q[:, :0], k, pos, norm=norm)
    assert yq.shape == (5, 0, 64) and torch.equal(yk, rot.rotate(q, k, pos, norm=norm)[1])


def test_streams_and_graphs(gpu):
    """Forward, backward and the 4-bit append on another stream, and captured, replayed on new values between eager work."""
    import torch
    rot, q, k, v, gq, gk, norm, pos = _inputs((300, 4, 2, 64, {}), torch.float32, 8)
    leaves = [x.requires_grad_() for x in (q, k, norm.q_weight, norm.k_weight)]
    pool, other = KV4Pool(24, 16, 2, 64, "cuda:0"), KV4Pool(24, 16, 2, 64, "cuda:0")
    dst = torch.arange(300, device="cuda")

    def step(p):
        y = rot.rotate(q, k, pos, norm=norm)
        got = torch.autograd.grad(y, leaves, (gq, gk))
        a = rot.append(q.detach(), k.detach(), v, pos, dst, p, norm=HeadNorm(leaves[2].detach(), leaves[3].detach(), norm.eps))
        return (*(x.detach() for x in y), *got, a)

    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        for _ in range(3):
            got = step(pool)
    torch.cuda.synchronize()
    want = step(other)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and torch.equal(pool.k, other.k)
    del got, want  # no eager graph of these leaves lives while the capture runs
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        got = step(pool)
    for i in range(4):
        with torch.no_grad():
            for x in (q, k, v, gq, gk, leaves[2]):
                x.copy_(torch.randn(x.shape, generator=torch.Generator().manual_seed(i)))
        graph.replay()
        want = step(other)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i
        assert torch.equal(pool.k, other.k) and torch.equal(pool.v_scales, other.v_scales), i


def test_refusals(gpu):
    import torch
    rot, q, k, v, _, _, norm, pos = _inputs(CASES[0], torch.float32, 9)
    with pytest.raises(ValueError, match="inverse"):
        rot.rotate(q, k, pos, norm=norm, inverse=True)
    with pytest.raises(ValueError):
        HeadNorm(norm.q_weight, norm.k_weight.bfloat16())
    with pytest.raises(ValueError):
        HeadNorm(norm.q_weight, norm.k_weight[:-1])
    for eps in (-1.0, float("nan"), float("inf")):
        with pytest.raises(ValueError):
            HeadNorm(norm.q_weight, norm.k_weight, eps)
    for w in (norm.q_weight[:32].contiguous(), norm.q_weight.double(), norm.q_weight.cpu(), torch.ones(128, device="cuda")[::2]):
        with pytest.raises(ValueError):
            rot.rotate(q, k, pos, norm=HeadNorm(w, w))
    w = norm.q_weight.clone().requires_grad_()
    with pytest.raises(ValueError, match="gradients"):
        rot.rotate(q, k, pos, norm=HeadNorm(w, w), q_out=torch.empty_like(q))
    with pytest.raises(ValueError, match="bit patterns"):
        rot.rotate(q.bfloat16().view(torch.int16), k.bfloat16().view(torch.int16), pos, norm=HeadNorm(w, w))
    pool, dst = KV4Pool(2, 16, 1, 64, "cuda:0"), torch.arange(5, device="cuda")
    with pytest.raises(ValueError):
        rot.append(q, k, v, pos, dst, pool, pool)
    with pytest.raises(ValueError):
        rot.append(q, k, v, pos, dst, KV4Pool(2, 16, 2, 64, "cuda:0"))
    with pytest.raises(ValueError):
        rot.append(q, k, v, pos, dst, KV4Pool(2, 16, 1, 128, "cuda:0"))
    with pytest.raises(ValueError):
        rot.append(q, k, v, pos, dst.int(), pool)
    with pytest.raises(ValueError):
        rot.append(q, k, v, pos, dst[:4], pool)
    with pytest.raises(ValueError, match="multiple of 4"):
        Rotary(64, rot_dim=30, device="cuda:0").append(q, k, v, pos, dst, pool)
    with pytest.raises(ValueError, match="shares memory"):
        pool = KV4Pool(40, 16, 1, 64, "cuda:0")
        out = pool.k.view(torch.bfloat16).view(-1)[:5 * 3 * 64].view(5, 3, 64)
        rot.append(q, k, v, pos, dst, pool, q_out=out)
    for bad in (dict(k=k[:, :, :32]), dict(v=v.bfloat16()), dict(k=k.double()), dict(k=k.cpu()), dict(dst_rows=dst[:3])):
        with pytest.raises(ValueError):
            pool.append(**{**dict(k=k, v=v, dst_rows=dst), **bad})


def test_gradients_of_gradients_are_refused(gpu):
    """create_graph gives the same first gradients; what would differentiate them raises."""
    import torch
    from exactattention_amd.step import HeadNorm, Rotary
    gen = torch.Generator(device="cuda").manual_seed(3)
    q, k = (torch.randn((5, h, 64), device="cuda", generator=gen).requires_grad_() for h in (4, 2))
    w = [(1 + 0.1 * torch.randn(64, device="cuda", generator=gen)).requires_grad_() for _ in range(2)]
    rot, pos = Rotary(64), torch.arange(5, dtype=torch.int32, device="cuda")
    loss = lambda: sum(x.square().sum() for x in rot.rotate(q, k, pos, norm=HeadNorm(*w, 1e-6)))  # noqa: E731
    plain = torch.autograd.grad(loss(), (q, k, *w))
    again = torch.autograd.grad(loss(), (q, k, *w), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))
    with pytest.raises(RuntimeError):
        again[0].sum().backward()

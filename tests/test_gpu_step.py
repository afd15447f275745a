"""GPU: the step plan against a plain restatement over Python integers, and the rotary positions against
the formula in 64 bits.

The rotation is computed in fp64 and rounded once. Its fp64 value is within 2^-45 of the exact one,
relative to |x| + |y| of the pair (angles below 2^21 half turns: the product's rounding is recovered by
an FMA, the frequency's own is 2^-53 of the angle, at most 2^-32 half turns at those angles, and the
reference below takes the same angle in fp64: both err by at most 2^-31), so an output differs from the
rounded reference only next to the midpoint of two values: by half a step (torch.finfo(t).eps / 2
relative) plus 2^-30 (|x| + |y|).
"""

import numpy as np
import pytest

pytestmark = pytest.mark.gpu


# ---------------------------------------------------------------------------
# step plan
# ---------------------------------------------------------------------------

def _plan_reference(L, c, bt, free, nf, P, N, T, slots, max_len):
    """The plan in plain integers, or None where it does not fit."""
    S, W = bt.shape
    if len(set(slots)) != len(slots) or any(not 0 <= s < S for s in slots) or any(x < 0 for x in (*L, *c)):
        return None
    if any(a + b > min(W * P, max_len) or b > T for a, b in zip(L, c)) or sum(c) > N:
        return None
    bt = bt.copy()
    top = nf
    for b, s in enumerate(slots):
        for p in range(-(-L[b] // P), -(-(L[b] + c[b]) // P)):
            if top == 0:
                return None
            top -= 1
            bt[s, p] = free[top]
    dst, pos, seq, rows = [], [], [], []
    kv = np.zeros((len(L), T), np.int32)
    for b, s in enumerate(slots):
        for j in range(c[b]):
            p = L[b] + j
            dst.append(int(bt[s, p // P]) * P + p % P)
            pos.append(p)
            seq.append(b)
            rows.append(b * T + j)
            kv[b, j] = p + 1
    pad = [-1] * (N - len(dst))
    return dict(dst_rows=dst + pad, positions=pos + pad, seq_of=seq + pad, q_rows=rows + pad, kv_len=kv,
                seq_len=[a + b for a, b in zip(L, c)], num_free=[top], bt=bt)


def _i32(x):
    import torch
    return torch.tensor(np.asarray(x), dtype=torch.int32, device="cuda")


def _run_plan(L, c, bt, free, nf, P, N, T, slots=None, max_len=None):
    from exactattention_amd.step import StepPlan
    plan = StepPlan(len(L), N, T)
    btd = _i32(bt)
    plan.build(_i32(L), _i32(c), btd, _i32(free), _i32([nf]), P, slots=None if slots is None else _i32(slots),
               max_seq_len=max_len)
    got = {n: getattr(plan, n).cpu().numpy() for n in ("dst_rows", "positions", "seq_of", "q_rows", "kv_len", "seq_len", "num_free",
                                                       "status")}
    got["bt"] = btd.cpu().numpy()
    return plan, got


def _check_plan(L, c, bt, free, nf, P, N, T, slots=None, max_len=None, status=0):
    L, c = [int(x) for x in L], [int(x) for x in c]
    want = _plan_reference(L, c, bt, free, nf, P, N, T, list(range(len(L))) if slots is None else [int(s) for s in slots],
                           max_len or 1 << 31)
    plan, got = _run_plan(L, c, bt, free, nf, P, N, T, slots, max_len)
    assert int(got["status"][0]) == status
    if status:
        assert want is None
        with pytest.raises(RuntimeError):
            plan.check()
        for n in ("dst_rows", "positions", "seq_of", "q_rows"):
            assert (got[n] == -1).all()
        assert (got["kv_len"] == 0).all() and (got["bt"] == bt).all()
        assert got["seq_len"].tolist() == L and got["num_free"].tolist() == [nf]
        return
    plan.check()
    for n, w in want.items():
        assert np.array_equal(got[n].reshape(-1), np.asarray(w).reshape(-1)), n


def _plan_case(rng, B, P, kv, tok, zeros=True):
    L = rng.integers(0, kv + 1, B)
    c = rng.integers(0 if zeros else 1, tok + 1, B)
    W = -(-(kv + tok) // P) + 1
    held, need = -(-L // P), -(-(L + c) // P) + L // -P
    pages = int(held.sum() + need.sum()) + 3
    perm = rng.permutation(pages).astype(np.int32)
    S = B + 3
    slots = rng.permutation(S)[:B].astype(np.int32)
    bt = np.full((S, W), -7, np.int32)
    at = 0
    for b in range(B):
        bt[slots[b], :held[b]] = perm[at:at + held[b]]
        at += held[b]
    return L, c, bt, perm[at:], slots


@pytest.mark.parametrize("B, P, kv, tok, pad", [
    (1, 16, 0, 1, 0), (1, 1, 5, 1, 0), (1, 64, 64, 1, 2), (7, 16, 100, 1, 0), (33, 16, 500, 40, 9), (64, 1, 30, 3, 1),
    (1023, 16, 60, 2, 0), (1024, 32, 60, 1, 5), (1025, 16, 60, 3, 0), (3000, 64, 300, 7, 100), (8192, 16, 40, 2, 0),
    (5, 128, 4000, 3000, 50),
])
def test_step_plan(gpu, B, P, kv, tok, pad):
    rng = np.random.default_rng(B * 1000 + kv)
    L, c, bt, free, slots = _plan_case(rng, B, P, kv, tok)
    _check_plan(L, c, bt, free, len(free), P, int(c.sum()) + pad, tok, slots)


def test_step_plan_rows_in_order(gpu):
    """slots None: sequence b is row b; a stack that holds exactly the step's pages; more entries than its height."""
    rng = np.random.default_rng(3)
    L, c, bt, free, _ = _plan_case(rng, 9, 16, 50, 20)
    bt = np.full((9, bt.shape[1]), 99, np.int32)
    need = int((-(-(L + c) // 16) + L // -16).sum())
    _check_plan(L, c, bt, free, need, 16, int(c.sum()), 20)
    _check_plan(L, c, bt, free, need - 1, 16, int(c.sum()), 20, status=1)


def test_step_plan_of_nothing(gpu):
    _check_plan([], [], np.zeros((2, 3), np.int32), np.arange(4), 4, 16, 5, 2)
    _check_plan([0, 16, 3], [0, 0, 0], np.zeros((3, 3), np.int32), np.zeros(0, np.int32), 0, 16, 0, 1)


@pytest.mark.parametrize("what, status", [("pages", 1), ("long", 2), ("table", 2), ("tokens", 4), ("pad", 4), ("negative", 8),
                                          ("count", 8), ("row", 8), ("twice", 8), ("stack", 8)])
def test_step_plan_that_does_not_fit(gpu, what, status):
    rng = np.random.default_rng(11)
    B, P = 1500, 16
    L, c, bt, free, slots = _plan_case(rng, B, P, 90, 5, zeros=False)
    N, T, nf, max_len = int(c.sum()), 5, len(free), None
    if what == "pages":
        nf = 2
    elif what == "long":
        max_len = int((L + c).max()) - 1
    elif what == "table":
        L[700] = bt.shape[1] * P - c[700] + 1
    elif what == "tokens":
        N -= 1
    elif what == "pad":
        T, c[-1] = int(c[:-1].max()), int(c[:-1].max()) + 1
        N += 9
    elif what == "negative":
        L[3] = -1
    elif what == "count":
        c[1499] = -1
    elif what == "row":
        slots[5] = bt.shape[0]
    elif what == "twice":
        slots[1400] = slots[2]
    else:
        nf = len(free) + 1
    want_extra = {"table": 1}  # a sequence that long may need more pages as well
    plan, got = _run_plan(L, c, bt, free, nf, P, N, T, slots, max_len)
    assert int(got["status"][0]) & status
    assert int(got["status"][0]) & ~(status | want_extra.get(what, 0)) == 0
    assert (got["dst_rows"] == -1).all() and (got["kv_len"] == 0).all() and (got["bt"] == bt).all()
    assert got["seq_len"].tolist() == L.tolist() and got["num_free"].tolist() == [nf]


def test_step_plan_largest_counts(gpu):
    """Sums past 32 bits are refused, not wrapped."""
    B = 4
    plan, got = _run_plan([0] * B, [1 << 30] * B, np.zeros((B, 4), np.int32), np.arange(8), 8, 1 << 30, 16, 16)
    assert int(got["status"][0]) & 4 and (got["dst_rows"] == -1).all()


# ---------------------------------------------------------------------------
# rotary positions
# ---------------------------------------------------------------------------

def _turn64(x, positions, inv_freq, axis, rot, adjacent, inverse, scale, offset=0):
    import torch
    x = x.double().cpu().clone()
    p = positions.cpu().view(-1, x.shape[0]).double() + offset
    ang = torch.stack([p[a] * float(f) for a, f in zip(axis, inv_freq)], 1)[:, None]
    c, s = ang.cos() * scale, ang.sin() * scale * (-1 if inverse else 1)
    i = torch.arange(rot // 2)
    i0, i1 = (2 * i, 2 * i + 1) if adjacent else (i, i + rot // 2)
    a, b = x[..., i0], x[..., i1]
    size = torch.zeros_like(x)
    size[..., i0] = size[..., i1] = (a.abs() + b.abs()) * scale
    x[..., i0], x[..., i1] = a * c - b * s, b * c + a * s
    return x, size


def _close(got, want, size, moved=True):
    import torch
    eps = torch.finfo(got.dtype).eps / 2
    tol = eps * want.abs() * (1 + 2.0 ** -10) + size * 2.0 ** -30 + torch.finfo(got.dtype).tiny * eps
    err = (got.double().cpu() - want).abs()
    bad = ~((err <= tol) | (torch.isnan(want) & torch.isnan(got.double().cpu())))
    assert not bool(bad.any()), f"{int(bad.sum())} of {bad.numel()} off, worst {float((err / tol)[bad].max())} tolerances"


CASES = [
    # N, Hq, Hkv, d, rot, axes, interleaved, adjacent, dtype
    (1, 1, 1, 8, 8, 1, False, False, "bf16"), (1, 32, 8, 128, 128, 1, False, False, "bf16"),
    (3, 5, 1, 64, 64, 1, False, True, "bf16"), (17, 4, 2, 128, 64, 3, True, False, "bf16"),
    (33, 6, 3, 96, 48, 2, False, True, "fp32"), (5, 2, 2, 80, 80, 3, False, False, "bf16"),
    (7, 3, 1, 20, 12, 1, False, False, "fp32"), (7, 3, 1, 22, 10, 2, True, True, "bf16"), (9, 2, 1, 13, 6, 1, False, False, "bf16"),
    (2, 1, 1, 256, 256, 4, True, False, "bf16"), (4100, 2, 1, 64, 64, 2, False, False, "bf16"), (4097, 1, 1, 16, 16, 1, False, True, "fp32"),
]


def _rotary_inputs(N, Hq, Hkv, d, rot, axes, dtype, seed=0, maxpos=4096):
    import torch
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dt = torch.float32 if dtype == "fp32" else torch.bfloat16
    qkv = torch.empty((N, (Hq + 2 * Hkv) * d), dtype=dt, device="cuda").normal_(generator=gen)
    q = qkv[:, :Hq * d].view(N, Hq, d)
    k = qkv[:, Hq * d:(Hq + Hkv) * d].view(N, Hkv, d)
    v = qkv[:, (Hq + Hkv) * d:].view(N, Hkv, d)
    pos = torch.randint(0, maxpos, (axes, N), generator=gen, device="cuda", dtype=torch.int32)
    return q, k, v, pos


def _axes(half, axes, interleaved):
    from exactattention_amd.step import _deal
    sec = [half // axes] * axes
    sec[-1] += half - sum(sec)
    return sec, _deal(list(sec), half, interleaved)


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("inverse", [False, True])
def test_rotate(gpu, case, inverse):
    from exactattention_amd.step import Rotary
    N, Hq, Hkv, d, rot, axes, inter, adj, dtype = case
    q, k, _, pos = _rotary_inputs(N, Hq, Hkv, d, rot, axes, dtype, seed=N + d)
    sec, axis = _axes(rot // 2, axes, inter)
    r = Rotary(d, rot_dim=rot, sections=sec, interleaved=inter, adjacent=adj, scale=1.25)
    qo, ko = r.rotate(q, k, pos, inverse=inverse)
    f = 10000.0 ** (-np.arange(rot // 2) / (rot // 2))
    for x, y in ((q, qo), (k, ko)):
        assert y.dtype == x.dtype and y.is_contiguous()
        w, size = _turn64(x, pos, f, axis, rot, adj, inverse, 1.25)
        _close(y, w, size)
        assert bool((y[..., rot:] == x[..., rot:]).all())
    # in place: the same values
    q2, k2 = q.clone(), k.clone()
    r.rotate(q2, k2, pos, inverse=inverse, q_out=q2, k_out=k2)
    assert bool((q2 == qo).all()) and bool((k2 == ko).all())


def test_rotate_far_positions(gpu):
    import torch
    from exactattention_amd.step import Rotary
    q, k, _, _ = _rotary_inputs(6, 2, 1, 64, 64, 1, "fp32")
    pos = torch.tensor([0, 1, -5, 1 << 20, (1 << 20) + 1, 131071], dtype=torch.int32, device="cuda")
    qo, _ = Rotary(64).rotate(q, k, pos)
    w, size = _turn64(q, pos, 10000.0 ** (-np.arange(32) / 32), [0] * 32, 64, False, False, 1.0)
    _close(qo, w, size)
    assert bool((qo[0] == q[0]).all())  # position 0 changes nothing


def test_rotate_inverse_is_the_gradient(gpu):
    """sum(g * rotate(x)) has the gradient rotate(g, inverse): checked against the formula's autograd in
    64 bits and, along a direction, against differences (the map is linear)."""
    import torch
    from exactattention_amd.step import Rotary
    N, H, d, rot = 19, 3, 48, 32
    x, g, _, pos = _rotary_inputs(N, H, H, d, rot, 2, "fp32", seed=5)
    x, g = x.contiguous(), g.contiguous()
    sec, axis = _axes(rot // 2, 2, False)
    r = Rotary(d, rot_dim=rot, sections=sec, scale=0.75)
    dx, _ = r.rotate(g, g, pos, inverse=True)
    x64 = x.double().cpu().requires_grad_()
    p = pos.cpu().double()
    ang = torch.stack([p[a] * float(f) for a, f in zip(axis, 10000.0 ** (-np.arange(rot // 2) / (rot // 2)))], 1)[:, None]
    a, b = x64[..., :rot // 2], x64[..., rot // 2:rot]
    y = torch.cat([0.75 * (a * ang.cos() - b * ang.sin()), 0.75 * (b * ang.cos() + a * ang.sin()), x64[..., rot:]], -1)
    (y * g.double().cpu()).sum().backward()
    _close(dx, x64.grad, g.double().cpu().abs().amax(-1, keepdim=True).expand_as(x64) * 2)
    u = torch.randn(x.shape, generator=torch.Generator().manual_seed(1)).cuda()
    y0, _ = r.rotate(x, x, pos)
    y1, _ = r.rotate(x + u, x, pos)
    lhs = float(((y1.double() - y0.double()) * g.double()).sum())
    rhs = float((dx.double() * u.double()).sum())
    # every output rounds by 2^-24 of values below 8, times |g| below 6, over the elements
    assert abs(lhs - rhs) <= x.numel() * 4 * 2.0 ** -24 * 8 * 6


@pytest.mark.parametrize("case", CASES)
def test_rotary_append(gpu, case):
    import torch
    from exactattention_amd.step import Rotary
    N, Hq, Hkv, d, rot, axes, inter, adj, dtype = case
    q, k, v, pos = _rotary_inputs(N, Hq, Hkv, d, rot, axes, dtype, seed=2 * N + d)
    sec, axis = _axes(rot // 2, axes, inter)
    r = Rotary(d, rot_dim=rot, sections=sec, interleaved=inter, adjacent=adj)
    P = 16
    pages = -(-N // P) + 2
    gen = np.random.default_rng(N)
    dst = gen.permutation(pages * P)[:N].astype(np.int64)
    if N > 4:
        dst[[1, -1]] = -1            # padding
        dst[2] = pages * P           # a row outside the pool
    kp = torch.randn(pages, P, Hkv, d, device="cuda").bfloat16()
    vp = torch.randn(pages, P, Hkv, d, device="cuda").bfloat16()
    k0, v0 = kp.clone(), vp.clone()
    rows = gen.permutation(N + 5)[:N].astype(np.int64)
    if N > 4:
        rows[0] = -1
    qo = torch.full((N + 5, Hq, d), 3.0, dtype=torch.bfloat16, device="cuda")
    ret = r.append(q, k, v, pos, torch.from_numpy(dst).cuda(), kp, vp, q_rows=torch.from_numpy(rows).cuda(), q_out=qo, pos_offset=3)
    assert ret is qo
    f = 10000.0 ** (-np.arange(rot // 2) / (rot // 2))
    wq, sq = _turn64(q, pos, f, axis, rot, adj, False, 1.0, 3)
    wk, sk = _turn64(k, pos, f, axis, rot, adj, False, 1.0, 3)
    keep = rows >= 0
    _close(qo.cpu()[rows[keep]], wq[keep], sq[keep])
    other = np.setdiff1d(np.arange(N + 5), rows)
    assert bool((qo.cpu()[other] == 3.0).all())  # rows no token names stay as they were
    put = (dst >= 0) & (dst < pages * P)
    kf, vf = kp.view(-1, Hkv, d).cpu(), vp.view(-1, Hkv, d).cpu()
    _close(kf[dst[put]], wk[put], sk[put])
    assert bool((vf[dst[put]] == v.cpu()[put].bfloat16()).all())
    other = np.setdiff1d(np.arange(pages * P), dst[put])
    assert bool((kf[other] == k0.view(-1, Hkv, d).cpu()[other]).all()) and bool((vf[other] == v0.view(-1, Hkv, d).cpu()[other]).all())


def test_rotary_append_without_rows(gpu):
    """q_out None: a new tensor in token order; int16 bit patterns; another stream than the default."""
    import torch
    from exactattention_amd.step import Rotary
    q, k, v, pos = _rotary_inputs(40, 4, 2, 128, 128, 1, "bf16")
    r = Rotary(128)
    kp, vp = (torch.zeros(3, 16, 2, 128, dtype=torch.int16, device="cuda") for _ in range(2))
    dst = torch.arange(40, device="cuda")
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        qo = r.append(q.view(torch.int16), k.view(torch.int16), v.view(torch.int16), pos[0], dst, kp, vp)
    st.synchronize()
    q2, k2 = r.rotate(q, k, pos)
    assert bool((qo == q2).all()) and bool((kp.view(torch.bfloat16).view(-1, 2, 128)[:40] == k2).all())
    assert bool((vp.view(-1, 2, 128)[:40] == v.view(torch.int16)).all())


def test_rotary_values_at_the_edges(gpu):
    """Infinities, NaN, zeros and subnormal values of a head, and bf16 ties: turned by no angle they come back
    as they are (fp32 values rounded once, to even)."""
    import torch
    from exactattention_amd.step import Rotary
    x = torch.zeros(1, 1, 16, device="cuda")
    x[0, 0, :8] = torch.tensor([1.0 + 2.0 ** -8, 1.0 + 3 * 2.0 ** -8, -1.0 - 2.0 ** -8, 2.0 ** -133, 3.0e38, 2.0 ** -140, 1.0 + 2.0 ** -8 + 2.0 ** -23,
                                 3.4e38])
    r = Rotary(16)
    pool = torch.zeros(1, 1, 1, 16, dtype=torch.bfloat16, device="cuda")
    pool2 = torch.zeros_like(pool)
    zero = torch.zeros(1, dtype=torch.int32, device="cuda")
    dst = torch.zeros(1, dtype=torch.int64, device="cuda")
    qo = r.append(x, x, x, zero, dst, pool, pool2)
    assert bool((qo == x.bfloat16()).all()) and bool((pool.view(-1) == x.bfloat16().view(-1)).all())
    assert bool((pool2.view(-1) == x.bfloat16().view(-1)).all())
    y = torch.tensor([float("inf"), float("nan"), -float("inf"), 1.0] * 4, device="cuda").view(1, 1, 16).bfloat16()
    qo, _ = Rotary(16, rot_dim=8).rotate(y, y, zero + 5)
    assert bool((qo[..., 8:].view(torch.int16) == y[..., 8:].view(torch.int16)).all())  # past rot_dim: the bits
    assert bool(torch.isnan(qo[..., 1]).all()) and not bool(torch.isfinite(qo[..., :3]).any()) and bool(torch.isfinite(qo[..., 3]).all())


def test_rotary_refuses_on_the_device(gpu):
    import torch
    from exactattention_amd.step import Rotary, StepPlan
    q, k, v, pos = _rotary_inputs(4, 2, 1, 64, 64, 2, "bf16")
    r = Rotary(64, sections=[16, 16])
    pool = torch.zeros(1, 16, 1, 64, dtype=torch.bfloat16, device="cuda")
    dst = torch.arange(4, device="cuda")
    bad = [lambda: r.rotate(q, k, pos[0]), lambda: r.rotate(q, k, pos.long()), lambda: r.rotate(q, k[:3], pos),
           lambda: r.rotate(q, k.float(), pos), lambda: r.rotate(q.half(), k.half(), pos), lambda: r.rotate(q[..., :32], k, pos),
           lambda: r.rotate(q, k, pos.t().contiguous().t()), lambda: r.rotate(q.cpu(), k, pos),
           lambda: r.rotate(q, k, pos, q_out=k), lambda: r.append(q, k, v, pos, dst.int(), pool, pool),
           lambda: r.append(q, k, v, pos, dst[:3], pool, pool), lambda: r.append(q, k, v, pos, dst, pool.float(), pool),
           lambda: r.append(q, k, v, pos, dst, pool, pool.expand(2, -1, -1, -1)), lambda: r.append(q, k, v, pos, dst, pool, pool, q_rows=dst),
           lambda: r.append(q, k, v, pos, dst, pool, pool, q_out=q[:2]), lambda: r.append(q, k, v[:, :0], pos, dst, pool, pool),
           lambda: r.append(q, k, v, pos, dst, pool, pool, pos_offset=1 << 31),
           lambda: r.append(q, k, v, pos, dst, pool, pool, q_rows=dst, q_out=q),  # rows that others read first
           lambda: r.rotate(q, k, pos, q_out=q[:1].expand(4, -1, -1)),
           lambda: r.rotate(q, k, pos, q_out=q.as_strided(q.shape, (32, 64, 1)))]
    for f in bad:
        with pytest.raises(ValueError):
            f()
    plan = StepPlan(2, 4, 2)
    L, bt, free, nf = _i32([1, 2]), _i32(np.zeros((2, 4))), _i32([1, 2]), _i32([2])
    bad = [lambda: plan.build(L, L[:1], bt, free, nf, 16), lambda: plan.build(L.long(), L, bt, free, nf, 16),
           lambda: plan.build(L, L, bt, free, nf, 12), lambda: plan.build(L, L, bt[0], free, nf, 16),
           lambda: plan.build(L, L, bt.t(), free, nf, 16), lambda: plan.build(plan.seq_len, L, bt, free, nf, 16),
           lambda: plan.build(L, L, bt, free, plan.num_free, 16), lambda: plan.build(L.cpu(), L, bt, free, nf, 16)]
    for f in bad:
        with pytest.raises(ValueError):
            f()

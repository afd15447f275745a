"""GPU: attention with interval masks, distance bias and capped scores, bit-exact against the definition
on every kernel (multi-row, general, int8 prefill, both parts of tier 2, host exact tier), and the same
bits from all of them at larger sizes."""

import numpy as np
import pytest

from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from gen import bf16
import mod_oracle as mo

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


def _prob(rng, B, T, Hq, Hkv, d, S, kind="normal", page=0, layout="NHD", qscale=1.0, seq=None):
    q = bf16(rng, (B, T, Hq, d), kind, qscale)
    k, v = bf16(rng, (B, Hkv, S, d)), bf16(rng, (B, Hkv, S, d))
    seq = np.full(B, S) if seq is None else np.asarray(seq)
    kv = np.maximum(seq[:, None] - T + 1 + np.arange(T), 0)
    p = problem.contiguous(q, k, v, kv, seq_len=seq)
    return problem.to_paged(p, page, np.random.default_rng(7), layout) if page else p


def _run(p, ab, mods, out="bf16", kernel="auto", splits=0, force=False, tier2=True):
    import torch
    dp = hip.DeviceProblem(p, out, splits, "cuda:0", kernel, mods=mods)
    dp.out.fill_(-1)
    dp.flags.fill_(9)
    hip.launch_hip(dp, ab, tier2=tier2, force_tier2=force)
    torch.cuda.synchronize()
    res = dp.out.cpu().numpy()
    return res.view(np.uint32 if out == "fp32" else np.uint16), dp.flags.cpu().numpy(), dict(zip(hip.STATS, dp.stats.cpu().numpy().tolist()))


def _slopes(Hq, steep=1.0):
    return (steep * LOG2E * 2.0 ** (-8.0 * (np.arange(Hq) + 1) / Hq)).astype(np.float32)


# ---------------------------------------------------------------------------
# the modified logit
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("cap", [0.0, 43.28085, 0.5, 1e30])
def test_mod_logit(gpu, cap):
    import torch
    rng = np.random.default_rng(8)
    n = 6000
    t = (rng.standard_normal(n) * 2.0 ** rng.uniform(-30, 8, n)).astype(np.float32)
    t[:6] = [0.0, -0.0, 3.4e38, -3.4e38, 1e-45, 1.0]
    dist = rng.integers(-(1 << 20), 1 << 20, n).astype(np.int32)
    dist[:4] = [0, 2147483647, -2147483648, 1]
    m = (rng.standard_normal(n) * 2.0 ** rng.uniform(-20, 2, n)).astype(np.float32)
    m[::7] = 0.0
    tb, dd, md = (torch.from_numpy(x).cuda() for x in (t.view(np.int32), dist, m))
    bits, st = torch.empty(n, dtype=torch.int32, device="cuda"), torch.empty(n, dtype=torch.int32, device="cuda")
    assert hip.load().ea_hip_kat_mod_logit(n, tb.data_ptr(), dd.data_ptr(), md.data_ptr(), cap, bits.data_ptr(), st.data_ptr(),
                                           torch.cuda.current_stream().cuda_stream) == 0
    got = bits.cpu().numpy().view(np.float32)
    c = float(np.float32(cap))
    want = np.array([mo.bias32(mo.cap32(float(x), c), float(y), int(z)) for x, y, z in zip(t, m, dist)])
    assert (st.cpu().numpy() == 0).all()
    assert np.array_equal(got, want.astype(np.float32))


def test_mod_logit_not_finite(gpu):
    import torch
    t = torch.tensor([1.0, 1.0, 1.0], device="cuda").view(torch.int32)
    dist = torch.tensor([1 << 30, 1, 1], dtype=torch.int32, device="cuda")
    m = torch.tensor([3e38, float("nan"), float("inf")], device="cuda")
    bits, st = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(3, dtype=torch.int32, device="cuda")
    assert hip.load().ea_hip_kat_mod_logit(3, t.data_ptr(), dist.data_ptr(), m.data_ptr(), 0.0, bits.data_ptr(), st.data_ptr(), None) == 0
    torch.cuda.synchronize()
    assert st.cpu().tolist() == [2, 2, 2]


# ---------------------------------------------------------------------------
# every kernel against the definition
# ---------------------------------------------------------------------------

def _mods_of(name, rng, p):
    """A named set of modifications for problem p, as keyword arguments of both ScoreMods and the oracle."""
    g = p["geom"]
    B, T, Hq = g["num_seqs"], g["num_tokens"], g["num_q_heads"]
    kv = np.asarray(p["kv_len"]).reshape(B, T)
    if name == "none":
        return {}
    if name == "window":
        return dict(window=37)
    if name == "docs":
        b = np.minimum((rng.integers(0, 90, (B, T))).astype(np.int32), kv + 2)  # some see nothing
        b[0, 0] = -5
        return dict(kv_begin=b)
    if name == "alibi":
        return dict(slopes=_slopes(Hq))
    if name == "steep":
        return dict(slopes=_slopes(Hq, 16.0), q_pos=rng.integers(-50, 300, (B, T)).astype(np.int32))
    if name == "cap":
        return dict(softcap=4.0)
    return dict(softcap=20.0, slopes=-_slopes(Hq, 0.1), window=70, kv_begin=rng.integers(0, 60, (B, T)).astype(np.int32),
                q_pos=kv - 1 + rng.integers(0, 3, (B, T)).astype(np.int32))


def _oracle_args(m):
    m = dict(m)
    return dict(begin=m.get("kv_begin"), window=m.get("window", 0), slopes=m.get("slopes"), q_pos=m.get("q_pos"), cap=m.get("softcap", 0.0))


SHAPES = [
    # B, T, Hq, Hkv, d, S, page, kernels
    (2, 1, 4, 2, 128, 150, 16, ("auto", "general")),
    (1, 3, 6, 2, 128, 133, 0, ("auto", "general", "prefill")),
    (2, 8, 4, 2, 64, 100, 16, ("auto", "general")),
    (1, 5, 8, 1, 96, 70, 8, ("auto",)),          # pages under 16 keys: the general kernel
    (1, 34, 2, 2, 128, 129, 32, ("auto", "prefill")),
    (1, 33, 4, 2, 96, 100, 16, ("auto", "general")),  # padded to 128 dims in the prefill kernel
    (2, 2, 4, 2, 72, 90, 16, ("auto", "prefill")),
    (1, 40, 4, 2, 64, 150, 16, ("prefill",)),
    (1, 33, 2, 1, 8, 90, 0, ("auto", "prefill")),
]


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("name", ["none", "window", "docs", "alibi", "steep", "cap", "all"])
def test_definition(gpu, shape, name):
    B, T, Hq, Hkv, d, S, page, kernels = shape
    rng = np.random.default_rng(B * 100 + T + S)
    p = _prob(rng, B, T, Hq, Hkv, d, S, page=page, qscale=3.0, seq=[S - 9 * b for b in range(B)])
    m = _mods_of(name, rng, p)
    ab = default_alpha_bits(d)
    out = "fp32" if T == 3 else "bf16"
    rows = B * T * Hq
    some = sorted(set(rng.permutation(rows)[:24].tolist()) | {0, rows - 1})
    want = {r: mo.row(p, ab, r, out, **_oracle_args(m)) for r in some}
    for kernel in kernels:
        for force in (False, True):
            res, fl, st = _run(p, ab, hip.ScoreMods(**m), out, kernel, force=force)
            assert (fl == 0).all(), (kernel, force, st)
            flat = res.reshape(rows, d)
            for r in some:
                assert np.array_equal(flat[r], want[r]), (kernel, force, r)
    # the double-double pass on every row: tier 2 after a tier 1 that flags what it listed
    if name == "none":
        plain = _run_plain(p, ab, out)
        assert np.array_equal(res, plain)


def _run_plain(p, ab, out):
    return hip.attention_problem(p, None, out, alpha_bits=ab)[0]


@pytest.mark.parametrize("kernel", ["auto", "prefill", "general"])
def test_head_sizes_and_strides(gpu, kernel):
    """K and V of different head sizes, rows that start on 4-byte boundaries with other data between them, a
    head size the prefill kernel pads: what lies past a row's end stays out."""
    rng = np.random.default_rng(77)
    B, T, Hq, Hkv, d, dv, S = 1, 40, 4, 2, 80, 104, 150
    q, k, v = bf16(rng, (B, T, Hq, d)), bf16(rng, (B, Hkv, S, d)), bf16(rng, (B, Hkv, S, dv))
    kv = S - T + 1 + np.arange(T)[None]
    p = problem.contiguous(q, k, v, kv)
    want, fl, _ = _run(p, default_alpha_bits(128), hip.ScoreMods(window=60, softcap=10.0), kernel="general")
    g = p["geom"]
    for x, w in (("k", d), ("v", dv)):
        wide = np.full((B, S, Hkv, w + 10), 0x7FC0, np.uint16)
        wide[..., :w] = p[x].transpose(0, 2, 1, 3)
        p[x] = wide
        g[x + "_page_stride"], g[x + "_slot_stride"], g[x + "_head_stride"] = S * Hkv * (w + 10), Hkv * (w + 10), w + 10
    got, f2, st = _run(p, default_alpha_bits(128), hip.ScoreMods(window=60, softcap=10.0), kernel=kernel)
    assert (fl == 0).all() and (f2 == 0).all()
    assert np.array_equal(got, want)
    assert st["prefill_kernel_rows"] == (T * Hq if kernel == "prefill" else 0)
    some = mo.row(p, default_alpha_bits(128), 5, window=60, cap=10.0)
    assert np.array_equal(got.reshape(-1, dv)[5], some)


@pytest.mark.parametrize("name", ["plain", "none", "all"])
@pytest.mark.parametrize("d", [128, 104])
def test_elements_rounded_at_slicing(gpu, d, name):
    """Rows of q with elements far below their largest: the prefill kernel takes their next 8 bits in, and
    decides their scores as it does the others'."""
    rng = np.random.default_rng(d)
    B, T, Hq, Hkv, S = 1, 64, 4, 2, 700
    p = _prob(rng, B, T, Hq, Hkv, d, S)
    q = (p["q"].astype(np.uint32) << 16).view(np.float32).reshape(T * Hq, d).copy()
    for r, (n, k) in enumerate([(1, 22), (1, 24), (1, 27), (1, 30), (1, 33), (3, 24), (3, 30), (40, 23), (d - 1, 25), (d - 1, 60)]):
        q[20 * r, rng.permutation(d)[:n]] *= 2.0 ** -k
    for r, x in ((210, 0.5), (211, -0.5), (212, 1.5), (213, -1.5), (214, 0.25)):
        q[r, np.abs(q[r]) > 1.9] = 1.0
        q[r, 0] = 1.0
        q[r, d - 1] = x * 2.0 ** -29  # of a largest element of 1 to 2: half steps and their neighbours
    bits = q.view(np.uint32) >> 16
    assert (bits << 16 == q.view(np.uint32)).all()
    p["q"] = bits.astype(np.uint16).reshape(p["q"].shape)
    ab = default_alpha_bits(d)
    m = None if name == "plain" else hip.ScoreMods(**_mods_of(name, rng, p))
    got, fl, st = _run(p, ab, m, "fp32", "prefill")
    want, f2, _ = _run(p, ab, m, "fp32", "general")
    assert (fl == 0).all() and (f2 == 0).all()
    assert np.array_equal(got, want)
    if st["prefill_kernel_rows"] == 0:  # heads below 128 dims without modifications are another kernel's
        assert name == "plain" and d != 128
        return
    # A score known to within e is undecided with probability 2 e / step, step = ulp of its fp32 value. e: n
    # rounded elements of q within 2^-8 units each of K's largest, n of k within half a unit of q's largest.
    k = (p["k"].astype(np.uint32) << 16).view(np.float32).reshape(Hkv, S, d).astype(np.float64)
    q = q.reshape(T, Hkv, Hq // Hkv, d).astype(np.float64)

    def unit(x):
        u = 2.0 ** (np.floor(np.log2(np.abs(x).max(-1))) - 29)
        return u, (np.rint(x / u[..., None]) != x / u[..., None]).sum(-1)

    (uq, nq), (uk, nk) = unit(q), unit(k)
    alpha = float(np.uint32(ab).view(np.float32))
    expect = 0.0
    for h in range(Hkv):
        t = alpha * (q[:, h] @ k[h].T)
        e = alpha * ((nq * uq * 1.01 * 2.0 ** -8)[:, h, :, None] * np.abs(k[h]).max(-1) +
                     np.abs(q[:, h]).max(-1)[..., None] * (0.5 * nk * uk)[h])
        expect += np.minimum(1.0, 2 * e / np.spacing(np.abs(t).astype(np.float32))).sum()
    assert st["prefill_kernel_rows"] == T * Hq and st["slow_path_scores"] <= expect + 6 * expect ** 0.5 + 10, expect


@pytest.mark.parametrize("T", [1, 3, 34])
@pytest.mark.parametrize("slope", [0.9, 7.0, 16.0, 40.0])
def test_channels_of_far_keys_alone(gpu, T, slope):
    """Channels whose values are zero but for keys of weights down to 2^-9000 of the row's largest."""
    rng = np.random.default_rng(T)
    S, Hq, d = 230, 2, 128
    p = _prob(rng, 1, T, Hq, 1, d, S)
    pos = (S - T + np.arange(T)).astype(np.int32)
    sl = np.full(Hq, slope, np.float32)
    ab = default_alpha_bits(d)
    for far in (0x3F80, 0xBF80):
        v = np.zeros((1, 1, S, d), np.uint16)
        v[:, :, :100], v[:, :, 100:150, ::2], v[:, :, 150:, 5] = far, far, 0x4000
        p["v"] = v
        want = {r: mo.row(p, ab, r, slopes=sl, q_pos=pos[None]) for r in (0, T * Hq - 1)}
        for kernel in ("auto", "general") + (("prefill",) if T == 34 else ()):
            for force in (False, True):
                res, fl, _ = _run(p, ab, hip.ScoreMods(slopes=sl, q_pos=pos), kernel=kernel, force=force)
                assert (fl == 0).all()
                for r, w in want.items():
                    assert np.array_equal(res.reshape(-1, d)[r], w), (kernel, force, far)


@pytest.mark.parametrize("name", ["docs", "steep", "cap", "all"])
def test_host_exact_tier(gpu, name):
    """Rows left at flag 1 finished by the host tier: the same bits."""
    import torch
    rng = np.random.default_rng(31)
    p = _prob(rng, 2, 2, 4, 2, 64, 90, page=16, qscale=2.0)
    mods = hip.ScoreMods(**_mods_of(name, rng, p))
    ab = default_alpha_bits(64)
    res, fl, _ = _run(p, ab, mods)
    dp = hip.DeviceProblem(p, "bf16", mods=mods)
    dp.out.fill_(0)
    dp.flags.fill_(1)
    hip.exact_rows(dp, ab)
    torch.cuda.synchronize()
    assert (dp.flags.cpu().numpy() == 0).all() and (fl == 0).all()
    assert np.array_equal(dp.out.cpu().numpy().view(np.uint16), res)


@pytest.mark.parametrize("kernel", ["auto", "general"])
@pytest.mark.parametrize("d", [128, 64])
def test_tree_and_interval(gpu, kernel, d):
    """Tree keys join the interval, wherever they lie: past it, inside it, before its first key."""
    rng = np.random.default_rng(5)
    B, T, Hq, Hkv, S = 2, 6, 4, 2, 150
    p = _prob(rng, B, T, Hq, Hkv, d, S, page=16)
    kv = np.array([[100, 80, 0, 130, 20, 150]] * B, np.int32)
    begin = np.array([[60, 90, 0, 100, 5, 10], [0, 0, 0, 0, 0, 149]], np.int32)
    p["kv_len"] = kv.reshape(-1)
    p["tree_mask"] = rng.integers(1, 1 << 62, B * T, dtype=np.int64).astype(np.uint64)
    p["tree_mask"][4] = 0
    p["tree_base"] = np.array([70, 95], np.int32)
    m = dict(kv_begin=begin, slopes=_slopes(Hq), q_pos=kv + 3)
    ab = default_alpha_bits(d)
    for force in (False, True):
        res, fl, _ = _run(p, ab, hip.ScoreMods(**m), kernel=kernel, force=force)
        assert (fl == 0).all()
        flat = res.reshape(-1, d)
        for r in range(0, B * T * Hq, 3):
            assert np.array_equal(flat[r], mo.row(p, ab, r, **_oracle_args(m))), r


@pytest.mark.parametrize("T, S", [(1, 200), (40, 200)])
def test_rows_that_see_nothing(gpu, T, S):
    rng = np.random.default_rng(6)
    p = _prob(rng, 2, T, 4, 2, 128, S, page=16)
    kv = np.asarray(p["kv_len"]).reshape(2, T)
    for kernel in ("auto", "general", "prefill"):
        for b in (kv, kv + 1000, np.full_like(kv, 2147483647)):
            res, fl, _ = _run(p, default_alpha_bits(128), hip.ScoreMods(kv_begin=b, slopes=_slopes(4)), kernel=kernel)
            assert (res == 0).all() and (fl == 0).all()


def test_what_is_masked_is_not_read(gpu):
    """NaN and infinities in keys outside every row's interval, in its first and last tile too, and pages
    before the first visible key's tile that hold nothing but NaN: no flag, the same bits."""
    rng = np.random.default_rng(12)
    ab = default_alpha_bits(128)
    for T, kernel in ((1, "auto"), (2, "general"), (40, "auto"), (40, "prefill")):
        p = _prob(rng, 1, T, 4, 2, 128, 500, page=16)
        begin = np.maximum(200 + np.arange(T)[None], 0).astype(np.int32)
        mods = hip.ScoreMods(kv_begin=begin)
        p["kv_len"] = np.minimum(np.asarray(p["kv_len"]), 420 + np.arange(T)).astype(np.int32)
        want, fl, _ = _run(p, ab, mods, kernel=kernel)
        assert (fl == 0).all()
        bt = np.asarray(p["block_table"]).reshape(-1)
        for n in list(range(0, 200)) + list(range(420 + T, 500)):
            pg, sl = bt[n // 16], n % 16
            p["k"].reshape(-1, 16, 2, 128)[pg, sl] = 0x7FC0
            p["v"].reshape(-1, 16, 2, 128)[pg, sl] = 0x7F80 if n % 2 else 0xFFC0
        got, fl, _ = _run(p, ab, mods, kernel=kernel)
        assert (fl == 0).all(), (T, kernel)
        assert np.array_equal(got, want)


def test_domain_errors(gpu):
    """A bias that is not finite, or a score past fp32 however capped, flags its rows and no others."""
    rng = np.random.default_rng(13)
    for T, kernel in ((1, "auto"), (1, "general"), (34, "prefill")):
        p = _prob(rng, 1, T, 4, 2, 128, 100, page=16)
        ab = default_alpha_bits(128)
        s = _slopes(4)
        s[1], s[2] = np.nan, np.inf
        res, fl, _ = _run(p, ab, hip.ScoreMods(slopes=s, q_pos=np.full((1, T), 200)), kernel=kernel)
        assert fl.reshape(T, 4).tolist() == [[0, 2, 2, 0]] * T
        assert (res.reshape(T, 4, -1)[:, 1:3] == 0).all()
        p["q"][0, 0, 0, :] = 0x7F00  # 1.7e38: the scores overflow fp32
        res, fl, _ = _run(p, ab, hip.ScoreMods(softcap=20.0), kernel=kernel)
        assert fl.reshape(T, 4)[0, 0] == 2 and (fl.reshape(-1)[1:] == 0).all()


def test_zero_scores_under_a_bias(gpu):
    """q = 0, k = 0 and disjoint supports: logits of 0 whose fast path knows only that they are tiny."""
    rng = np.random.default_rng(14)
    for d, T, kernel in ((128, 1, "auto"), (64, 3, "auto"), (128, 2, "general"), (128, 34, "prefill")):
        p = _prob(rng, 1, T, 2, 1, d, 90, page=16)
        q, k = p["q"], p["k"]
        q[:, 0, 0] = 0
        q[..., d // 2:] = 0
        k.reshape(-1, d)[::2, :d // 2] = 0  # every other slot: orthogonal to every q
        ab = default_alpha_bits(d)
        for m in (dict(slopes=_slopes(2)), dict(slopes=_slopes(2), softcap=3.0), dict(softcap=3.0), dict(slopes=np.float32([0.0, 1e-9]))):
            res, fl, st = _run(p, ab, hip.ScoreMods(**m), kernel=kernel)
            assert (fl == 0).all()
            for r in range(0, T * 2, max(1, T // 4)):
                assert np.array_equal(res.reshape(-1, d)[r], mo.row(p, ab, r, **_oracle_args(m))), (d, T, kernel, r)


# ---------------------------------------------------------------------------
# larger sizes: the same bits from every kernel, split count and layout
# ---------------------------------------------------------------------------

@pytest.mark.parametrize("case", [
    dict(B=3, T=1, Hq=16, Hkv=4, d=128, S=9000, m=dict(window=1500)),
    dict(B=2, T=4, Hq=8, Hkv=4, d=128, S=5000, m=dict(softcap=30.0)),
    dict(B=1, T=1, Hq=8, Hkv=8, d=64, S=20000, m="steep"),
    dict(B=1, T=200, Hq=4, Hkv=2, d=128, S=700, m="docs"),
    dict(B=1, T=300, Hq=4, Hkv=4, d=128, S=1300, m="steepwin"),
    dict(B=2, T=150, Hq=4, Hkv=1, d=80, S=400, m="all"),
    dict(B=40, T=1, Hq=16, Hkv=8, d=128, S=3000, m="ragged"),
])
@pytest.mark.parametrize("out", ["bf16", "fp32"])
def test_same_bits_everywhere(gpu, case, out):
    rng = np.random.default_rng(case["S"])
    B, T, Hq, Hkv, d, S = (case[x] for x in ("B", "T", "Hq", "Hkv", "d", "S"))
    seq = rng.integers(S // 3, S + 1, B)
    p = _prob(rng, B, T, Hq, Hkv, d, S, page=16, qscale=2.0, seq=seq)
    kv = np.asarray(p["kv_len"]).reshape(B, T)
    m = {"steep": dict(slopes=_slopes(Hq, 1.0)), "steepwin": dict(slopes=_slopes(Hq, 4.0), window=333, q_pos=kv - 1),
         "docs": dict(kv_begin=np.minimum(kv - 1, (np.arange(T) // 23 * 23)[None] + 0 * kv)),
         "all": dict(slopes=_slopes(Hq), softcap=25.0, window=100),
         "ragged": dict(kv_begin=rng.integers(0, 2900, (B, T)), slopes=_slopes(Hq))}.get(str(case["m"]), case["m"])
    ab = default_alpha_bits(d)
    res, fl, st = _run(p, ab, hip.ScoreMods(**m), out)
    assert (fl == 0).all()
    if out == "bf16":
        # far keys under a steep bias are not what sends rows to tier 2 (in fp32 the int8 kernel's bounds
        # leave most rows of large scores to it, with and without modifications)
        assert st["tier1_flagged"] <= 0.01 * st["rows"] + 1, st
    kinds = [dict(kernel="general"), dict(splits=1), dict(splits=7)]
    if d == 128:
        kinds.append(dict(kernel="prefill"))
    if B * T * Hq <= 512:
        kinds.append(dict(force=True))
    for kw in kinds:
        r2, f2, s2 = _run(p, ab, hip.ScoreMods(**m), out, **kw)
        assert (f2 == 0).all() and np.array_equal(r2, res), (kw, s2)
    for span in (1, 100, S):  # hints below and above the real span
        r2, f2, _ = _run(p, ab, hip.ScoreMods(**m, max_span=span), out)
        assert (f2 == 0).all() and np.array_equal(r2, res), span
    p2 = problem.to_paged(problem.contiguous(p["q"], *(_unpage(p, x) for x in "kv"), kv, seq_len=seq), 64, np.random.default_rng(1), "HND")
    r2, f2, _ = _run(p2, ab, hip.ScoreMods(**m), out)
    assert (f2 == 0).all() and np.array_equal(r2, res)
    # some rows against the definition
    for r in rng.permutation(B * T * Hq)[:2]:
        if S <= 1300:
            assert np.array_equal(res.reshape(-1, d)[r], mo.row(p, ab, int(r), out, **_oracle_args(m)))


def _unpage(p, x):
    """The contiguous (B, Hkv, S, d) form of a paged NHD cache."""
    g = p["geom"]
    bt = np.asarray(p["block_table"])
    pool = p[x].reshape(-1, g["page_size"], g["num_kv_heads"], g["head_dim"])
    rows = pool[np.maximum(bt, 0)].reshape(bt.shape[0], -1, g["num_kv_heads"], g["head_dim"])
    return np.ascontiguousarray(rows.transpose(0, 2, 1, 3))


def test_against_the_formula(gpu):
    """A window of a long context against the formula in 64 bits. t2 carries three roundings of at most 2^-24 of
    numbers below 2^6 here and each weight one more of 2^-24: a relative 2^-18 ln 2 3 + 2^-24 < 2^-16.9 of every weight, so
    the output moves by at most 2^-15.9 max|v|, and rounds by half a step."""
    import torch
    rng = np.random.default_rng(21)
    B, Hq, Hkv, d, S, W = 2, 8, 4, 128, 40000, 3000
    p = _prob(rng, B, 1, Hq, Hkv, d, S, page=64, seq=[S, S - 777])
    sl = _slopes(Hq, 0.05)
    cap = 20.0
    ab = default_alpha_bits(d)
    res, fl, _ = _run(p, ab, hip.ScoreMods(window=W, slopes=sl, softcap=cap))
    assert (fl == 0).all()
    alpha = float(np.uint32(ab).view(np.float32))
    f = lambda x: torch.from_numpy((x.astype(np.uint32) << 16).view(np.float32)).double()
    K, V, q = f(_unpage(p, "k")), f(_unpage(p, "v")), f(p["q"])
    for b in range(B):
        L = int(np.asarray(p["kv_len"])[b])
        n = torch.arange(L - W, L)
        for h in range(Hq):
            t = alpha * (K[b, h // 2, L - W:L] @ q[b, 0, h])
            t = cap * torch.tanh(t / cap) - float(sl[h]) * (L - 1 - n)
            o = torch.softmax(t * np.log(2.0), 0) @ V[b, h // 2, L - W:L]
            got = f(res[b, 0, h][None])[0]
            assert float(t.abs().max()) < 2 ** 8
            tol = o.abs() * 2.0 ** -8 + 2.0 ** -13.9 * float(V[b].abs().max())
            assert bool(((got - o).abs() <= tol).all())


def test_graph_replays(gpu):
    """A captured step with modifications, replayed with other lengths written between, equals eager steps."""
    import torch
    from exactattention_amd.graph import HipGraph
    rng = np.random.default_rng(22)
    p = _prob(rng, 4, 1, 16, 8, 128, 2000, page=16)
    ab = default_alpha_bits(128)
    mods = hip.ScoreMods(window=300, slopes=_slopes(16), softcap=30.0)
    dp = hip.DeviceProblem(p, "bf16", mods=mods)
    hip.launch_hip(dp, ab)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    g = HipGraph()
    with torch.cuda.stream(st):
        g.capture(st, lambda: hip.launch_hip(dp, ab))
    for i in range(4):
        kv = rng.integers(1, 2001, 4).astype(np.int32)
        dp.t["kv_len"].copy_(torch.from_numpy(kv))
        dp.out.fill_(0)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            g.replay(st)
        torch.cuda.synchronize()
        got = dp.out.cpu().numpy().view(np.uint16)
        want, fl, _ = _run(dict(p, kv_len=kv), ab, mods)
        assert (fl == 0).all() and np.array_equal(got, want), i
    g.close()


@pytest.mark.parametrize("name", ["docs", "alibi", "cap"])
def test_more_items_than_blocks(gpu, name):
    """Prefill steps whose row blocks outnumber the CUs: blocks take several, and the fp64 kernel's bits come
    out, also from two steps in flight at once and from a captured step replayed after others."""
    import torch
    from exactattention_amd.graph import HipGraph
    rng = np.random.default_rng(31)
    p = _prob(rng, 1, 1300, 8, 8, 128, 1300, qscale=2.0)  # 8 x 41 row blocks
    ab = default_alpha_bits(128)
    m = _mods_of(name, rng, p)
    want, fl, st = _run(p, ab, hip.ScoreMods(**m), kernel="decode")
    assert (fl == 0).all() and st["mrow_kernel_rows"] == 8 * 1300
    dps = [hip.DeviceProblem(p, "bf16", 0, "cuda:0", "prefill", mods=hip.ScoreMods(**m)) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in dps]
    torch.cuda.synchronize()
    for _ in range(2):
        for dp, s in zip(dps, streams):
            with torch.cuda.stream(s):
                dp.out.fill_(-1)
                hip.launch_hip(dp, ab)
    torch.cuda.synchronize()
    for dp in dps:
        assert np.array_equal(dp.out.cpu().numpy().view(np.uint16), want) and not bool(dp.flags.any())
        assert dp.stats.tolist()[10] == 2 * 8 * 1300
    dp, g = dps[0], HipGraph()
    with torch.cuda.stream(streams[0]):
        g.capture(streams[0], lambda: hip.launch_hip(dp, ab))
    for _ in range(3):
        dp.out.fill_(-1)
        dp.flags.fill_(9)
        hip.launch_hip(dps[1], ab)
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            g.replay(streams[0])
        torch.cuda.synchronize()
        assert np.array_equal(dp.out.cpu().numpy().view(np.uint16), want) and not bool(dp.flags.any())
    g.close()

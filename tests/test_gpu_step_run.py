"""GPU: the step's operators together, as a serving loop uses them: plan, rotary positions with the cache
append, modified attention. The reference turns q and k with Rotary.rotate (tested by itself against
the formula), keeps every sequence's keys in plain arrays and attends each step as a problem of its
own; the loop's outputs must equal it bit for bit."""

import numpy as np
import pytest

from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from gen import bf16

pytestmark = pytest.mark.gpu
LOG2E = 1.4426950408889634


def _dev(x):
    import torch
    return torch.from_numpy(np.ascontiguousarray(x).view(np.int16)).cuda()


def _bits(t):
    import torch
    return t.contiguous().view(torch.int16).cpu().numpy().view(np.uint16)


class _Reference:
    """Sequences of turned keys in plain arrays, attended one step at a time."""

    def __init__(self, rotary, Hq, Hkv, d, mods):
        self.r, self.Hq, self.Hkv, self.d, self.mods = rotary, Hq, Hkv, d, mods
        self.k, self.v = {}, {}

    def turn(self, q, k, pos):
        import torch
        p = torch.from_numpy(np.ascontiguousarray(pos, dtype=np.int32)).cuda()
        if self.r is None:
            return q, k
        q, k = self.r.rotate(_dev(q), _dev(k), p)
        return _bits(q), _bits(k)

    def step(self, seqs, ql, q, k, v, pos=None):
        """Outputs and flags of the new tokens, in order."""
        out, at = [], 0
        for s, n in zip(seqs, ql):
            K, V = self.k.get(s, np.zeros((0, self.Hkv, self.d), np.uint16)), self.v.get(s, np.zeros((0, self.Hkv, self.d), np.uint16))
            L = len(K)
            p = np.arange(L, L + n) if pos is None else np.asarray(pos)[..., at:at + n]
            qn, kn = self.turn(q[at:at + n], k[at:at + n], p)
            self.k[s], self.v[s] = np.concatenate([K, kn]), np.concatenate([V, v[at:at + n]])
            out.append(self.attend(s, qn, (L + 1 + np.arange(n))[None]))
            at += n
        return np.concatenate(out)

    def attend(self, s, q, kv_len, mods=None, **tree):
        p = problem.contiguous(q[None], self.k[s].transpose(1, 0, 2)[None], self.v[s].transpose(1, 0, 2)[None], kv_len, **tree)
        m = self.mods if mods is None else mods
        return hip.attention_problem(p, None, alpha_bits=default_alpha_bits(self.d), mods=m)[0][0]


def _mods(name, Hq):
    sl = (LOG2E * 2.0 ** (-8.0 * (np.arange(Hq) + 1) / Hq)).astype(np.float32)
    return {"none": None, "window": hip.ScoreMods(window=50), "cap": hip.ScoreMods(softcap=8.0),
            "all": hip.ScoreMods(window=90, softcap=20.0, slopes=sl)}[name]


def _backend(name, rotary, d=128, Hq=4, Hkv=2, page=16, digits=True, max_len=1500):
    from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache
    cache = PagedKVCache(400, page, Hkv, d, 8, max_len, digits=digits)
    return cache, ExactAttentionBackend(cache, Hq, alpha_bits=default_alpha_bits(d), mods=_mods(name, Hq), rotary=rotary)


@pytest.mark.parametrize("name", ["none", "window", "cap", "all"])
@pytest.mark.parametrize("d, page, rot", [(128, 16, 128), (64, 8, 32), (128, 64, None)])
def test_forward(gpu, name, d, page, rot):
    """Mixed batches through forward: prompts, decode steps, chunks, a dropped sequence's slot used again."""
    from exactattention_amd.serving import Rotary
    rng = np.random.default_rng(d + page)
    r = None if rot is None else Rotary(d, rot_dim=rot, adjacent=page == 8)
    cache, be = _backend(name, r, d, page=page)
    ref = _Reference(r, 4, 2, d, be.mods)
    s = [cache.add_sequence() for _ in range(4)]
    steps = [([0, 1], [70, 33]), ([1, 0], [1, 1]), ([2, 0, 1], [40, 1, 5]), ([3, 2, 1, 0], [9, 1, 1, 1]), ([0, 1, 2, 3], [1, 1, 1, 1]),
             ([2], [100]), ([1, 2], [3, 3])]
    for i, (seqs, ql) in enumerate(steps):
        n = sum(ql)
        q, k, v = bf16(rng, (n, 4, d), "normal", 2.0), bf16(rng, (n, 2, d)), bf16(rng, (n, 2, d))
        out, flags = be.forward(_dev(q), _dev(k), _dev(v), [s[x] for x in seqs], ql)
        be.check_flags(flags)
        want = ref.step([s[x] for x in seqs], ql, q, k, v)
        assert np.array_equal(_bits(out), want), i
        if i == 4:
            cache.drop_sequence(s[3])
            ref.k.pop(s[3], None)
            ref.v.pop(s[3], None)
            s[3] = cache.add_sequence()
    for x in s[:3]:
        idx = np.concatenate([np.arange(p * page, p * page + page) for p in cache.pages[x]])[:cache.length[x]]
        assert np.array_equal(_bits(cache.k).reshape(-1, 2, d)[idx], ref.k[x])
        assert np.array_equal(cache.block_table.cpu().numpy()[x, :len(cache.pages[x])], cache.pages[x])


@pytest.mark.parametrize("turned", [False, True])
@pytest.mark.parametrize("B, slots", [(8200, 8200), (3, 65540)])
def test_batches_past_a_plan(gpu, B, slots, turned):
    """More sequences, or table rows, than a StepPlan takes: the step's vectors are made on the host, and the
    batch's parts, each small enough for a plan, give the same."""
    from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache, Rotary
    rng = np.random.default_rng(B)
    r = Rotary(16) if turned else None
    got = []
    ql = [3] + [1, 2] * (B // 2)
    ql = ql[:B]
    steps = [[bf16(rng, (sum(ql), h, 16)) for h in (2, 1, 1)] for _ in range(2)]
    for whole in (True, False):
        cache = PagedKVCache(2 * B, 4, 1, 16, slots if whole else B, 8, digits=False)
        be = ExactAttentionBackend(cache, 2, alpha_bits=default_alpha_bits(16), rotary=r)
        s = [cache.add_sequence() for _ in range(B)] if whole is False or slots == B else list(range(slots - B, slots))
        if whole and slots != B:
            for x in s:
                cache.live[x] = True
        for q, k, v in steps:  # up to 6 keys, two pages
            outs, cut, t0 = [], (B if whole else B // 2 + 1), 0
            for i in range(0, B, cut):
                n = sum(ql[i:i + cut])
                o, f = be.forward(*(_dev(x[t0:t0 + n]) for x in (q, k, v)), s[i:i + cut], ql[i:i + cut])
                be.check_flags(f)
                outs.append(_bits(o))
                t0 += n
            got.append(np.concatenate(outs))
    assert np.array_equal(got[0], got[2]) and np.array_equal(got[1], got[3])


def test_forward_positions(gpu):
    """Three position axes, fp32 projections as parts of one row, and given positions for one axis."""
    import torch
    from exactattention_amd.serving import Rotary
    rng = np.random.default_rng(3)
    r = Rotary(128, sections=[16, 24, 24], interleaved=True)
    cache, be = _backend("window", r)
    ref = _Reference(r, 4, 2, 128, be.mods)
    s = [cache.add_sequence() for _ in range(2)]
    for ql in ([30, 7], [1, 1]):
        n = sum(ql)
        qkv = torch.from_numpy(rng.standard_normal((n, 8 * 128)).astype(np.float32)).cuda()
        q, k, v = (x.view(n, -1, 128) for x in qkv.split([512, 256, 256], 1))
        pos = torch.from_numpy(rng.integers(0, 5000, (3, n)).astype(np.int32)).cuda()
        out, flags = be.forward(q, k, v, s, ql, positions=pos)
        be.check_flags(flags)
        # the reference turns in fp32 inputs too: rounded once, as append rounds
        pool = torch.zeros(-(-n // 16), 16, 2, 128, dtype=torch.bfloat16, device="cuda")
        pv = torch.zeros_like(pool)
        qn = r.append(q, k, v, pos, torch.arange(n, device="cuda"), pool, pv)
        kn, vn = _bits(pool).reshape(-1, 2, 128)[:n], _bits(pv).reshape(-1, 2, 128)[:n]
        ref.r = None
        assert np.array_equal(_bits(out), ref.step(s, ql, _bits(qn), kn, vn))
        ref.r = r
    with pytest.raises(ValueError):
        be.forward(q, k, v, s, ql)  # three axes have no default
    before = [list(x) for x in cache.pages], list(cache.length), list(cache.free)
    for bad in (dict(positions=pos[:2]), dict(positions=pos[:, :1]), dict(positions=pos.long())):
        with pytest.raises(ValueError):
            be.forward(q, k, v, s, ql, **bad)
    with pytest.raises(ValueError):
        be.forward(q, k[:, :1], v, s, ql, positions=pos)
    with pytest.raises(ValueError):
        be.forward(q, k.bfloat16(), v, s, ql, positions=pos)
    assert before == ([list(x) for x in cache.pages], list(cache.length), list(cache.free))


@pytest.mark.parametrize("name", ["none", "window", "all"])
def test_decode_graph(gpu, name):
    """Replayed decode steps, each against the reference, the eager forward between them on other slots."""
    from exactattention_amd.serving import DecodeGraph, Rotary
    rng = np.random.default_rng(17)
    r = Rotary(128)
    cache, be = _backend(name, r)
    ref = _Reference(r, 4, 2, 128, be.mods)
    s = [cache.add_sequence() for _ in range(3)]
    ql = [60, 15, 100]
    q, k, v = (bf16(rng, (175, h, 128)) for h in (4, 2, 2))
    out, fl = be.forward(_dev(q), _dev(k), _dev(v), s, ql)
    be.check_flags(fl)
    assert np.array_equal(_bits(out), ref.step(s, ql, q, k, v))
    g = DecodeGraph(be, s[:2], max_len=200)
    for i in range(5):
        q, k, v = (bf16(rng, (2, h, 128)) for h in (4, 2, 2))
        g.q.copy_(_dev(q)[:, None])
        g.k.copy_(_dev(k))
        g.v.copy_(_dev(v))
        out, fl = g.step()
        g.check_flags(fl)
        assert np.array_equal(_bits(out), ref.step(s[:2], [1, 1], q, k, v)), i
        q, k, v = (bf16(rng, (2, h, 128)) for h in (4, 2, 2))
        out, fl = be.forward(_dev(q), _dev(k), _dev(v), s[2:], [2])
        be.check_flags(fl)
        assert np.array_equal(_bits(out), ref.step(s[2:], [2], q, k, v)), i
    g.close()


@pytest.mark.parametrize("window", [0, 3, 40])
@pytest.mark.parametrize("turned", [False, True])
def test_verify_tree(gpu, window, turned):
    """Draft trees under a window: a node sees its last `window` keys, path and prefix together. Its output is that
    of the path appended as a chain."""
    from exactattention_amd.serving import Rotary
    rng = np.random.default_rng(window)
    r = Rotary(128) if turned else None
    cache, be = _backend("none", r)
    be2 = _backend("none", r)[1]
    mods = hip.ScoreMods(window=window, softcap=9.0)
    be.mods = mods
    be._mods_args, be._mods_keep = mods.bind(dict(num_seqs=0, num_tokens=0, num_q_heads=4), cache.dev)
    ref = _Reference(r, 4, 2, 128, mods)
    s = cache.add_sequence()
    q, k, v = (bf16(rng, (50, h, 128)) for h in (4, 2, 2))
    be.prefill(s, q, k, v)
    ref.step([s], [50], q, k, v)
    K0, V0 = ref.k[s], ref.v[s]
    parents = [-1, 0, 0, 1, 3, -1, 5, 4]
    q, k, v = (bf16(rng, (8, h, 128)) for h in (4, 2, 2))
    out, fl = be.verify_tree(s, q, k, v, parents)
    assert (fl == 0).all()
    for i in range(8):
        path = [i]
        while parents[path[0]] >= 0:
            path.insert(0, parents[path[0]])
        ref.k[s], ref.v[s] = K0, V0
        want = ref.step([s], [len(path)], q[path], k[path], v[path])
        assert np.array_equal(out[i], want[-1]), i
    # the accepted path stays, and the next step goes on from it
    be.accept(s, 50, [0, 1, 3], k, v)
    ref.k[s], ref.v[s] = K0, V0
    ref.step([s], [3], q[[0, 1, 3]], k[[0, 1, 3]], v[[0, 1, 3]])
    q, k, v = (bf16(rng, (1, h, 128)) for h in (4, 2, 2))
    out, _ = be.decode([s], q, k, v)
    assert np.array_equal(out, ref.step([s], [1], q, k, v))
    be.mods = hip.ScoreMods(slopes=np.ones(4, np.float32))
    with pytest.raises(ValueError):
        be.verify_tree(s, q, k, v, [-1])


def test_backend_refuses(gpu):
    from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache, Rotary
    cache = PagedKVCache(4, 16, 2, 64, 2, 64)
    for kw in (dict(mods=hip.ScoreMods(kv_begin=np.zeros(1))), dict(mods=hip.ScoreMods(q_pos=np.zeros(1))),
               dict(mods=hip.ScoreMods(slopes=np.ones(3, np.float32))), dict(rotary=Rotary(128))):
        with pytest.raises(ValueError):
            ExactAttentionBackend(cache, 4, alpha_bits=default_alpha_bits(64), **kw)
    be = ExactAttentionBackend(cache, 4, alpha_bits=default_alpha_bits(64))
    import torch
    z = torch.zeros(1, 2, 64, dtype=torch.int16, device="cuda")
    with pytest.raises(ValueError):
        be.forward(torch.zeros(1, 4, 64, dtype=torch.int16, device="cuda"), z, z, [cache.add_sequence()], [1],
                   positions=torch.zeros(1, dtype=torch.int32, device="cuda"))


def test_steps_without_the_host(gpu):
    """A loop whose lengths, block table and free pages stay on the device: plan, rotary append and attention
    of a step in one captured graph, replayed; the state goes round by device copies in the graph."""
    import torch
    from exactattention_amd.graph import HipGraph
    from exactattention_amd.step import Rotary, StepPlan
    rng = np.random.default_rng(9)
    B, Hq, Hkv, d, P, W, T = 3, 4, 2, 128, 16, 20, 2
    dev = "cuda"
    r = Rotary(d)
    mods = hip.ScoreMods(window=64)
    kp, vp = (torch.zeros(60, P, Hkv, d, dtype=torch.int16, device=dev) for _ in range(2))
    perm = rng.permutation(60).astype(np.int32)
    i32 = lambda x: torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).to(dev)
    L, cnt, nf, free = i32([0, 0, 0]), i32([2, 1, 2]), i32([60]), i32(perm)
    bt = torch.zeros(B, W, dtype=torch.int32, device=dev)
    plan = StepPlan(B, B * T, T)
    q = torch.zeros(B * T, Hq, d, dtype=torch.int16, device=dev)
    k, v = (torch.zeros(B * T, Hkv, d, dtype=torch.int16, device=dev) for _ in range(2))
    qd = torch.zeros(B * T, Hq, d, dtype=torch.int16, device=dev)
    geom = dict(num_seqs=B, num_tokens=T, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=d, head_dim_v=d, q_seq_stride=T * Hq * d,
                q_tok_stride=Hq * d, q_head_stride=d, o_seq_stride=T * Hq * d, o_tok_stride=Hq * d, o_head_stride=d,
                k_page_stride=P * Hkv * d, k_slot_stride=Hkv * d, k_head_stride=d, v_page_stride=P * Hkv * d,
                v_slot_stride=Hkv * d, v_head_stride=d, page_size=P, block_table_stride=W, max_seq_len=W * P)
    dp = hip.DeviceProblem(dict(geom=geom, q=qd, k=kp, v=vp, seq_len=plan.seq_len, kv_len=plan.kv_len, block_table=bt,
                                out_shape=(B, T, Hq, d)), mods=mods)
    assert dp.t["kv_len"].data_ptr() == plan.kv_len.data_ptr()

    def step():
        plan.build(L, cnt, bt, free, nf, P)
        r.append(q, k, v, plan.positions, plan.dst_rows, kp, vp, q_rows=plan.q_rows, q_out=qd)
        hip.launch_hip(dp, default_alpha_bits(d))
        L.copy_(plan.seq_len)
        nf.copy_(plan.num_free)

    step()  # allocations and lookups outside the capture
    torch.cuda.synchronize()
    st, g = torch.cuda.Stream(), HipGraph()
    with torch.cuda.stream(st):
        g.capture(st, step)
    L.zero_()
    nf.fill_(60)
    kp.zero_()
    ref = _Reference(r, Hq, Hkv, d, mods)
    for i in range(7):
        n = rng.integers(0, T + 1, B)
        m = int(n.sum())
        Q, K, V = (bf16(rng, (m, h, d)) for h in (Hq, Hkv, Hkv))
        cnt.copy_(i32(n))
        for t, x in ((q, Q), (k, K), (v, V)):
            t[:m].copy_(_dev(x))
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            g.replay(st)
        torch.cuda.synchronize()
        plan.check()
        rows = plan.q_rows[:m].cpu().numpy()
        out = _bits(dp.out.view(B * T, Hq, d))[rows]
        live = [b for b in range(B) if n[b]]
        want = ref.step(live, [int(n[b]) for b in live], Q, K, V) if live else out
        assert np.array_equal(out, want), i
        dead = np.setdiff1d(np.arange(B * T), rows)
        assert (_bits(dp.out.view(B * T, Hq, d))[dead] == 0).all()
    g.close()


def test_hf_softcap(gpu):
    import torch
    from exactattention_amd.serving import hf_attention
    rng = np.random.default_rng(30)
    q, k, v = bf16(rng, (2, 5, 4, 128), "normal", 4.0), bf16(rng, (2, 2, 60, 128)), bf16(rng, (2, 2, 60, 128))
    f = lambda x: _dev(x).view(torch.bfloat16)
    kv = np.tile(56 + np.arange(5), (2, 1))
    p = problem.contiguous(q, k, v, kv)
    from exactattention_amd.formats import alpha_bits_for
    for cap in (None, 20.0, 0.0):
        out, _ = hf_attention(None, f(q).transpose(1, 2), f(k), f(v), scaling=128 ** -0.5, softcap=cap)
        c = np.uint32(alpha_bits_for(cap)).view(np.float32) if cap else 0.0
        want = hip.attention_problem(p, None, alpha_bits=alpha_bits_for(128 ** -0.5), mods=hip.ScoreMods(softcap=c) if cap else None)[0]
        assert np.array_equal(_bits(out), want)
    with pytest.raises(ValueError):
        hf_attention(None, f(q).transpose(1, 2), f(k), f(v), scaling=1.0, softcap=-2.0)


def test_far_pages(gpu):
    """Pools of more than 2^31 elements: the last pages are written and read."""
    import torch
    from exactattention_amd.step import Rotary
    rng = np.random.default_rng(5)
    P, Hq, Hkv, d, n = 16, 4, 2, 128, 75
    pages = (1 << 31) // (P * Hkv * d) + 8
    q, k, v = (_dev(bf16(rng, (n, h, d))) for h in (Hq, Hkv, Hkv))
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    r, m = Rotary(d), _mods("all", Hq)
    last = np.arange(-(-n // P))[::-1] + pages - 6
    far = [torch.empty((pages, P, Hkv, d), dtype=torch.int16, device="cuda") for _ in range(2)]
    near = [torch.zeros((8, P, Hkv, d), dtype=torch.int16, device="cuda") for _ in range(2)]
    outs = []
    for (kp, vp), pg in ((far, last), (near, last - (pages - 8))):
        rows = torch.from_numpy(pg[np.arange(n) // P] * P + np.arange(n) % P).cuda()
        qr = r.append(q, k, v, pos, rows, kp, vp)
        for T in (1, 40):
            g = dict(num_seqs=1, num_tokens=T, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=d, head_dim_v=d, q_seq_stride=T * Hq * d,
                     q_tok_stride=Hq * d, q_head_stride=d, o_seq_stride=T * Hq * d, o_tok_stride=Hq * d, o_head_stride=d,
                     k_page_stride=P * Hkv * d, k_slot_stride=Hkv * d, k_head_stride=d, v_page_stride=P * Hkv * d,
                     v_slot_stride=Hkv * d, v_head_stride=d, page_size=P, block_table_stride=len(pg), max_seq_len=n)
            p = dict(geom=g, q=qr[n - T:], k=kp, v=vp, seq_len=np.array([n], np.int32),
                     kv_len=(n - T + 1 + np.arange(T)).astype(np.int32), block_table=pg[None].astype(np.int32), out_shape=(1, T, Hq, d))
            for kernel in ("auto", "general") if T == 1 else ("auto", "prefill"):
                res, fl, _ = hip.attention_problem(p, None, alpha_bits=default_alpha_bits(d), kernel=kernel, mods=m)
                outs.append(res)
    for a, b in zip(outs[:4], outs[4:]):
        assert np.array_equal(a, b)
    assert np.array_equal(outs[2], outs[3])


def test_two_streams(gpu):
    """Steps in flight on two streams, each with its workspace: the outputs of each alone."""
    import torch
    rng = np.random.default_rng(6)
    ab = default_alpha_bits(128)

    def problem_of(B, T, S):
        q, k, v = bf16(rng, (B, T, 4, 128), "normal", 2.0), bf16(rng, (B, 2, S, 128)), bf16(rng, (B, 2, S, 128))
        return problem.contiguous(q, k, v, np.tile(S - T + 1 + np.arange(T), (B, 1)))

    a = hip.DeviceProblem(problem_of(6, 1, 900), mods=_mods("all", 4))
    b = hip.DeviceProblem(problem_of(1, 300, 700), kernel="prefill", mods=_mods("cap", 4))
    c = hip.DeviceProblem(problem_of(2, 9, 1300), "fp32", mods=_mods("window", 4))
    want = []
    for dp in (a, b, c):
        hip.launch_hip(dp, ab)
        torch.cuda.synchronize()
        want.append((dp.out.clone(), dp.flags.clone()))
        dp.out.fill_(-1)
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        for dp, s in ((b, s1), (a, s2), (c, s1), (a, s2), (a, s2)):
            with torch.cuda.stream(s):
                hip.launch_hip(dp, ab)
    torch.cuda.synchronize()
    for dp, (o, f) in zip((a, b, c), want):
        assert torch.equal(dp.out, o) and torch.equal(dp.flags, f)

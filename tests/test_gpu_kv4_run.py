"""GPU: a serving loop over a cache held in 4 bits, its operators together: head norms, rotary positions and the append, attention,
the check of drafted tokens, the accepted path. Attention is compared, bit for bit, with the bf16 kernels on the values that the
cache holds; what it holds is checked where it is written (test_gpu_norm_rotary.py)."""

import numpy as np
import pytest

import draft_oracle
from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from exactattention_amd.serving import DecodeGraph, DraftCheck, ExactAttentionBackend, HeadNorm, PagedKVCache, Rotary

pytestmark = pytest.mark.gpu


class _Loop:
    def __init__(self, d=128, Hq=8, Hkv=2, P=16, seqs=3, max_len=400, mods=None, normed=True, turned=True, out="bf16", seed=0):
        import torch
        self.g = torch.Generator().manual_seed(seed)
        self.Hq, self.Hkv, self.d = Hq, Hkv, d
        self.c = PagedKVCache(num_pages=100, page_size=P, num_kv_heads=Hkv, head_dim=d, max_seqs=seqs + 1, max_seq_len=max_len, bits=4)
        w = [(1 + 0.2 * torch.randn(d, generator=self.g)).bfloat16().cuda() for _ in range(2)]
        self.rot = Rotary(d, device="cuda:0") if turned else None
        self.norm = HeadNorm(*w) if normed and turned else None
        self.mods, self.out = mods, out
        self.be = ExactAttentionBackend(self.c, Hq, None, out, alpha_bits=default_alpha_bits(d), rotary=self.rot, norm=self.norm,
                                        mods=None if mods is None else hip.ScoreMods(**mods))
        self.seqs = [self.c.add_sequence() for _ in range(seqs)]

    def new(self, n):
        import torch
        return [torch.randn((n, h, self.d), generator=self.g).bfloat16().cuda() for h in (self.Hq, self.Hkv, self.Hkv)]

    def q_of(self, q, pos):
        """q as the attention sees it, bits."""
        import torch
        if self.rot is None:
            return q.view(torch.int16).cpu().numpy().view(np.uint16)
        p = torch.tensor(pos, dtype=torch.int32, device="cuda")
        y = self.rot.rotate(q, q[:, :0], p, norm=self.norm)[0]
        return y.view(torch.int16).cpu().numpy().view(np.uint16)

    def want(self, s, q, kv_len, **tree):
        """Attention over the values of slot s's cache: q (T, Hq, d) bits."""
        import torch
        c = self.c
        n = c.length[s]
        k, v = ((x.view(torch.int16).cpu().numpy().view(np.uint16)[c.pages[s]].transpose(1, 0, 2, 3).reshape(self.Hkv, -1, self.d)[:, :n])
                for x in c.pool4.values())
        p = problem.contiguous(q[None], k[None], v[None], np.asarray(kv_len)[None], **tree)
        m = None if self.mods is None else hip.ScoreMods(**self.mods)
        return hip.attention_problem(p, None, self.out, alpha_bits=default_alpha_bits(self.d), mods=m, device="cuda:0")[0][0]


def _bits(x, fp32=False):
    return x.cpu().numpy().view(np.uint32 if fp32 else np.uint16)


@pytest.mark.parametrize("kw", [dict(), dict(d=64, P=32), dict(normed=False), dict(turned=False), dict(turned=False, d=72),
                                dict(mods=dict(window=50)), dict(mods=dict(softcap=10.0), out="fp32"), dict(Hq=2, d=96)])
def test_forward_and_decode(gpu, kw):
    """Mixed batches of chunks and single tokens, then prefill and decode."""
    L = _Loop(**kw)
    fp32 = L.out == "fp32"
    c = L.c
    for ql in ([70, 3, 40], [1, 1, 1], [1, 5, 1], [90, 2, 1], [1, 1, 1]):
        q, k, v = L.new(sum(ql))
        before = [c.length[s] for s in L.seqs]
        out, flags = L.be.forward(q, k, v, L.seqs, ql)
        L.be.check_flags(flags)
        got, at = _bits(out, fp32), 0
        for s, n, b in zip(L.seqs, ql, before):
            pos = b + np.arange(n)
            assert np.array_equal(got[at:at + n], L.want(s, L.q_of(q[at:at + n], pos), pos + 1)), (ql, s)
            at += n
    s = L.seqs[1]
    q, k, v = L.new(33)
    b = c.length[s]
    got, _ = L.be.prefill(s, q, k, v)
    assert np.array_equal(got, L.want(s, L.q_of(q, b + np.arange(33)), b + 1 + np.arange(33)))
    q, k, v = L.new(3)
    before = [c.length[s] for s in L.seqs]
    got, _ = L.be.decode(L.seqs, q, k, v)
    for i, s in enumerate(L.seqs):
        assert np.array_equal(got[i:i + 1], L.want(s, L.q_of(q[i:i + 1], [before[i]]), [before[i] + 1]))


@pytest.mark.parametrize("turned", [True, False])
def test_draft_tree_and_acceptance(gpu, turned):
    """A draft tree verified, its nodes checked against the target's probabilities (a head on the attention's output), the path that
    stands accepted: the cache then holds what it would had those tokens been appended."""
    import torch
    L = _Loop(turned=turned)
    c, s, V, N = L.c, L.seqs[0], 500, 12
    rng = np.random.default_rng(1)
    head = torch.randn((L.Hq * L.d, V), generator=L.g).cuda() * 0.05
    q, k, v = L.new(90)
    L.be.prefill(s, q, k, v)
    parents = [-1, -1, 0, 0, 1, 2, 2, 5, 3, 7, 9, 9]
    check = DraftCheck(1, N, V, "cuda:0")
    stood = 0
    for turn in range(6):
        n0 = c.length[s]
        q, k, v = L.new(N)
        host = [x.view(torch.int16).cpu().numpy().view(np.uint16) for x in (k, v)]
        a, b = (k, v) if turned else host
        out, _ = L.be.verify_tree(s, q, a, b, parents)
        depth = []
        for p in parents:
            depth.append(depth[p] + 1 if p >= 0 else 0)
        mask = np.zeros((1, N), np.uint64)
        for i in range(N):
            j = i
            while j >= 0:
                mask[0, i] |= np.uint64(1 << j)
                j = parents[j]
        want = L.want(s, L.q_of(q, n0 + np.array(depth)), np.full(N, n0), tree_mask=mask, tree_base=[n0])
        assert np.array_equal(out, want)
        hidden = torch.from_numpy(out.view(np.int16)).cuda().view(torch.bfloat16).float().view(N, -1)
        rows = torch.cat([hidden[:1], hidden]) @ head  # the prefix's own row: any
        probs = torch.softmax(12.0 * rows, -1)[None]  # sharp enough that drafted tokens stand
        # drafted: likely tokens of their parents' rows
        top = rows.topk(3, -1).indices.cpu().numpy()
        drafted = np.array([[top[parents[i] + 1, sum(p == parents[i] for p in parents[:i])] for i in range(N)]])
        u = rng.random((1, N + 1), dtype=np.float32) * 0.5
        check.verify(probs, torch.from_numpy(drafted).int().cuda(), torch.from_numpy(u).cuda(),
                     parents=torch.tensor([parents], dtype=torch.int32, device="cuda"))
        path = check.paths()[0]
        want_path, _, _, _ = draft_oracle.check(probs[0].cpu().numpy(), drafted[0], u[0], None, parents)
        assert path == want_path
        stood += len(path)
        L.be.accept(s, n0, path, a, b)
        assert c.length[s] == n0 + len(path)
        # the same tokens appended to a fresh loop's slot after the same prefix
        got = [x.float().cpu().numpy() for x in c.pool4.values()]
        other = _Loop(turned=turned)
        t = other.seqs[0]
        if path:
            idx = torch.tensor(path, device="cuda")
            other.c.length[t] = 0
            pos = torch.arange(n0, n0 + len(path), dtype=torch.int32, device="cuda")
            rows_at = torch.arange(len(path), device="cuda")
            if turned:
                L.rot.append(q[:len(path)], k[idx], v[idx], pos, rows_at, other.c.pool4, norm=L.norm)
            else:
                other.c.pool4.append(k[idx], v[idx], rows_at)
            ref = [x.float().cpu().numpy() for x in other.c.pool4.values()]
            for g, r in zip(got, ref):
                for i in range(len(path)):
                    page, slot = c.pages[s][(n0 + i) // c.P], (n0 + i) % c.P
                    assert np.array_equal(g[page, :, slot], r[i // c.P, :, i % c.P])
    assert stood > 3


@pytest.mark.parametrize("kw", [dict(), dict(d=64, mods=dict(window=40)), dict(turned=False)])
def test_decode_graph(gpu, kw):
    """The captured decode step against the eager one of a second loop on the same inputs."""
    import torch
    a, b = _Loop(**kw), _Loop(**kw)
    for L in (a, b):
        q, k, v = L.new(60 + 7 + 30)
        L.be.forward(q, k, v, L.seqs, [60, 7, 30])
    torch.cuda.synchronize()
    g = DecodeGraph(a.be, a.seqs, max_len=300)
    for i in range(40):
        q, k, v = a.new(3)
        g.q.copy_(q.view(torch.int16)[:, None])
        g.k.copy_(k.view(torch.int16))
        g.v.copy_(v.view(torch.int16))
        out, flags = g.step()
        g.check_flags(flags)
        out2, flags2 = b.be.forward(q, k, v, b.seqs, [1, 1, 1])
        b.be.check_flags(flags2)
        assert torch.equal(out, out2), i
    assert torch.equal(a.c.pool4.k, b.c.pool4.k) and torch.equal(a.c.pool4.v_scales, b.c.pool4.v_scales)
    g.close()


def test_truncated_and_reused_pages(gpu):
    """Slots dropped and taken again, sequences cut back, pages in another order."""
    L = _Loop(seqs=2)
    c = L.c
    for turn in range(3):
        q, k, v = L.new(50 + 20)
        L.be.forward(q, k, v, L.seqs, [50, 20])
        c.truncate(L.seqs[0], c.length[L.seqs[0]] - 33)
        c.drop_sequence(L.seqs[1])
        L.seqs[1] = c.add_sequence()
        q, k, v = L.new(2)
        before = [c.length[s] for s in L.seqs]
        out, flags = L.be.forward(q, k, v, L.seqs, [1, 1])
        L.be.check_flags(flags)
        for i, s in enumerate(L.seqs):
            assert np.array_equal(_bits(out)[i:i + 1], L.want(s, L.q_of(q[i:i + 1], [before[i]]), [before[i] + 1]))


def test_norms_over_a_bf16_cache(gpu):
    """The backend's norms with 16-bit pages: what the rotation with the norm by itself gives, appended unturned."""
    import torch
    d, Hq, Hkv = 128, 4, 2
    g = torch.Generator().manual_seed(3)
    rot = Rotary(d, device="cuda:0")
    norm = HeadNorm(*((1 + 0.2 * torch.randn(d, generator=g)).cuda() for _ in range(2)))
    caches = [PagedKVCache(20, 16, Hkv, d, 2, 200) for _ in range(2)]
    ab = default_alpha_bits(d)
    one = ExactAttentionBackend(caches[0], Hq, alpha_bits=ab, rotary=rot, norm=norm)
    two = ExactAttentionBackend(caches[1], Hq, alpha_bits=ab)
    s = [c.add_sequence() for c in caches]
    at = 0
    for n in (70, 1, 9):
        q, k, v = (torch.randn((n, h, d), generator=g).bfloat16().cuda() for h in (Hq, Hkv, Hkv))
        a, fa = one.forward(q, k, v, s[:1], [n])
        pos = torch.arange(at, at + n, dtype=torch.int32, device="cuda")
        b, fb = two.forward(*rot.rotate(q, k, pos, norm=norm), v, s[1:], [n])
        assert torch.equal(a, b) and not bool(fa.any()) and not bool(fb.any())
        at += n


def test_refusals(gpu):
    import torch
    c = PagedKVCache(4, 16, 2, 64, 1, 64, bits=4)
    w = torch.ones(64, device="cuda")
    with pytest.raises(ValueError, match="rotary"):
        ExactAttentionBackend(c, 2, 0.1, norm=HeadNorm(w, w))
    with pytest.raises(ValueError):
        ExactAttentionBackend(c, 2, 0.1, rotary=Rotary(64, device="cuda:0"), norm=HeadNorm(w[:32], w[:32]))
    with pytest.raises(ValueError, match="multiple of 4"):
        ExactAttentionBackend(c, 2, 0.1, rotary=Rotary(64, rot_dim=30, device="cuda:0"))
    with pytest.raises(ValueError):
        PagedKVCache(4, 8, 2, 64, 1, 64, bits=4)
    with pytest.raises(ValueError):
        PagedKVCache(4, 16, 2, 60, 1, 64, bits=4)
    p = problem.contiguous(np.zeros((1, 1, 2, 64), np.uint16), np.zeros((1, 2, 8, 64), np.uint16), np.zeros((1, 2, 8, 64), np.uint16), [[8]])
    with pytest.raises(ValueError, match="geometry"):
        hip.DeviceProblem({**p, "kv4": c.pool4})

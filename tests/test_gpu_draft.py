"""GPU: which drafted tokens stand, against the definition with Python numbers, and against the distribution that it keeps."""

import numpy as np
import pytest

import draft_oracle as oracle
from exactattention_amd.step import DraftCheck

pytestmark = pytest.mark.gpu


def _cuda(x, dt):
    import torch
    return None if x is None else torch.from_numpy(np.ascontiguousarray(x, dtype=dt)).cuda()


def _run(p, x, u, q=None, par=None, counts=None, check=None, pt=None):
    import torch
    B, n1, V = p.shape
    c = check or DraftCheck(B, n1 - 1, V, "cuda:0")
    c.verify(_cuda(p, np.float32) if pt is None else pt, _cuda(x, np.int32), _cuda(u, np.float32), draft_probs=_cuda(q, np.float32),
             parents=_cuda(par, np.int32), counts=_cuda(counts, np.int32))
    torch.cuda.synchronize()
    return c.accepted.tolist(), c.path.tolist(), c.tokens.tolist(), c


def _check(p, x, u, q=None, par=None, counts=None, **kw):
    B, n1, _ = p.shape
    acc, path, tok, c = _run(p, x, u, q, par, counts, **kw)
    for b in range(B):
        want = oracle.check(p[b], x[b], u[b], None if q is None else q[b], None if par is None else par[b],
                            None if counts is None else counts[b])
        # masses of siblings are sums in two orders: fp64 roundings of up to 64 terms
        assert want[3] > 2.0 ** -46 or want[3] == 0.0
        n, pp, tt = oracle.outputs(n1 - 1, *want[:3])
        assert (acc[b], path[b], tok[b]) == (n, pp, tt), b
    assert not bool(c._work.view(B, -1)[:, -1].any())
    assert c.paths() == [[i for i in q_ if i >= 0] for q_ in path]
    return acc, path, tok


def _tree(rng, B, N):
    return np.array([[rng.integers(-1, i) if i else -1 for i in range(N)] for _ in range(B)]).reshape(B, N)


@pytest.mark.parametrize("op", ["chain", "given", "tree"])
@pytest.mark.parametrize("B,N,V", [(1, 1, 7), (3, 4, 1000), (2, 16, 5001), (5, 64, 130), (40, 3, 2049), (2, 5, 70001), (3, 0, 50),
                                   (4, 2, 1)])
def test_against_the_definition(gpu, op, B, N, V):
    rng = np.random.default_rng(B + 10 * N + V)
    p = oracle.softmax(rng, (B, N + 1, V), 2.5)
    q = par = None
    if op == "chain":
        q = np.sqrt(p[:, :N] * oracle.softmax(rng, (B, N, V), 2.0))
        q = (q / q.sum(-1, keepdims=True)).astype(np.float32)
        x = np.array([[rng.choice(V, p=r.astype(np.float64) / r.astype(np.float64).sum()) for r in rows] for rows in q]).reshape(B, N)
    else:
        par = _tree(rng, B, N) if op == "tree" else None
        src = (par if par is not None else np.broadcast_to(np.arange(N) - 1, (B, N))) + 1
        top = np.argsort(-p, -1)[..., :4]
        x = np.array([[top[b, src[b, i], rng.integers(0, min(4, V))] for i in range(N)] for b in range(B)]).reshape(B, N)
    for counts in (None, rng.integers(0, N + 1, B)):
        _check(p, x, rng.random((B, N + 1), dtype=np.float32), q, par, counts)


def test_edges_of_the_numbers(gpu):
    """Uniform numbers of 0, just below 1 and outside; certain and impossible tokens; rows of zeros, of NaN and of numbers past 1."""
    rng = np.random.default_rng(1)
    N, V = 3, 300
    one = np.float32(1 - 2.0 ** -24)
    for u in (0.0, one, 1.0, 2.0, -1.0, float("nan"), 2.0 ** -30):
        p = oracle.softmax(rng, (6, N + 1, V), 3.0)
        q = oracle.softmax(rng, (6, N, V), 3.0)
        x = rng.integers(0, V, (6, N))
        p[0] = 0
        p[0, :, 7] = 1
        x[0] = 7
        p[1] = 0
        p[2] = np.nan
        p[3, :, ::2] = np.nan
        p[4] *= 1000
        q[5, :, x[5]] = 0
        uu = np.full((6, N + 1), u, np.float32)
        for kw in (dict(q=q), dict()):
            _check(p, x, uu, **kw)
    # the target's and the draft's probabilities the same: all stand; the draft's larger everywhere: p itself is taken
    p = oracle.softmax(rng, (2, N + 1, V), 3.0)
    q = p[:, :N].copy()
    q[1] = np.minimum(1, q[1] * 3)
    acc, _, tok = _check(p, np.argmax(q, -1), np.full((2, N + 1), 0.9, np.float32), q)
    assert acc[0] == N


def test_nodes_that_are_none(gpu):
    """Tokens outside the vocabulary, parents at or past their node, the same token twice, and counts outside 0 .. N."""
    rng = np.random.default_rng(2)
    B, N, V = 8, 6, 40
    p = oracle.softmax(rng, (B, N + 1, V), 1.0)
    x = rng.integers(0, 3, (B, N))
    par = _tree(rng, B, N)
    par[1, 2], par[1, 0], par[2, 3] = 2, 5, -7
    x[3, 0], x[4, 1], x[5, 0] = -1, V, 1 << 30
    par[6], x[6] = -1, 5
    for counts in (None, np.array([-3, 0, 1, 2, 6, 7, 100, 5])):
        for _ in range(4):
            _check(p, x, rng.random((B, N + 1), dtype=np.float32), None, par, counts)


def test_strides_and_alignment(gpu):
    """Rows of a larger tensor that start anywhere, sequences far apart."""
    import torch
    rng = np.random.default_rng(3)
    B, N, V = 3, 2, 1023
    p = oracle.softmax(rng, (B, N + 1, V), 2.0)
    x, u = rng.integers(0, V, (B, N)), rng.random((B, N + 1), dtype=np.float32)
    big = torch.full((B, N + 3, V + 9), float("nan"), device="cuda")
    view = big[:, 1:N + 2, 5:V + 5]
    view.copy_(_cuda(p, np.float32))
    _check(p, x, u, pt=view)


@pytest.mark.parametrize("V", [1 << 19, 300001])
def test_large_vocabularies(gpu, V):
    """The largest vocabulary; a flat distribution, whose borders lie closest, and tokens at both ends."""
    rng = np.random.default_rng(V)
    p = np.full((2, 2, V), np.float32(1.0 / V))
    p[1] = 0
    p[1, :, V - 1] = 0.5
    p[1, :, 0] = 0.5
    for _ in range(3):
        u = rng.random((2, 2), dtype=np.float32)
        x = rng.integers(0, V, (2, 1))
        acc, _, tok, _ = _run(p, x, u)
        w = (p.astype(np.float64) * 2.0 ** 44).astype(np.int64)
        for b in range(2):
            assert acc[b] == int(u[b, 0] < p[b, 0, x[b, 0]])
            row = w[b, acc[b]].copy()
            if not acc[b]:
                row[x[b, 0]] = 0
            c = np.cumsum(row)
            assert tok[b][acc[b]] == int(np.searchsorted(c, int(float(u[b, 1]) * float(c[-1])), "right"))


@pytest.mark.parametrize("op", ["chain", "tree"])
def test_the_distribution_stays(gpu, op):
    """First tokens of many sequences with one target distribution: each token's count is a binomial one, within 6 deviations of its
    mean (10 of them: wrong once in 10^8)."""
    rng = np.random.default_rng(4)
    B, V, N = 60000, 5, 3
    p1, q1 = oracle.softmax(rng, (V,), 1.0), oracle.softmax(rng, (V,), 1.0)
    p = np.broadcast_to(p1, (B, N + 1, V))
    q = par = None
    if op == "chain":
        q = np.broadcast_to(q1, (B, N, V))
        x = rng.choice(V, (B, N), p=q1.astype(np.float64) / q1.astype(np.float64).sum())
    else:
        par = np.broadcast_to(np.array([-1, -1, 0]), (B, N))
        x = np.broadcast_to(np.array([2, 0, 1]), (B, N))
    _, _, tok, _ = _run(p, x, rng.random((B, N + 1), dtype=np.float32), q, par)
    tok = np.array(tok)
    for place in (0, 1):
        t = tok[:, place][tok[:, place] >= 0]
        n, c = len(t), np.bincount(t, minlength=V)
        pr = p1.astype(np.float64) / p1.astype(np.float64).sum()
        if place == 0:
            assert n == B
        assert np.all(np.abs(c - n * pr) <= 6 * np.sqrt(n * pr * (1 - pr)) + 1)


def test_streams_graphs_and_reuse(gpu):
    """One object called again and again, captured and replayed on new numbers, and two objects in flight on two streams."""
    import torch
    rng = np.random.default_rng(5)
    B, N, V = 9, 4, 40000
    p = oracle.softmax(rng, (B, N + 1, V), 3.0)
    x = np.argsort(-p, -1)[:, :N, 0]
    u = rng.random((B, N + 1), dtype=np.float32)
    pt, xt, ut = _cuda(p, np.float32), _cuda(x, np.int32), _cuda(u, np.float32)
    a, b = DraftCheck(B, N, V, "cuda:0"), DraftCheck(B, N, V, "cuda:0")
    st = torch.cuda.Stream()
    torch.cuda.synchronize()
    for _ in range(20):
        with torch.cuda.stream(st):
            a.verify(pt, xt, ut)
        b.verify(pt, xt, ut)
    torch.cuda.synchronize()
    want = [oracle.outputs(N, *oracle.check(p[i], x[i], u[i])[:3]) for i in range(B)]
    for c in (a, b):
        assert list(zip(c.accepted.tolist(), c.path.tolist(), c.tokens.tolist())) == want
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        a.verify(pt, xt, ut)
    for i in range(4):
        ut.copy_(torch.rand((B, N + 1), generator=torch.Generator().manual_seed(i)))
        graph.replay()
        b.verify(pt, xt, ut)
        torch.cuda.synchronize()
        assert torch.equal(a.tokens, b.tokens) and torch.equal(a.path, b.path) and torch.equal(a.accepted, b.accepted)


def test_calls_in_a_row(gpu):
    """Many blocks a sequence, whose last one joins the sums, called again and again without a wait in between."""
    import torch
    rng = np.random.default_rng(11)
    B, N, V = 48, 3, 40000
    c = DraftCheck(B, N, V, "cuda:0")
    sets, want = [], []
    for _ in range(2):
        p = oracle.softmax(rng, (B, N + 1, V), 2.5)
        x = np.argsort(-p, -1)[:, :N, 0].copy()
        u = rng.random((B, N + 1)).astype(np.float32)
        want.append(_check(p, x, u))
        sets.append((_cuda(p, np.float32), _cuda(x, np.int32), _cuda(u, np.float32)))
    got = []
    for i in range(200):
        c.verify(*sets[i % 2])
        got.append(torch.cat([c.accepted[:, None], c.path, c.tokens], 1))
    for i, t in enumerate(got):
        acc, path, tok = want[i % 2]
        assert t.tolist() == [[a, *b, *d] for a, b, d in zip(acc, path, tok)], i


def test_refusals(gpu):
    import torch
    for a in ((-1, 1, 5), (1, 65, 5), (1, 1, 0), (1, 1, (1 << 19) + 1), (65536, 1, 5)):
        with pytest.raises(ValueError):
            DraftCheck(*a, "cuda:0")
    with pytest.raises(ValueError):
        DraftCheck(1, 1, 5, "cpu")
    B, N, V = 2, 3, 50
    c = DraftCheck(B, N, V, "cuda:0")
    p, q = torch.zeros((B, N + 1, V), device="cuda"), torch.zeros((B, N, V), device="cuda")
    x, u = torch.zeros((B, N), dtype=torch.int32, device="cuda"), torch.zeros((B, N + 1), device="cuda")
    ok = dict(probs=p, drafted=x, uniforms=u)
    for bad in (dict(probs=p[:, :N]), dict(probs=p.half()), dict(probs=p.transpose(1, 2)), dict(probs=p.cpu()), dict(drafted=x.long()),
                dict(drafted=x[:, :2]), dict(uniforms=u.double()), dict(uniforms=u[:, :N]), dict(draft_probs=p), dict(counts=x),
                dict(parents=x[0]), dict(draft_probs=q, parents=x), dict(drafted=c.path), dict(parents=c.path), dict(counts=c.accepted)):
        with pytest.raises(ValueError):
            c.verify(**{**ok, **bad})
    c.verify(**ok)
    DraftCheck(0, 2, 5, "cuda:0").verify(p[:0, :3, :5].contiguous(), x[:0, :2].contiguous(), u[:0, :3].contiguous())

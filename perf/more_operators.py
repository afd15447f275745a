"""The operators of a serving step over a cache held in 4 bits, with drafted tokens, as cases that can be timed.

A step of a model that norms its queries and keys for each head runs them in turn, and each is
measured by itself:

  append  q and k normed for each head and turned by their positions; q goes to the attention, k and v
          into the paged cache in 4 bits (elements of 1 sign, 2 exponent and 1 mantissa bit, a power
          of two for each 32 of them)
  turn    the same norm and rotation in training: forward and backward, with the weights' gradients
  attend  attention over that cache: decode, drafted tokens, prompt chunks
  verify  which drafted tokens stand, from the target's probabilities and given uniform numbers, and
          the token after them

With own = False `run` computes an operator in its plain form (torch, elementary operations); with
own = True it makes the library's calls. Both read what `prepare` made.
"""

from __future__ import annotations

import math
import random
from types import SimpleNamespace

import numpy as np
import torch

own = False

LOG2E = 1.0 / math.log(2.0)

# append: N tokens, the last `pad` of them without a slot; rot rotated dims of d; norm: weights for the
# heads of q and k; adjacent: pairs (2i, 2i+1), else (i, i + rot/2)
_APPEND = dict(kind="append", d=128, rot=128, norm=True, adjacent=False, page=16, dtype="bf16", pad=0, maxpos=8192)
# turn: N tokens forward and backward
_TURN = dict(kind="turn", d=128, rot=128, adjacent=False, dtype="bf16", maxpos=8192)
# attend: B sequences of kv_min..kv keys (spread over the logarithm by `lens`), T tokens at the end of each
_ATTEND = dict(kind="attend", T=1, d=128, page=16, lens=0, qscale=1.0)
# verify: N drafted nodes of each of B sequences (fewer for some, `lens`), V tokens; op "chain": drawn from
# given probabilities, "given": a chain of given tokens, "tree": trees of given tokens; sharp: scale of the logits
_VERIFY = dict(kind="verify", op="chain", lens=0, sharp=3.0)


def _case(base, name, **kw):
    c = dict(base, **kw)
    if base is _ATTEND:
        c.setdefault("kv_min", c["kv"])
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # the new tokens of a decode step
        _case(_APPEND, "append_decode_33", N=33, Hq=32, Hkv=8),
        # prompt chunks of a scheduler's largest step, the last tokens are padding
        _case(_APPEND, "append_prompts_16k", N=16384, Hq=32, Hkv=8, page=64, pad=5),
        # a training step's tokens
        _case(_TURN, "turn_train_4096", N=4096, Hq=16, Hkv=8),
        # in fp32, on part of each head
        _case(_TURN, "turn_train_fp32_2001", N=2001, Hq=12, Hkv=4, d=96, rot=64, dtype="fp32"),
        # one token of a chat turn: latency
        _case(_ATTEND, "attend_decode_900", B=1, kv=900, Hq=16, Hkv=8),
        # a running batch's decode, wide groups
        _case(_ATTEND, "attend_decode_ragged", B=32, kv=4096, kv_min=512, lens=3, Hq=32, Hkv=8),
        # decode far into long contexts, what a small cache is for
        _case(_ATTEND, "attend_decode_long", B=8, kv=131072, kv_min=30000, lens=5, Hq=16, Hkv=8, page=64),
        # drafted tokens on long prefixes
        _case(_ATTEND, "attend_draft_8x16k", B=8, T=8, kv=16384, kv_min=9000, lens=7, Hq=16, Hkv=8),
        # a prompt chunk after a cached prefix
        _case(_ATTEND, "attend_chunk_1500", B=1, T=1500, kv=4000, Hq=16, Hkv=8),
        # one sequence's drafted tokens: latency
        _case(_VERIFY, "verify_chat_4", B=1, N=4, V=32000),
        # a running batch's, some of them with fewer tokens
        _case(_VERIFY, "verify_batch_64x8", B=64, N=8, V=128000, lens=3),
        # draft trees
        _case(_VERIFY, "verify_trees_16", op="tree", B=16, N=16, V=50021, sharp=4.0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges: no more tokens, pairs, keys or probabilities than the largest listed."""
    kind = rng.choice(["append", "append", "turn", "attend", "attend", "attend", "verify", "verify"])
    Hkv = rng.choice([1, 2, 4, 8])
    grp = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 16, 32, 64])
    d = rng.choice([128, 128, 64, 96, 80])
    if kind == "append":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        most = 16384 * 48 * 128 // (Hkv * (grp + 2) * d)
        N = _log(rng, 1, min(16384, most if dtype == "bf16" else most // 2))
        return _case(_APPEND, None, N=N, Hq=Hkv * grp, Hkv=Hkv, d=d, rot=rng.choice([d, d, d // 2]), norm=rng.random() < 0.7,
                     adjacent=rng.random() < 0.3, page=page, dtype=dtype, pad=rng.choice([0, 0, min(N, 7)]),
                     maxpos=rng.choice([4096, 32768]))
    if kind == "turn":
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        most = 4096 * 24 * 128 // (Hkv * (grp + 1) * d)
        N = _log(rng, 1, min(4096, most if dtype == "bf16" else most // 2))
        return _case(_TURN, None, N=N, Hq=Hkv * grp, Hkv=Hkv, d=d, rot=rng.choice([d, d, d // 2]), adjacent=rng.random() < 0.3,
                     dtype=dtype, maxpos=rng.choice([4096, 32768]))
    if kind == "attend":
        lens = rng.randrange(1 << 20)
        what = rng.choice(["decode", "decode", "draft", "chunk"])
        base = dict(Hq=Hkv * grp, Hkv=Hkv, d=d, page=page, lens=lens, qscale=rng.choice([1.0, 1.0, 2.0]))
        if what == "decode":
            B = _log(rng, 1, 32)
            kv = _log(rng, 1, min(131072, 400_000 // (B * grp)))
            return _case(_ATTEND, None, B=B, kv=kv, kv_min=rng.choice([kv, max(1, kv // 8)]), **base)
        if what == "draft":
            T, B = _log(rng, 2, 20), _log(rng, 1, 8)
            kv = _log(rng, T, max(T, 400_000 // (B * T * grp)))
            return _case(_ATTEND, None, B=B, T=T, kv=kv, kv_min=rng.choice([kv, max(T, kv // 4)]), **base)
        T = _log(rng, 20, 1500)
        kv = T + rng.choice([0, _log(rng, 1, 3000)])
        if T * kv * Hkv * grp > 1500 * 4000 * 16:
            base["Hkv"], base["Hq"] = 1, grp
        return _case(_ATTEND, None, B=1, T=T, kv=kv, **base)
    op = rng.choice(["chain", "chain", "given", "tree"])
    V = _log(rng, 1000, 128000)
    N = rng.randint(2, 16) if op == "tree" else _log(rng, 1, 10)
    B = _log(rng, 1, max(1, min(64, 64 * 8 * 128000 // (V * N) // 2)))
    return _case(_VERIFY, None, op=op, B=B, N=N, V=V, lens=rng.choice([0, rng.randrange(1, 1 << 20)]),
                 sharp=rng.choice([2.0, 3.0, 5.0]))


# ---- what a case holds

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _width(d):
    """Elements a row of d takes in the cache: whole groups of 32."""
    return (d + 31) // 32 * 32


def _four_bits(x):
    """(magnitudes 0..6, exponents) of x (..., whole groups of 32): the smallest power of two e with max|x| <
    7 * 2^e, elements to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 times it, ties to the even code."""
    g = x.unflatten(-1, (-1, 32))
    m, e = torch.frexp(g.abs().amax(-1))
    e = torch.where(m < 0.875, e - 3, e - 2)
    e = torch.where(m == 0, torch.full_like(e, -125), e.clamp(-125, 125))
    y = torch.ldexp(g, -e[..., None]).abs()
    s = torch.where(y < 2, 0.5, torch.where(y < 4, 1.0, 2.0))
    y = (torch.round(y / s) * s).clamp(max=6.0)
    return y, e


def _values(x):
    """x in 4 bits, as the values that stands for."""
    y, e = _four_bits(x)
    return (torch.ldexp(y, e[..., None]) * torch.sign(x.unflatten(-1, (-1, 32)))).flatten(-2)


def _codes(x):
    """x (..., d) in 4 bits: bytes of two elements, the first in the low half, and the exponents + 127."""
    x = torch.nn.functional.pad(x.float(), (0, _width(x.shape[-1]) - x.shape[-1]))
    y, e = _four_bits(x)
    c = torch.where(y < 2, 2 * y, torch.where(y < 4, y + 2, y / 2 + 4)).to(torch.uint8).flatten(-2)
    c = c | (torch.signbit(x).to(torch.uint8) << 3)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).contiguous(), (e + 127).to(torch.uint8)


def _spell(codes, scales, d):
    """The values of _codes' bytes, in 32 bits."""
    c = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    lut = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
    y = torch.cat([lut, -lut])[c.long()].unflatten(-1, (-1, 32))
    return torch.ldexp(y, (scales.int() - 127)[..., None]).flatten(-2)[..., :d]


def _pool(pages, Hkv, P, d, gen):
    """A cache's pages: the codes and scales of normal values, some channels larger than the others."""
    big = torch.exp(0.5 * torch.randn(d, device="cuda", generator=gen))
    parts = [_codes(_normal((min(4096, pages - a), Hkv, P, d), gen, torch.float32) * big) for a in range(0, pages, 4096)]
    return torch.cat([c for c, _ in parts]), torch.cat([e for _, e in parts])


def _lens(case):
    """Keys of each sequence, the tokens' own among them."""
    lo, hi = max(case["kv_min"], case["T"]), case["kv"]
    r = random.Random(case["lens"])
    return [hi] + [_log(r, lo, hi) for _ in range(case["B"] - 1)]


def _attend_inputs(case, seed):
    gen, r = _gen(seed), np.random.default_rng(seed)
    B, T, Hq, Hkv, d, P = (case[x] for x in ("B", "T", "Hq", "Hkv", "d", "page"))
    lens = _lens(case)
    s = SimpleNamespace(lens=lens)
    s.q = _normal((B, T, Hq, d), gen) * case["qscale"]
    need = [-(-n // P) for n in lens]
    perm = r.permutation(sum(need)).astype(np.int32)
    bt, at = np.zeros((B, max(need)), np.int32), 0
    for b, n in enumerate(need):
        bt[b, :n] = perm[at:at + n]
        at += n
    s.bt = _i32(bt)
    s.kc, s.ks = _pool(sum(need), Hkv, P, d, gen)
    s.vc, s.vs = _pool(sum(need), Hkv, P, d, gen)
    s.kv_len = _i32([[n - T + 1 + t for t in range(T)] for n in lens])
    s.alpha = float(np.float32(d ** -0.5 * LOG2E))
    return s


def _qkv(case, seed, grads):
    """q, k and v as a projection leaves them, parts of one row per token; positions, weights."""
    gen, r = _gen(seed), np.random.default_rng(seed)
    N, Hq, Hkv, d = (case[x] for x in ("N", "Hq", "Hkv", "d"))
    dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    s = SimpleNamespace()
    qkv = _normal((N, (Hq + 2 * Hkv) * d), gen, dt)
    s.q = qkv[:, :Hq * d].view(N, Hq, d)
    s.k = qkv[:, Hq * d:(Hq + Hkv) * d].view(N, Hkv, d)
    s.v = qkv[:, (Hq + Hkv) * d:].view(N, Hkv, d)
    s.qw, s.kw = (1 + 0.2 * _normal((d,), gen, torch.float32)).to(dt), (1 + 0.2 * _normal((d,), gen, torch.float32)).to(dt)
    s.positions = _i32(r.integers(0, case["maxpos"], N))
    half = case["rot"] // 2
    s.inv_freq = 10000.0 ** (-np.arange(half, dtype=np.float64) / half)
    s.eps = 1e-6
    if grads:
        s.gq, s.gk = _normal((N, Hq, d), gen, dt), _normal((N, Hkv, d), gen, dt)
    return s, gen, r


def _append_inputs(case, seed):
    s, gen, r = _qkv(case, seed, False)
    N, P, Hkv, d = case["N"], case["page"], case["Hkv"], case["d"]
    pages = (N + P - 1) // P + 3
    dst = r.permutation(pages * P)[:N].astype(np.int64)
    if case["pad"]:
        dst[N - case["pad"]:] = -1
    s.dst = torch.from_numpy(dst).cuda()
    s.pools = _pool(pages, Hkv, P, d, gen) + _pool(pages, Hkv, P, d, gen)
    return s


def _tree(case):
    """(B, N) parents of the nodes (-1: the prefix), and how many each sequence has."""
    r = random.Random(case["lens"])
    B, N = case["B"], case["N"]
    n = [N] + [r.randint(0, N) if case["lens"] else N for _ in range(B - 1)]
    if case["op"] != "tree":
        return np.broadcast_to(np.arange(N) - 1, (B, N)), n
    return np.array([[r.randint(max(-1, i - 6), i - 1) for i in range(N)] for _ in range(B)]), n


def _verify_inputs(case, seed):
    gen = _gen(seed)
    B, N, V = case["B"], case["N"], case["V"]
    par, n = _tree(case)
    s = SimpleNamespace()
    logits = case["sharp"] * _normal((B, N + 1, V), gen, torch.float32)
    s.p = torch.softmax(logits, -1)
    s.qp = None
    if case["op"] == "chain":
        # a draft model near the target, and what it drew
        logits = logits[:, :N] + 0.7 * _normal((B, N, V), gen, torch.float32)
        s.qp = torch.softmax(logits, -1)
        logits -= torch.empty_like(logits).exponential_(generator=gen).log_()
        s.drafted = logits.argmax(-1).int()
    else:
        # the draft's likeliest tokens, the j-th child of a node its j-th one
        top = (logits + 0.5 * _normal(logits.shape, gen, torch.float32)).topk(min(V, 8), -1).indices
        rank = np.array([[sum(p[j] == p[i] for j in range(i)) for i in range(N)] for p in par])
        b = torch.arange(B, device="cuda")[:, None]
        s.drafted = top[b, torch.from_numpy(par + 1).cuda(), torch.from_numpy(rank % min(V, 8)).cuda()].int()
    s.u = torch.rand((B, N + 1), device="cuda", generator=gen)
    s.count = _i32(n)
    s.parents = _i32(par) if case["op"] == "tree" else None
    # a node's ancestors and itself, as the attention's masks have them
    anc = np.zeros((B, N, N), bool)
    for b in range(B):
        for i in range(N):
            anc[b, i, i] = True
            if par[b][i] >= 0:
                anc[b, i] |= anc[b, par[b][i]]
    s.par, s.anc = torch.from_numpy(np.ascontiguousarray(par)).cuda(), torch.from_numpy(anc).cuda()
    return s


def prepare(case, seed):
    kind = case["kind"]
    if kind == "attend":
        s = _attend_inputs(case, seed)
    elif kind == "append":
        s = _append_inputs(case, seed)
    elif kind == "turn":
        s = _qkv(case, seed, True)[0]
    else:
        s = _verify_inputs(case, seed)
    s.case = case
    if own:
        _plans(s)
    elif kind in ("append", "turn"):
        s.w = torch.from_numpy(s.inv_freq).cuda()
        if kind == "append":  # the plain form keeps its cache in values
            s.kp, s.vp = (_spell(*s.pools[i:i + 2], case["d"]).to(torch.bfloat16) for i in (0, 2))
    return s


def _plans(s):
    """What a program that serves or trains keeps beside its inputs."""
    c = s.case
    if c["kind"] in ("append", "turn"):
        from exactattention_amd.serving import HeadNorm, KV4Pool, Rotary
        s.rotary = Rotary(c["d"], rot_dim=c["rot"], inv_freq=s.inv_freq, adjacent=c["adjacent"])
        s.norm = HeadNorm(s.qw, s.kw, s.eps) if c.get("norm", True) else None
        if c["kind"] == "append":
            s.pool = KV4Pool.of(*s.pools, head_dim=c["d"])
        else:
            s.leaves = [x.requires_grad_() for x in (s.q.detach(), s.k.detach(), s.qw, s.kw)]
    elif c["kind"] == "attend":
        from exactattention_amd import hip
        from exactattention_amd.serving import KV4Pool
        B, T, Hq, Hkv, d, P = (c[x] for x in ("B", "T", "Hq", "Hkv", "d", "page"))
        pool = KV4Pool.of(s.kc, s.ks, s.vc, s.vs, head_dim=d)
        geom = dict(num_seqs=B, num_tokens=T, num_q_heads=Hq, q_seq_stride=T * Hq * d, q_tok_stride=Hq * d, q_head_stride=d,
                    o_seq_stride=T * Hq * d, o_tok_stride=Hq * d, o_head_stride=d, block_table_stride=s.bt.shape[1],
                    max_seq_len=max(s.lens), **pool.geometry())
        prob = dict(geom=geom, q=s.q, kv4=pool, seq_len=_i32(s.lens), kv_len=s.kv_len.reshape(-1), block_table=s.bt,
                    out_shape=(B, T, Hq, d))
        s.dp = hip.DeviceProblem(prob)
        s.alpha_bits = int(np.float32(s.alpha).view(np.uint32))
    else:
        from exactattention_amd.serving import DraftCheck
        s.check = DraftCheck(c["B"], c["N"], c["V"])


# ---- one pass

def run(s):
    return {"append": _run_append, "turn": _run_turn, "attend": _run_attend, "verify": _run_verify}[s.case["kind"]](s)


def _angles(s):
    """(N, 1, rot / 2) cosines and sines, the angles in 64 bits."""
    ang = (s.positions.double()[:, None] * s.w)[:, None]
    return ang.cos(), ang.sin()


def _turned(x, cos, sin, rot, adjacent):
    h = rot // 2
    if adjacent:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _normed(x, w, eps):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + eps) * w


def _run_append(s):
    c = s.case
    if own:
        q = s.rotary.append(s.q, s.k, s.v, s.positions, s.dst, s.pool, norm=s.norm)
        k, v = s.pool.values()
        return {"q": q, "k": k, "v": v}
    d, P, n = c["d"], c["page"], c["N"] - c["pad"]
    cos, sin = _angles(s)
    # k in 64 bits: a value next to the border of two codes becomes one or the other
    q, k = s.q.float(), s.k.double()
    if c["norm"]:
        q, k = _normed(q, s.qw.float(), s.eps), _normed(k, s.kw.double(), s.eps)
    q = _turned(q, cos.float(), sin.float(), c["rot"], c["adjacent"])
    k = _turned(k, cos, sin, c["rot"], c["adjacent"])
    page, slot = s.dst[:n] // P, s.dst[:n] % P
    for pool, new in ((s.kp, k[:n]), (s.vp, s.v[:n].float())):
        new = _values(torch.nn.functional.pad(new, (0, _width(d) - d)))[..., :d]
        pool[page, :, slot] = new.to(pool.dtype)
    return {"q": q.to(torch.bfloat16), "k": s.kp, "v": s.vp}


def _run_turn(s):
    c = s.case
    if own:
        q, k = s.rotary.rotate(*s.leaves[:2], s.positions, norm=s.norm)
        dq, dk, dqw, dkw = torch.autograd.grad((q, k), s.leaves, (s.gq, s.gk))
        return {"q": q.detach(), "k": k.detach(), "dq": dq, "dk": dk, "dqw": dqw, "dkw": dkw}
    cos, sin = (x.float() for x in _angles(s))
    out = {}
    for name, x, w, g in (("q", s.q, s.qw, s.gq), ("k", s.k, s.kw, s.gk)):
        xf, wf = x.float(), w.float()
        r = torch.rsqrt(xf.square().mean(-1, keepdim=True) + s.eps)
        xh = xf * r
        out[name] = _turned(xh * wf, cos, sin, c["rot"], c["adjacent"]).to(x.dtype)
        gf = _turned(g.float(), cos, -sin, c["rot"], c["adjacent"])
        gw = gf * wf
        out["d" + name] = (r * (gw - xh * (gw * xh).mean(-1, keepdim=True))).to(x.dtype)
        out["d" + name + "w"] = (gf * xh).sum((0, 1)).to(w.dtype)
    return out


def _run_attend(s):
    c = s.case
    if own:
        from exactattention_amd import hip
        hip.launch_hip(s.dp, s.alpha_bits)
        return {"out": s.dp.out.view(torch.bfloat16), "flags": s.dp.flags}
    B, T, Hq, Hkv, d = (c[x] for x in ("B", "T", "Hq", "Hkv", "d"))
    at = s.bt.long()
    # (B, pages, Hkv, slots, d) to (B, Hkv, keys, d)
    k, v = (_spell(codes[at], scales[at], d).transpose(1, 2).flatten(2, 3) for codes, scales in ((s.kc, s.ks), (s.vc, s.vs)))
    q = s.q.float().view(B, T, Hkv, Hq // Hkv, d).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, d)
    t = torch.matmul(q, k.transpose(2, 3).contiguous()).mul_(s.alpha).unflatten(2, (-1, T))
    dead = torch.arange(k.shape[2], device="cuda") >= s.kv_len[..., None]
    t = t.masked_fill_(dead[:, None, None], -math.inf)
    w = torch.exp2(t - t.amax(-1, keepdim=True))
    o = torch.matmul(w.flatten(2, 3), v).unflatten(2, (-1, T)) / w.sum(-1, keepdim=True)
    out = o.permute(0, 3, 1, 2, 4).reshape(B, T, Hq, d).to(torch.bfloat16)
    return {"out": out, "flags": torch.zeros(B * T * Hq, dtype=torch.uint8, device="cuda")}


def _run_verify(s):
    if own:
        s.check.verify(s.p, s.drafted, s.u, draft_probs=s.qp, parents=s.parents, counts=s.count)
        return {"accepted": s.check.accepted, "path": s.check.path, "tokens": s.check.tokens}
    B, N = s.drafted.shape
    V = s.p.shape[-1]
    i = torch.arange(N, device="cuda")
    b = torch.arange(B, device="cuda")[:, None]
    x, u, par = s.drafted.long(), s.u.double(), s.par
    px = s.p[b, par + 1, x].double()
    there = i < s.count[:, None]
    if s.qp is not None:
        ok = u[:, :N] * s.qp[b, i, x].double() < px
        first = ok
    else:
        # tried after its siblings: the mass that they have taken, a token once
        sib = (par[:, :, None] == par[:, None, :]) & (i[:, None] > i)
        twice = (sib & (x[:, :, None] == x[:, None, :])).any(-1)
        gone = (sib * (px * ~twice)[:, None, :]).sum(-1)
        ok = ~twice & (u[:, :N] * (1.0 - gone) < px)
        first = ok & ~(sib & ok[:, None, :]).any(-1)
    stands = ~(s.anc & ~(first & there)[:, None, :]).any(-1)
    accepted = stands.sum(-1)
    order = torch.where(stands, i, N).sort(-1).values
    path = torch.where(order < N, order, -1)
    last = torch.where(stands, i, -1).amax(-1)
    p = s.p[b[:, 0], last + 1].double().clamp(0.0, 1.0)
    left = p
    if s.qp is not None:
        q = s.qp[b[:, 0], (last + 1).clamp(max=N - 1)].double().clamp(0.0, 1.0)
        left = torch.where((last + 1 < s.count)[:, None], (p - q).clamp(min=0.0), p)
    else:
        child = (par == last[:, None]) & there
        left = p.scatter(1, x, torch.where(child, torch.zeros_like(px), p.gather(1, x)))
    # in whole numbers of 2^-44, whose sums are exact
    w, w0 = (left * 2.0**44).long(), (p * 2.0**44).long()
    w = torch.where((w.sum(-1) == 0)[:, None], w0, w)
    upto = w.cumsum(-1)
    goal = (u[:, N] * upto[:, -1].double()).long()
    new = (upto <= goal[:, None]).sum(-1)
    new = torch.where(upto[:, -1] == 0, -1, new).clamp(max=V - 1)
    at = torch.arange(N + 1, device="cuda")
    tok = torch.cat([x.gather(1, path.clamp(min=0)), torch.full_like(accepted, -1)[:, None]], 1)
    tok = torch.where(at < accepted[:, None], tok, torch.where(at == accepted[:, None], new[:, None], -1))
    return {"accepted": accepted.int(), "path": path.int(), "tokens": tok.int()}


# ---- what a pass cannot do without

def work(case):
    if case["kind"] == "attend":
        T, Hq, Hkv, d = (case[x] for x in ("T", "Hq", "Hkv", "d"))
        lens = _lens(case)
        pairs = sum(T * n - T * (T - 1) // 2 for n in lens)
        rows = case["B"] * T * Hq
        return {"bytes": sum(lens) * Hkv * 2 * _width(d) * 17 // 32 + rows * d * 4, "flops": 4 * d * pairs * Hq}
    if case["kind"] == "verify":
        # a row of the target's probabilities and one of the draft's for each sequence
        rows = case["B"] * (2 if case["op"] == "chain" else 1)
        return {"bytes": rows * case["V"] * 4 + case["B"] * case["N"] * 24, "flops": 4 * rows * case["V"]}
    sz = 4 if case["dtype"] == "fp32" else 2
    N, Hq, Hkv, d = (case[x] for x in ("N", "Hq", "Hkv", "d"))
    if case["kind"] == "turn":  # x and dy read, y and dx written
        return {"bytes": N * d * (Hq + Hkv) * 4 * sz + 4 * N, "flops": 30 * N * (Hq + Hkv) * d}
    # q, k and v read, q written, the rows' codes, and the cache's values that are returned
    rows = (N + case["page"] - 1) // case["page"] * case["page"] + 3 * case["page"]
    by = N * d * (Hq * (sz + 2) + 2 * Hkv * sz) + 2 * N * Hkv * _width(d) * 17 // 32 + 2 * rows * Hkv * (_width(d) * 17 // 32 + 2 * d)
    return {"bytes": by + 12 * N, "flops": 12 * N * (Hq + 2 * Hkv) * d}


# ---- the same outputs from the definitions in 64 bits

def exact(case, seed):
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    if case["kind"] == "append":
        return _exact_append(case, seed)
    if case["kind"] == "turn":
        return _exact_turn(case, seed)
    return None  # whole numbers


def _levels(device):
    """All that a code can stand for, in order, and the borders between neighbours."""
    a = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=device)
    return a, (a[1:] + a[:-1]) / 2


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    T, Hq, Hkv, d, P = (case[x] for x in ("T", "Hq", "Hkv", "d", "page"))
    lv, _ = _levels("cuda")
    lv = torch.cat([lv, -lv])
    out = torch.zeros((case["B"], T, Hq, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s.lens):
        keys = torch.arange(n, device="cuda")
        page, slot = s.bt[b].long()[keys // P], keys % P
        for g in range(Hkv):
            kv = []
            for codes, scales in ((s.kc, s.ks), (s.vc, s.vs)):
                c = codes[page, g, slot]
                x = torch.empty((n, 2 * c.shape[1]), dtype=torch.float64, device="cuda")
                x[:, 0::2], x[:, 1::2] = lv[(c & 15).long()], lv[(c >> 4).long()]
                kv.append((x.view(n, -1, 32) * 2.0 ** (scales[page, g, slot].double() - 127)[..., None]).view(n, -1)[:, :d])
            for h in range(g * (Hq // Hkv), (g + 1) * (Hq // Hkv)):
                x = s.alpha * math.log(2.0) * (s.q[b, :, h].double() @ kv[0].t().contiguous())
                x[keys[None] >= s.kv_len[b][:, None]] = -math.inf
                out[b, :, h] = torch.softmax(x, -1) @ kv[1]
    return {"out": out, "flags": None}


def _phases(case, s, sign=1.0):
    ang = s.positions.double()[:, None] * torch.from_numpy(s.inv_freq).cuda()
    return torch.polar(torch.ones_like(ang), sign * ang)[:, None]


def _exact_turned(case, x, z):
    rot, h = case["rot"], case["rot"] // 2
    first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["adjacent"] else (slice(0, h), slice(h, rot))
    y = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
    x = x.clone()
    x[..., first], x[..., second] = y.real, y.imag
    return x


def _exact_append(case, seed):
    s = _append_inputs(case, seed)
    z = _phases(case, s)
    d, P, Hkv = case["d"], case["page"], case["Hkv"]
    x = {}
    for name, t, w in (("q", s.q, s.qw), ("k", s.k, s.kw)):
        t = t.double()
        if case["norm"]:
            t = t / torch.sqrt((t * t).sum(-1, keepdim=True) / d + s.eps) * w.double()
        x[name] = _exact_turned(case, t, z)
    lv, border = _levels("cuda")
    put = s.dst >= 0
    page, slot = s.dst[put] // P, s.dst[put] % P
    out = {"q": x["q"]}
    for name, new, at in (("k", x["k"], 0), ("v", s.v.double(), 2)):
        pool = _spell(s.pools[at], s.pools[at + 1], d).double()
        new = torch.nn.functional.pad(new[put], (0, _width(d) - d)).view(int(put.sum()), Hkv, -1, 32)
        top = new.abs().amax(-1, keepdim=True)
        step = 2.0 ** torch.floor(torch.log2(top.clamp(min=2.0**-140) / 7.0) + 1.0)
        step = torch.where(top >= 7.0 * step, 2 * step, torch.where(top < 3.5 * step, step / 2, step)).clamp(2.0**-125, 2.0**125)
        y = new.abs() / step
        # the nearest level; on a border the even one
        n = torch.bucketize(y, border)
        on = (n < 7) & (y == border[n.clamp(max=6)])
        n = torch.where(on & (n % 2 == 1), n + 1, n)
        pool[page, :, slot] = (lv[n] * step * torch.sign(new)).flatten(-2)[..., :d]
        out[name] = pool
    return out


def _exact_turn(case, seed):
    s = _qkv(case, seed, True)[0]
    z, back = _phases(case, s), _phases(case, s, -1.0)
    d, out = case["d"], {}
    for name, x, w, g in (("q", s.q, s.qw, s.gq), ("k", s.k, s.kw, s.gk)):
        x, w, g = x.double(), w.double(), _exact_turned(case, g.double(), back)
        n = torch.sqrt((x * x).sum(-1, keepdim=True) / d + s.eps)
        out[name] = _exact_turned(case, x / n * w, z)
        out["d" + name] = g * w / n - x * (g * w * x).sum(-1, keepdim=True) / (d * n**3)
        out["d" + name + "w"] = (g * x / n).flatten(0, 1).sum(0)
    return out

"""The operators of a serving step around the certified attention, as cases that can be timed.

A step of a serving loop runs three of them in turn, each of which is measured by itself:

  plan    where the step's tokens go: block-table growth from the stack of free pages, the slot of
          each new token, its position and its visible length, from the requests' lengths
  rotary  q and k rotated by positions of one or several axes (time, height, width), k and v
          written into the paged cache on the way ("append"), or the rotation and its inverse (the
          gradient) by themselves ("rotate")
  attend  attention over the cache with interval masks (sliding windows, packed documents, a prefix
          that all tokens see), a bias that falls with the distance, or scores capped by a tanh

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

# attend: B sequences of kv_min..kv keys in the cache (spread over the logarithm by `lens`), T query
# tokens at the end of each; window: keys a token sees at most (0: all before it); docs: mean length
# of the documents packed in a sequence (0: one); prefix: leading tokens that every token sees;
# alibi: distance bias with the usual geometric slopes; cap: bound of the scores (0: none);
# qscale: scale of the queries (large scores meet the cap)
_ATTEND = dict(kind="attend", T=1, d=128, page=16, out="bf16", lens=0, window=0, docs=0, prefix=0, alibi=False, cap=0.0,
               qscale=1.0)
# rotary: N tokens, `pad` of them padding without a slot; rot rotated dims of d; axes position axes
# (interleaved: neighbouring pairs take different axes); adjacent: pairs (2i, 2i+1), else (i, i + rot/2)
_ROTARY = dict(kind="rotary", op="append", d=128, rot=128, axes=1, interleaved=False, adjacent=False, page=16, dtype="bf16",
               pad=0, inverse=False, maxpos=8192)
# plan: B sequences of up to kv keys that take 1..tok new tokens each, room for `pad` more than that
_PLAN = dict(kind="plan", page=16, pad=0, lens=0)


def _case(base, name, **kw):
    c = dict(base, **kw)
    if base is _ATTEND:
        c.setdefault("kv_min", c["kv"])
    if name:
        c["name"] = name
    return c


def listed():
    return [
        # one token of a chat turn on a model with distance bias: latency
        _case(_ATTEND, "attend_decode_alibi_900", B=1, kv=900, Hq=16, Hkv=8, alibi=True),
        # a running batch's decode, capped scores, wide GQA
        _case(_ATTEND, "attend_decode_cap_ragged", B=32, kv=4096, kv_min=512, lens=3, Hq=32, Hkv=8, cap=30.0, qscale=3.0),
        # sliding-window decode far into long contexts: only the window's keys are read
        _case(_ATTEND, "attend_decode_window_long", B=8, kv=131072, kv_min=30000, lens=5, Hq=16, Hkv=8, window=4096, page=64),
        # a prompt of packed documents, each token sees its own document
        _case(_ATTEND, "attend_documents_4096", B=1, T=4096, kv=4096, Hq=16, Hkv=8, page=0, docs=600),
        # a prompt with capped scores: the whole causal triangle
        _case(_ATTEND, "attend_prefill_cap_2500", B=1, T=2500, kv=2500, Hq=16, Hkv=8, cap=50.0, qscale=3.0),
        # a prompt whose first part all tokens see, distance bias, 64-dim heads
        _case(_ATTEND, "attend_prefix_alibi_d64", B=2, T=777, kv=777, Hq=16, Hkv=4, d=64, prefix=300, alibi=True),
        # the new tokens of a decode step
        _case(_ROTARY, "rotary_append_33", N=33, Hq=32, Hkv=8),
        # prompt chunks of a vision model: three axes, the last tokens are padding
        _case(_ROTARY, "rotary_append_axes_16k", N=16384, Hq=32, Hkv=8, axes=3, page=64, pad=5),
        # the rotation's gradient in fp32 on part of each head
        _case(_ROTARY, "rotary_inverse_2001", op="rotate", N=2001, Hq=12, Hkv=4, d=96, rot=64, dtype="fp32", inverse=True),
        # a decode step's plan
        _case(_PLAN, "plan_decode_33", B=33, kv=6000, tok=1),
        # a mixed step: prompt chunks among decoding requests
        _case(_PLAN, "plan_mixed_256", B=256, kv=9000, tok=300, pad=100, lens=7),
        # the largest step a scheduler hands out
        _case(_PLAN, "plan_large_1000", B=1000, kv=32000, tok=500, lens=2, page=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A case of the listed ranges: no more pairs, keys or tokens than the largest listed."""
    kind = rng.choice(["attend", "attend", "attend", "rotary", "rotary", "plan"])
    Hkv = rng.choice([1, 2, 4, 8])
    grp = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 16, 32, 64])
    if kind == "attend":
        d = rng.choice([128, 128, 64, 96, 80])
        out = rng.choice(["bf16", "bf16", "bf16", "fp32"])
        lens = rng.randrange(1 << 20)
        mod = rng.choice([dict(alibi=True), dict(cap=rng.choice([20.0, 30.0, 50.0]), qscale=rng.choice([1.0, 3.0])), dict(),
                          dict(alibi=True, cap=30.0, qscale=2.0)])
        what = rng.choice(["decode", "window", "verify", "docs", "prefix", "prefill"])
        if what in ("decode", "window"):
            B = _log(rng, 1, 32)
            kv = _log(rng, 1, min(131072, 400_000 // B) if what == "window" else min(32768, 90_000 // B))
            win = _log(rng, 1, 8192) if what == "window" else 0
            return _case(_ATTEND, None, B=B, kv=kv, kv_min=rng.choice([kv, max(1, kv // 8)]), lens=lens, Hq=Hkv * grp,
                         Hkv=Hkv, d=d, page=rng.choice([0, page]), out=out, window=win, **mod)
        if what == "verify":
            T, B = _log(rng, 2, 40), _log(rng, 1, 8)
            kv = _log(rng, T, max(T, 60_000 // (B * grp)))
            return _case(_ATTEND, None, B=B, T=T, kv=kv, kv_min=rng.choice([kv, max(T, kv // 4)]), lens=lens, Hq=Hkv * grp,
                         Hkv=Hkv, d=d, page=page, out=out, window=rng.choice([0, _log(rng, 1, 5000)]), **mod)
        lim = 2500 * 2500 * 16  # pairs over the heads
        T = min(_log(rng, 2, 3000), int(math.sqrt(lim / (Hkv * grp))))
        kv = T if what != "prefill" else min(T + rng.choice([0, _log(rng, 1, 4000)]), max(T, lim // (T * Hkv * grp)))
        extra = dict(docs=_log(rng, 5, 1500)) if what == "docs" else dict(prefix=_log(rng, 1, T)) if what == "prefix" else {}
        return _case(_ATTEND, None, B=1, T=T, kv=kv, Hq=Hkv * grp, Hkv=Hkv, d=d, page=rng.choice([0, page]), out=out,
                     window=_log(rng, 1, 2000) if what == "prefill" and rng.random() < 0.5 else 0, **extra, **mod)
    if kind == "rotary":
        d = rng.choice([128, 128, 64, 96, 80])
        op = rng.choice(["append", "append", "rotate"])
        dtype = rng.choice(["bf16", "bf16", "fp32"])
        # no more elements than the largest listed, at 4 bytes a third fewer
        most = 16384 * 48 * 128 // (Hkv * (grp + 2) * d)
        N = _log(rng, 1, min(16384, most if dtype == "bf16" else most * 2 // 3))
        return _case(_ROTARY, None, op=op, N=N, Hq=Hkv * grp, Hkv=Hkv, d=d, rot=rng.choice([d, d, d // 2]),
                     axes=rng.choice([1, 1, 2, 3, 4]), interleaved=rng.random() < 0.5, adjacent=rng.random() < 0.5, page=page,
                     dtype=dtype, pad=rng.choice([0, 0, min(N, 7)]),
                     inverse=op == "rotate" and rng.random() < 0.5, maxpos=rng.choice([4096, 131072, 1 << 20]))
    B = _log(rng, 1, 1000)
    tok = rng.choice([1, rng.randint(2, 16), _log(rng, 2, 500)])
    return _case(_PLAN, None, B=B, kv=_log(rng, 1, 32000), tok=tok, page=rng.choice([1, 16, 64]), pad=rng.choice([0, 50]),
                 lens=rng.randrange(1 << 20))


# ---- what a case holds

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(shape, gen, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda").normal_(generator=gen)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a, dtype=np.int32)).cuda()


def _lens(case):
    """Keys in the cache of each sequence, the query tokens' own among them."""
    lo, hi = max(case["kv_min"], case["T"]), case["kv"]
    r = random.Random(case["lens"])
    return [hi] + [_log(r, lo, hi) for _ in range(case["B"] - 1)]


def _intervals(case, r=None):
    """(begin, end, position) of each query token's visible keys, (B, T) int64 arrays."""
    T, lens = case["T"], np.asarray(_lens(case), np.int64)
    pos = lens[:, None] - T + np.arange(T)
    end, begin = pos + 1, np.zeros_like(pos)
    if case["prefix"]:
        end = np.maximum(end, np.minimum(case["prefix"], lens[:, None]))
    if case["window"]:
        begin = np.maximum(begin, end - case["window"])
    if case["docs"]:
        # documents of 1 .. 2 * mean tokens; the last few tokens are padding that sees nothing
        r = random.Random(case["lens"] + 17)
        at, starts = 0, np.zeros(T, np.int64)
        while at < T:
            n = r.randint(1, 2 * case["docs"])
            starts[at:at + n] = at
            at += n
        begin = np.broadcast_to(starts, pos.shape).copy()
        npad = min(T // 4, 3)
        if npad:
            begin[:, T - npad:] = end[:, T - npad:]
    return begin, end, pos


def _attend_inputs(case, seed):
    gen, r = _gen(seed), np.random.default_rng(seed)
    B, T, Hq, Hkv, d, P = (case[x] for x in ("B", "T", "Hq", "Hkv", "d", "page"))
    lens = _lens(case)
    s = SimpleNamespace(lens=lens)
    s.q = _normal((B, T, Hq, d), gen)
    if case["qscale"] != 1.0:
        s.q *= case["qscale"]
    S = max(lens)
    if P:
        need = [-(-n // P) for n in lens]
        perm = r.permutation(sum(need)).astype(np.int32)
        bt, at = np.zeros((B, max(need)), np.int32), 0
        for b, n in enumerate(need):
            bt[b, :n] = perm[at:at + n]
            at += n
        s.bt = _i32(bt)
        s.k, s.v = _normal((sum(need), P, Hkv, d), gen), _normal((sum(need), P, Hkv, d), gen)
    else:
        s.bt = None
        s.k, s.v = _normal((B, Hkv, S, d), gen), _normal((B, Hkv, S, d), gen)
    begin, end, pos = _intervals(case)
    s.kv_begin = _i32(begin) if case["docs"] else None
    s.begin, s.end, s.pos = _i32(begin), _i32(end), _i32(pos)
    s.slopes = None
    if case["alibi"]:
        s.slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / Hq) * LOG2E for h in range(Hq)], dtype=torch.float32, device="cuda")
    s.cap = float(np.float32(case["cap"] * LOG2E))  # in base-2 logits, as alpha
    s.alpha = float(np.float32(d ** -0.5 * LOG2E))
    return s


def _axis_of_pair(case):
    """The position axis of each rotated pair: sections of about a quarter for the first axis and
    equal parts of the rest, one after another or dealt in turn."""
    half, A = case["rot"] // 2, case["axes"]
    if A == 1:
        return [0] * half
    first = half // 4
    sec = [first] + [(half - first) // (A - 1)] * (A - 1)
    sec[-1] += half - sum(sec)
    if not case["interleaved"]:
        return [a for a in range(A) for _ in range(sec[a])]
    out, left, a = [], list(sec), 0
    while len(out) < half:
        if left[a]:
            out.append(a)
            left[a] -= 1
        a = (a + 1) % A
    return out


def _rotary_inputs(case, seed):
    gen, r = _gen(seed), np.random.default_rng(seed)
    N, Hq, Hkv, d = (case[x] for x in ("N", "Hq", "Hkv", "d"))
    dt = torch.float32 if case["dtype"] == "fp32" else torch.bfloat16
    s = SimpleNamespace()
    # q, k and v as a projection leaves them: parts of one row per token
    qkv = _normal((N, (Hq + 2 * Hkv) * d), gen, dt)
    s.q = qkv[:, :Hq * d].view(N, Hq, d)
    s.k = qkv[:, Hq * d:(Hq + Hkv) * d].view(N, Hkv, d)
    s.v = qkv[:, (Hq + Hkv) * d:].view(N, Hkv, d)
    pos = r.integers(0, case["maxpos"], (case["axes"], N))
    s.positions = _i32(pos)
    half = case["rot"] // 2
    s.inv_freq = 10000.0 ** (-np.arange(half, dtype=np.float64) / half)
    s.axis = _axis_of_pair(case)
    if case["op"] == "append":
        P = case["page"]
        rows = (N + P - 1) // P * P + 3 * P
        dst = r.permutation(rows)[:N].astype(np.int64)
        if case["pad"]:
            dst[N - case["pad"]:] = -1
        s.dst = torch.from_numpy(dst).cuda()
        s.kp, s.vp = (_normal((rows // P, P, Hkv, d), gen) for _ in range(2))
    return s


def _counts(case):
    """New tokens of the step's requests, in some order: most requests decode, the others bring
    chunks, and some have nothing this step."""
    r = np.random.default_rng(case["lens"])
    B, tok = case["B"], case["tok"]
    if tok == 1:
        return np.ones(B, np.int64)
    c = np.where(r.random(B) < 0.5, 1, r.integers(1, tok + 1, B))
    c[r.random(B) < 0.05] = 0
    return c


def _plan_inputs(case, seed):
    r = np.random.default_rng(seed)
    B, P = case["B"], case["page"]
    s = SimpleNamespace(B=B, P=P)
    L = np.exp(r.uniform(0.0, math.log(case["kv"] + 1), B)).astype(np.int64) - 1
    c = r.permutation(_counts(case))
    s.T = case["tok"]
    s.W = int((case["kv"] + case["tok"] + P - 1) // P) + 1
    held = -(-L // P)
    need = -(-(L + c) // P) - held
    S = B + 5  # slots of the cache, some of them not in the step
    pages = int(held.sum() + need.sum()) + 20
    perm = r.permutation(pages).astype(np.int32)
    slots = r.permutation(S)[:B].astype(np.int32)
    bt = np.zeros((S, s.W), np.int32)
    at = 0
    for b in range(B):
        bt[slots[b], :held[b]] = perm[at:at + held[b]]
        at += held[b]
    free = perm[at:]
    s.N = max(int(c.sum()) + case["pad"], 1)
    s.seq_len, s.counts, s.slots, s.bt, s.free = _i32(L), _i32(c), _i32(slots), _i32(bt), _i32(free)
    s.num_free = _i32([len(free)])
    return s


def prepare(case, seed):
    s = {"attend": _attend_inputs, "rotary": _rotary_inputs, "plan": _plan_inputs}[case["kind"]](case, seed)
    s.case = case
    if not own:
        if case["kind"] == "rotary":
            s.w = torch.from_numpy(s.inv_freq).cuda()
            s.axis_t = torch.tensor(s.axis, device="cuda")
        return s
    if case["kind"] == "attend":
        from exactattention_amd import hip
        B, T, Hq, Hkv, d, P = (case[x] for x in ("B", "T", "Hq", "Hkv", "d", "page"))
        S = max(s.lens)
        ks = (P * Hkv * d, Hkv * d, d) if P else (Hkv * S * d, d, S * d)
        geom = dict(num_seqs=B, num_tokens=T, num_q_heads=Hq, num_kv_heads=Hkv, head_dim=d, head_dim_v=d,
                    q_seq_stride=T * Hq * d, q_tok_stride=Hq * d, q_head_stride=d, o_seq_stride=T * Hq * d,
                    o_tok_stride=Hq * d, o_head_stride=d, k_page_stride=ks[0], k_slot_stride=ks[1], k_head_stride=ks[2],
                    v_page_stride=ks[0], v_slot_stride=ks[1], v_head_stride=ks[2], page_size=P or 1,
                    block_table_stride=s.bt.shape[1] if P else 0, max_seq_len=S)
        mods = hip.ScoreMods(kv_begin=s.kv_begin, window=case["window"], slopes=s.slopes,
                             q_pos=s.pos if case["alibi"] else None, softcap=s.cap)
        prob = dict(geom=geom, q=s.q, k=s.k, v=s.v, seq_len=_i32(s.lens), kv_len=s.end.reshape(-1), block_table=s.bt,
                    out_shape=(B, T, Hq, d))
        s.dp = hip.DeviceProblem(prob, case["out"], mods=mods)
        s.alpha_bits = int(np.float32(s.alpha).view(np.uint32))
    elif case["kind"] == "rotary":
        from exactattention_amd.serving import Rotary
        s.rotary = Rotary(case["d"], rot_dim=case["rot"], inv_freq=s.inv_freq, axis_of_pair=s.axis, adjacent=case["adjacent"])
    else:
        from exactattention_amd.serving import StepPlan
        s.plan = StepPlan(s.B, s.N, s.T)
    return s


# ---- one pass

def run(s):
    kind = s.case["kind"]
    if kind == "attend":
        return _run_attend(s)
    if kind == "rotary":
        return _run_rotary(s)
    return _run_plan(s)


def _run_attend(s):
    c = s.case
    if own:
        from exactattention_amd import hip
        hip.launch_hip(s.dp, s.alpha_bits)
        return {"out": s.dp.out.view(torch.float32 if s.dp.out_fp32 else torch.bfloat16), "flags": s.dp.flags}
    B, T, Hq, Hkv, d, P = (c[x] for x in ("B", "T", "Hq", "Hkv", "d", "page"))
    grp = Hq // Hkv
    out = torch.empty((B, T, Hq, d), dtype=torch.float32 if c["out"] == "fp32" else torch.bfloat16, device="cuda")
    for b, n in enumerate(s.lens):
        # the keys that some token of the sequence sees
        n0 = max(0, n - T + 1 - c["window"]) if c["window"] else 0
        if P:
            n0 = n0 // P * P
            idx = s.bt[b, n0 // P:-(-n // P)].long()
            k, v = (x[idx].reshape(-1, Hkv, d)[:n - n0].transpose(0, 1).float().contiguous() for x in (s.k, s.v))
        else:
            k, v = (x[b, :, n0:n].float() for x in (s.k, s.v))
        q = s.q[b].float().view(T, Hkv, grp, d).permute(1, 2, 0, 3).reshape(Hkv, grp * T, d)
        t = torch.matmul(q, k.transpose(1, 2).contiguous()).mul_(s.alpha).view(Hkv, grp, T, n - n0)
        if s.cap:
            t = t.div_(s.cap).tanh_().mul_(s.cap)
        key = torch.arange(n0, n, device="cuda")
        if s.slopes is not None:
            dist = (key[None, :] - s.pos[b][:, None]).abs().float()
            t = t.sub_(s.slopes.view(Hkv, grp, 1, 1) * dist)
        vis = (key[None, :] >= s.begin[b][:, None]) & (key[None, :] < s.end[b][:, None])
        t = t.masked_fill_(~vis, -math.inf)
        m = t.amax(-1, keepdim=True)
        w = torch.exp2(t.sub_(torch.where(m == -math.inf, torch.zeros_like(m), m)))
        z = w.sum(-1, keepdim=True)
        o = torch.matmul(w.view(Hkv, grp * T, n - n0), v).view(Hkv, grp, T, d) / torch.where(z == 0, torch.ones_like(z), z)
        out[b] = o.permute(2, 0, 1, 3).reshape(T, Hq, d).to(out.dtype)
    return {"out": out, "flags": torch.zeros(B * T * Hq, dtype=torch.uint8, device="cuda")}


def _rotate(x, cos, sin, rot, adjacent):
    """x (N, H, d) float; cos, sin (N, 1, rot / 2)."""
    h = rot // 2
    if adjacent:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        y = torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)
    else:
        a, b = x[..., :h], x[..., h:rot]
        y = torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
    return torch.cat([y, x[..., rot:]], -1)


def _run_rotary(s):
    c = s.case
    if own:
        if c["op"] == "append":
            q = s.rotary.append(s.q, s.k, s.v, s.positions, s.dst, s.kp, s.vp)
            return {"q": q, "k": s.kp, "v": s.vp}
        q, k = s.rotary.rotate(s.q, s.k, s.positions, inverse=c["inverse"])
        return {"q": q, "k": k}
    ang = s.positions.double()[s.axis_t].t() * s.w  # far positions: the angle in 64 bits
    cos, sin = ang.cos().float()[:, None], ang.sin().float()[:, None]
    if c["inverse"]:
        sin = -sin
    q, k = (_rotate(x.float(), cos, sin, c["rot"], c["adjacent"]) for x in (s.q, s.k))
    if c["op"] == "rotate":
        return {"q": q.to(s.q.dtype), "k": k.to(s.k.dtype)}
    n = c["N"] - c["pad"]  # the tokens with a slot
    for pool, new in ((s.kp, k), (s.vp, s.v)):
        pool.view(-1, c["Hkv"], c["d"]).index_copy_(0, s.dst[:n], new[:n].to(pool.dtype))
    return {"q": q.to(torch.bfloat16), "k": s.kp, "v": s.vp}


def _run_plan(s):
    if own:
        p = s.plan
        p.build(s.seq_len, s.counts, s.bt, s.free, s.num_free, s.P, slots=s.slots)
        return {"dst": p.dst_rows, "positions": p.positions, "seq": p.seq_of, "q_rows": p.q_rows, "kv_len": p.kv_len,
                "seq_len": p.seq_len, "num_free": p.num_free, "block_table": s.bt, "status": p.status}
    L, cnt, slots = s.seq_len.long(), s.counts.long(), s.slots.long()
    P, T, N, W = s.P, s.T, s.N, s.W
    held = (L + P - 1) // P
    need = (L + cnt + P - 1) // P - held
    cu, npg = cnt.cumsum(0), need.cumsum(0)
    total, news = cu[-1], npg[-1]
    cu0, np0 = cu - cnt, npg - need
    # the new pages, top of the free stack first
    i = torch.arange(s.free.numel(), device="cuda")
    ok = i < news
    b = torch.searchsorted(npg, i, right=True).clamp_(max=s.B - 1)
    at = torch.where(ok, slots[b] * W + held[b] + i - np0[b], s.bt.numel())
    page = s.free[(s.num_free.long() - 1 - i).clamp_(min=0)]
    flat = torch.cat([s.bt.view(-1), s.bt.new_zeros(1)])
    flat[at] = page
    s.bt.view(-1).copy_(flat[:-1])
    # the new tokens
    i = torch.arange(N, device="cuda")
    ok = i < total
    b = torch.searchsorted(cu, i, right=True).clamp_(max=s.B - 1)
    j = i - cu0[b]
    pos = L[b] + j
    dst = s.bt[slots[b], (pos // P).clamp(max=W - 1)].long() * P + pos % P
    none = torch.full_like(i, -1)
    jt = torch.arange(T, device="cuda")[None, :]
    kv_len = torch.where(jt < cnt[:, None], L[:, None] + jt + 1, 0)
    return {"dst": torch.where(ok, dst, none), "positions": torch.where(ok, pos, none).int(),
            "seq": torch.where(ok, b, none).int(), "q_rows": torch.where(ok, b * T + j, none), "kv_len": kv_len.int(),
            "seq_len": (L + cnt).int(), "num_free": (s.num_free - news).int(), "block_table": s.bt,
            "status": torch.zeros(1, dtype=torch.int32, device="cuda")}


# ---- what a pass cannot do without

def work(case):
    if case["kind"] == "attend":
        begin, end, _ = _intervals(case)
        pairs = int(np.maximum(end - begin, 0).sum())
        live = end > begin
        keys = 0
        for b in range(case["B"]):
            if live[b].any():
                # the keys that some token sees: intervals in order of their begin
                e = 0
                o = np.argsort(begin[b], kind="stable")
                for x, y in zip(begin[b][o].tolist(), end[b][o].tolist()):
                    if y > x:
                        keys += max(0, y - max(x, e))
                        e = max(e, y)
        osz = 4 if case["out"] == "fp32" else 2
        rows = case["B"] * case["T"] * case["Hq"]
        d = case["d"]
        return {"bytes": keys * case["Hkv"] * 4 * d + rows * d * (2 + osz), "flops": 4 * d * pairs * case["Hq"]}
    if case["kind"] == "rotary":
        sz = 4 if case["dtype"] == "fp32" else 2
        N, Hq, Hkv, d = (case[x] for x in ("N", "Hq", "Hkv", "d"))
        if case["op"] == "append":
            by = N * d * (Hq * (sz + 2) + 2 * Hkv * (sz + 2)) + 8 * N
        else:
            by = N * d * (Hq + Hkv) * 2 * sz
        return {"bytes": by + 4 * N * case["axes"], "flops": 3 * N * (Hq + Hkv) * case["rot"]}
    # lengths, counts and slots; a slot, a row, a position and a sequence per token; padded lengths; pages
    B, n = case["B"], int(_counts(case).sum())
    return {"bytes": B * 20 + (n + case["pad"]) * 24 + B * case["tok"] * 4 + n // case["page"] * 8, "flops": 20 * n}


# ---- the same outputs from the definitions in 64 bits

def exact(case, seed):
    if case["kind"] == "attend":
        return _exact_attend(case, seed)
    if case["kind"] == "rotary":
        return _exact_rotary(case, seed)
    return None  # whole numbers


def _exact_attend(case, seed):
    s = _attend_inputs(case, seed)
    T, Hq, Hkv, d, P = (case[x] for x in ("T", "Hq", "Hkv", "d", "page"))
    begin, end, pos = _intervals(case)
    out = torch.zeros((case["B"], T, Hq, d), dtype=torch.float64, device="cuda")
    for b, n in enumerate(s.lens):
        lo = int(begin[b].min())
        keys = torch.arange(lo, n, device="cuda")
        bb, ee, pp = (torch.from_numpy(x[b]).cuda() for x in (begin, end, pos))
        for h in range(Hq):
            g = h // (Hq // Hkv)
            if P:
                page, slot = s.bt[b].long()[keys // P], keys % P
                kh, vh = s.k[page, slot, g].double(), s.v[page, slot, g].double()
            else:
                kh, vh = s.k[b, g, lo:n].double(), s.v[b, g, lo:n].double()
            step = max(1, 32_000_000 // max(1, n - lo))
            for t0 in range(0, T, step):
                t1 = min(T, t0 + step)
                x = s.alpha * (s.q[b, t0:t1, h].double() @ kh.t().contiguous())
                if case["cap"]:
                    x = s.cap * torch.tanh(x / s.cap)
                if s.slopes is not None:
                    x = x - s.slopes[h].double() * (keys[None] - pp[t0:t1, None]).abs().double()
                dead = (keys[None] < bb[t0:t1, None]) | (keys[None] >= ee[t0:t1, None])
                live = (ee > bb)[t0:t1]
                x[dead] = -math.inf
                w = torch.softmax(x[live] * math.log(2.0), -1)
                out[b, t0:t1, h][live] = w @ vh
    return {"out": out, "flags": None}


def _exact_rotary(case, seed):
    s = _rotary_inputs(case, seed)
    rot, h = case["rot"], case["rot"] // 2
    ang = torch.stack([s.positions[a].double() * float(f) for a, f in zip(s.axis, s.inv_freq)], 1)
    z = torch.polar(torch.ones_like(ang), -ang if case["inverse"] else ang)[:, None]

    def turn(x):
        x = x.double()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["adjacent"] else (slice(0, h), slice(h, rot))
        y = torch.complex(x[..., first].contiguous(), x[..., second].contiguous()) * z
        x = x.clone()
        x[..., first], x[..., second] = y.real, y.imag
        return x

    q, k = turn(s.q), turn(s.k)
    if case["op"] == "rotate":
        return {"q": q, "k": k}
    kp, vp = s.kp.double(), s.vp.double()
    put = s.dst >= 0
    kp.view(-1, case["Hkv"], case["d"])[s.dst[put]] = k[put]
    vp.view(-1, case["Hkv"], case["d"])[s.dst[put]] = s.v.double()[put]
    return {"q": q, "k": kp, "v": vp}

"""Oracle of the score modifications (test infrastructure): the definition over Python integers, built on
the CPU oracle's exact logits and weights. The cap's fixed sequence of fp64 operations is restated with
the C library's fma; its exponential table is computed here, in decimal arithmetic."""

from __future__ import annotations

import ctypes
import ctypes.util
import math
from decimal import Decimal, getcontext
from functools import lru_cache

import numpy as np

from oracle import exact, oracle

_libm = ctypes.CDLL(ctypes.util.find_library("m") or "libm.so.6")
_libm.fma.argtypes = [ctypes.c_double] * 3
_libm.fma.restype = ctypes.c_double
fma = _libm.fma
getcontext().prec = 60

LN2 = Decimal(2).ln()


@lru_cache(None)
def _table():
    return [float(Decimal(2) ** (Decimal(j) / 256)) for j in range(256)]


_POLY = [float((-LN2 / 256) ** k / math.factorial(k)) for k in (4, 3, 2, 1)]


def cap32(t: float, c: float) -> float:
    """RN32(c tanh(t / c)) as ea_mod.h computes it; t and c fp32 values."""
    if not c:
        return t
    y = min(abs(t) * (float(512 / LN2) / c), 16384.0)
    i = math.floor(y)
    r = y - i
    p = _POLY[0]
    for q in _POLY[1:]:
        p = fma(r, p, q)
    p = r * p
    s = math.ldexp(_table()[-i & 255], -i >> 8)
    g = fma(s, p, s - 1.0)
    return math.copysign(float(np.float32(c * (-g / (2.0 + g)))), t)


def tanh_exact(t: float, c: float) -> Decimal:
    x = Decimal(t) / Decimal(c) * 2
    e = (-abs(x)).exp()
    return (Decimal(c) * (1 - e) / (1 + e)).copy_sign(Decimal(t))


def bias32(t: float, m: float, dist: int) -> float:
    """RN32(t - m RN32(|dist|)), one rounding."""
    d = float(np.float32(abs(dist)))
    (tm, te), (mm, me), (dm, de) = (exact.decode_fp32_bits(exact.fp32_bits(x)) for x in (t, m, d))
    pm, pe = -mm * dm, me + de
    e = min(te, pe)
    num = (tm << (te - e)) + (pm << (pe - e))
    q, qe = exact.round_dyadic(num, e, exact.FP32)
    return math.ldexp(q, qe)


def keys_of(tok: int, b: int, prob: dict, begin, window: int):
    """The visible keys of token `tok` of sequence b, in order."""
    sl = int(np.asarray(prob["seq_len"])[b])
    kvl = int(np.asarray(prob["kv_len"]).reshape(-1)[tok])
    lo = max(0, 0 if begin is None else int(np.asarray(begin).reshape(-1)[tok]))
    if window:
        lo = max(lo, kvl - window)
    keys = set(range(lo, min(kvl, sl)))
    if prob.get("tree_mask") is not None:
        m, tb = int(prob["tree_mask"][tok]), int(prob["tree_base"][b])
        keys |= {tb + i for i in range(64) if m >> i & 1 and tb + i < sl}
    return sorted(keys)


def row(prob: dict, alpha_bits: int, r: int, out="bf16", begin=None, window=0, slopes=None, q_pos=None, cap=0.0):
    """Output bits of row r (uint16 or uint32 array)."""
    gm = prob["geom"]
    T, Hq, Hkv, d, dv = (gm[x] for x in ("num_tokens", "num_q_heads", "num_kv_heads", "head_dim", "head_dim_v"))
    b, t, h = r // (T * Hq), (r // Hq) % T, r % Hq
    tok, hk = b * T + t, h // (Hq // Hkv)
    kvl = int(np.asarray(prob["kv_len"]).reshape(-1)[tok])
    p = kvl - 1 if q_pos is None else int(np.asarray(q_pos).reshape(-1)[tok])
    m = 0.0 if slopes is None else float(np.float32(slopes[h]))
    c = float(np.float32(cap))
    flat = {x: np.asarray(prob[x]).reshape(-1) for x in ("q", "k", "v")}

    def addr(n, x):
        page, slot = b, n
        if prob.get("block_table") is not None:
            page = int(np.asarray(prob["block_table"]).reshape(-1)[b * gm["block_table_stride"] + n // gm["page_size"]])
            slot = n % gm["page_size"]
        return page * gm[x + "_page_stride"] + slot * gm[x + "_slot_stride"] + hk * gm[x + "_head_stride"]

    q0 = b * gm["q_seq_stride"] + t * gm["q_tok_stride"] + h * gm["q_head_stride"]
    q = flat["q"][q0:q0 + d]
    fmt, enc = (exact.BF16, exact.encode_bf16) if out == "bf16" else (exact.FP32, exact.encode_fp32)
    res = np.zeros(dv, np.uint16 if out == "bf16" else np.uint32)
    keys = keys_of(tok, b, prob, begin, window)
    if not keys:
        return res
    W, V = [], []
    for n in keys:
        tb = oracle.logit_bits(q, flat["k"][addr(n, "k"):addr(n, "k") + d], alpha_bits)
        assert tb is not None
        t1 = cap32(float(np.uint32(tb).view(np.float32)), c)
        t2 = bias32(t1, m, n - p)
        w = oracle.weight(exact.fp32_bits(t2))
        if w is None:
            tm, te = exact.decode_fp32_bits(exact.fp32_bits(t2))
            w = exact.exp2_rn(tm, te)
        W.append(w)
        V.append([exact.decode_bf16(x) for x in flat["v"][addr(n, "v"):addr(n, "v") + dv].tolist()])
    emin = min(e for _, e in W)
    Z = sum(mm << (e - emin) for mm, e in W)
    for ch in range(dv):
        num = sum((mm * V[j][ch][0]) << (e - emin + V[j][ch][1] + 140) for j, (mm, e) in enumerate(W) if V[j][ch][0])
        om, oe = exact.round_rational(num, Z << 140, fmt)
        res[ch] = 0 if om == 0 else enc(om, oe)
    return res

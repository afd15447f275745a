"""The check of drafted tokens restated with Python numbers: tests in fp64, sums in integers. Test infrastructure."""

import math

import numpy as np


def _clip(x):
    x = float(x)
    return 0.0 if not x > 0 else min(x, 1.0)


def check(probs, drafted, uniforms, draft_probs=None, parents=None, count=None):
    """One sequence: (accepted path, its tokens, the new token, its margin): probs (N + 1, V), drafted (N,), uniforms (N + 1,) fp32. margin:
    how near, relative to 1 or to the total, any decision came to going the other way."""
    N, V = len(drafted), probs.shape[1]
    n = N if count is None else min(max(int(count), 0), N)
    par = [i - 1 if parents is None else int(parents[i]) for i in range(n)]
    par = [p if -1 <= p < i and 0 <= drafted[i] < V else -2 for i, p in enumerate(par)]
    cur, path, lost, margin = -1, [], [], math.inf
    mass = 0.0
    for i in range(n):
        if par[i] != cur:
            continue
        x, u = int(drafted[i]), float(uniforms[i])
        p = _clip(probs[cur + 1][x])
        if draft_probs is not None:
            a = u * _clip(draft_probs[i][x])
            take = a < p
        elif x in lost:
            lost.append(x)
            continue
        else:
            a = u * (1.0 - mass)
            take = a < p
        margin = min(margin, abs(a - p))
        if take:
            path.append(i)
            cur, lost, mass = i, [], 0.0
        else:
            lost.append(x)
            mass += p
            if draft_probs is not None:
                break
    row = [_clip(y) for y in probs[cur + 1]]
    if draft_probs is not None:
        w = list(row)
        if len(path) < n:
            w = [max(a - _clip(b), 0.0) for a, b in zip(row, draft_probs[len(path)])]
    else:
        w = [0.0 if j in set(lost) else a for j, a in enumerate(row)]
    w = [int(a * 2.0 ** 44) for a in w]
    if not sum(w):
        w = [int(a * 2.0 ** 44) for a in row]
    total = sum(w)
    new = -1
    if total:
        u = float(uniforms[N])
        goal = int(u * float(total)) if u > 0 else 0
        goal = min(goal, total - 1)
        at = 0
        for j, a in enumerate(w):
            at += a
            if at > goal:
                new = j
                break
    return path, [int(drafted[i]) for i in path], new, margin


def outputs(N, path, toks, new):
    return (len(path), path + [-1] * (N - len(path)), toks + [new] + [-1] * (N - len(path)))


def softmax(rng, shape, sharp):
    z = sharp * rng.standard_normal(shape)
    z = np.exp(z - z.max(-1, keepdims=True))
    return (z / z.sum(-1, keepdims=True)).astype(np.float32)

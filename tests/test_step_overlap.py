"""Which outputs of the rotary positions share memory with their inputs: the test of it, on the CPU, against
sets of bytes."""

import random

import pytest

from exactattention_amd.step import _apart, _same


def _bytes(x, d):
    p, n, h, st, sh, e = x
    return {p + (t * st + g * sh) * e + b for t in range(n) for g in range(h) for b in range(d * e)}


def test_against_sets_of_bytes():
    rng = random.Random(5)
    seen = [0, 0]
    for _ in range(6000):
        d = rng.choice([2, 4, 6])
        e = rng.choice([2, 4])

        def rows():
            n, h = rng.randrange(0, 5), rng.randrange(0, 4)
            sh = rng.choice([d, d + rng.randrange(8), 3 * d])
            st = rng.choice([max(1, h) * sh, max(1, h) * sh + rng.randrange(12), 3 * d * rng.randrange(1, 6)])
            if rng.random() < 0.3:
                st, sh = d, d * max(1, n) * rng.randrange(1, 3)  # heads first
            return (4096 + rng.randrange(0, 200) * 2, n, h, st, sh, rng.choice([e, 2]))

        x, y = rows(), rows()
        if rng.random() < 0.5:
            y = (x[0] + rng.randrange(-6, 30) * 2, y[1], y[2], x[3], x[4], x[5])
        apart = not (_bytes(x, d) & _bytes(y, d))
        seen[apart] += 1
        assert _apart(x, y, d) == apart == _apart(y, x, d), (x, y, d)
        if _same(x, y) and x[1:3] == y[1:3]:
            assert _bytes(x, d) == _bytes(y, d)
    assert min(seen) > 500


@pytest.mark.parametrize("n", [1, 7, 40000])
def test_views_of_a_fused_projection(n):
    """q, k and v of one (tokens, heads, dims) tensor, one after another or dealt head by head, at its sizes."""
    hq, hk, d, base = 16, 8, 128, 1 << 33
    row = (hq + 2 * hk) * d
    q, k = (base, n, hq, row, d, 2), (base + hq * d * 2, n, hk, row, d, 2)
    assert _apart(q, k, d) and _apart(k, q, d)
    assert not _apart(q, (base + 2 * (hq - 1) * d, n, hk, row, d, 2), d)
    dealt = [(base + 2 * i * d, n, hk, 3 * hk * d, 3 * d, 2) for i in range(3)]
    for i in range(3):
        assert not _apart(dealt[i], dealt[i], d) and _same(dealt[i], dealt[i])
        assert _apart(dealt[i], dealt[(i + 1) % 3], d)
    assert not _apart(dealt[0], (base + 2 * (d - 1), n, hk, 3 * hk * d, 3 * d, 2), d)
    first = [(base + 2 * i * n * d, n, hk, d, 2 * n * d, 2) for i in range(2)]  # heads of q and k in turn, tokens within
    assert _apart(*first, d)

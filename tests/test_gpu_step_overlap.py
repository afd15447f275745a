"""GPU: the rotary positions on tensors that share memory: in place on views of one projection, and the
outputs that are refused because a thread would read what another one has written."""

import pytest

from exactattention_amd.step import Rotary

pytestmark = pytest.mark.gpu


def _rand(shape, seed, dtype="bfloat16"):
    import torch
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(getattr(torch, dtype)).cuda()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("n", [1, 3, 1000])
@pytest.mark.parametrize("order", ["side", "dealt", "heads first"])
def test_in_place_on_views(gpu, n, order, dtype):
    import torch
    h, d = 4, 64
    x = _rand((n, 2 * h, d) if order != "heads first" else (2 * h, n, d), n, dtype)
    if order == "heads first":
        x = x.transpose(0, 1)
    q, k = (x[:, ::2], x[:, 1::2]) if order == "dealt" else (x[:, :h], x[:, h:])
    rot = Rotary(d, device="cuda:0")
    pos = torch.arange(n, dtype=torch.int32, device="cuda") * 3
    want = rot.rotate(q.clone(), k.clone(), pos)
    got = rot.rotate(q, k, pos, q_out=q, k_out=k)
    assert got[0] is q and torch.equal(q, want[0]) and torch.equal(k, want[1])
    if dtype == "bfloat16":
        # q in place and k on its way to the cache
        kp, vp = (torch.zeros((n, 1, h, d), dtype=torch.bfloat16, device="cuda") for _ in range(2))
        q2, v = q.clone(), _rand((n, h, d), 9)
        rot.append(q, k, v, pos, torch.arange(n, device="cuda"), kp, vp, q_out=q)
        w = rot.rotate(q2, k, pos)
        assert torch.equal(q, w[0]) and torch.equal(kp[:, 0], w[1]) and torch.equal(vp[:, 0], v)


def test_refused(gpu):
    import torch
    n, h, d = 6, 2, 32
    rot = Rotary(d, device="cuda:0")
    x = _rand((n + 2, 3 * h, d), 1)
    before = x.clone()
    q, k, v = x[:n, :h], x[:n, h:2 * h], x[:n, 2 * h:]
    pos = torch.arange(n, dtype=torch.int32, device="cuda")
    out = torch.empty((n, h, d), dtype=torch.bfloat16, device="cuda")
    wide = torch.empty((n, 2 * h, d), dtype=torch.bfloat16, device="cuda")
    pools = torch.zeros((2, n, 1, h, d), dtype=torch.bfloat16, device="cuda")
    dst = torch.arange(n, device="cuda")
    f32 = torch.empty((n, h, d), device="cuda")
    cases = [
        lambda: rot.rotate(q, k, pos, q_out=k),
        lambda: rot.rotate(q, k, pos, k_out=q),
        lambda: rot.rotate(q, k, pos, q_out=k, k_out=q),
        lambda: rot.rotate(q, k, pos, q_out=out, k_out=out),
        lambda: rot.rotate(q, k, pos, q_out=wide[:, :h], k_out=wide[:, 1:h + 1]),
        lambda: rot.rotate(q, k, pos, q_out=x[1:n + 1, :h]),              # the next token's q
        lambda: rot.rotate(q, k, pos, k_out=x[:n, h + 1:2 * h + 1]),      # the next head's k
        lambda: rot.append(q, k, v, pos, dst, pools[0], pools[0]),
        lambda: rot.append(q, k, v, pos, dst, pools[0], pools[1], q_out=k),
        lambda: rot.append(q, k, v, pos, dst, pools[0], pools[1], q_out=v),
        lambda: rot.append(q, k, v, pos, dst, pools[0], pools[1], q_out=x[1:n + 1, :h]),
        lambda: rot.append(q, k, v, pos, dst, pools[0], pools[1], q_out=pools[1, :, 0]),
        lambda: rot.append(q, k, v, pos, dst, pools[0], pools[1], q_rows=dst, q_out=x[2:, :h]),
        lambda: rot.append(f32, f32.clone(), f32.clone(), pos, dst, pools[0], pools[1],
                           q_out=f32.view(torch.bfloat16).view(n, h, 2 * d)[..., :d]),
    ]
    for i, call in enumerate(cases):
        with pytest.raises(ValueError, match="share"):
            call()
            pytest.fail(f"case {i}")
    torch.cuda.synchronize()
    assert torch.equal(x, before) and not bool(pools.any())
    # v and q_out where q_rows leave their memory alone, and k and v of a pool's pages that are not named again
    rot.append(q, k, v, pos, dst, pools[0], pools[1], q_rows=dst, q_out=out)
    a = rot.rotate(q, k, pos)
    assert torch.equal(out, a[0]) and torch.equal(pools[0, :, 0], a[1])

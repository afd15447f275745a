"""GPU: the rotary positions at token counts around which a block takes one, two or four tokens, against the
same tokens turned a few at a time: the same bits."""

import pytest

from exactattention_amd.step import Rotary

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq, hk, d, kw", [(2, 1, 64, {}), (5, 1, 128, {}), (16, 4, 128, {}), (3, 1, 40, dict(rot_dim=12)),
                                           (2, 2, 72, dict(adjacent=True, rot_dim=48)), (40, 8, 128, {})])
@pytest.mark.parametrize("n", [767, 1535, 1537, 8191, 8193, 16385])
def test_blocks_of_tokens(gpu, n, hq, hk, d, kw):
    import torch
    g = torch.Generator().manual_seed(n)
    rot = Rotary(d, device="cuda:0", **kw)
    x = torch.randn((n, hq + 2 * hk, d), generator=g).bfloat16().cuda()
    q, k, v = x[:, :hq], x[:, hq:hq + hk], x[:, hq + hk:]
    pos = torch.randint(0, 1 << 20, (n,), generator=g, dtype=torch.int32).cuda()
    dst = torch.randperm(n + 7, generator=g)[:n].cuda()
    dst[::13] = -1
    rows = (n + 7 + 15) // 16
    pools = [torch.full((rows, 16, hk, d), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(4)]
    whole = rot.append(q, k, v, pos, dst, pools[0], pools[1])
    parts = [rot.append(*(t[a:a + 700] for t in (q, k, v, pos, dst)), pools[2], pools[3]) for a in range(0, n, 700)]
    assert torch.equal(whole, torch.cat(parts))
    assert torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    skipped = sorted(set(range(n + 7)) - set(dst.tolist()))[:50]
    assert bool((pools[0].view(-1, hk, d)[skipped] == 3.0).all())

"""GPU: forward() without rotary positions plans its step on the host, in the append's own launch."""

import numpy as np
import pytest

from exactattention_amd.formats import default_alpha_bits
from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache
from gen import bf16

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("counts", [[3, 2, 1], [1, 40, 2], [5, 5, 5], [1, 1, 1]])
def test_one_launch_for_plan_and_append(gpu, counts, monkeypatch):
    import torch
    Hq, Hkv, d = 4, 2, 64

    def run(singly):
        r = np.random.default_rng(4)
        c = PagedKVCache(num_pages=60, page_size=16, num_kv_heads=Hkv, head_dim=d, max_seqs=3, max_seq_len=200)
        be = ExactAttentionBackend(c, Hq, None, alpha_bits=default_alpha_bits(d))
        slots = [c.add_sequence() for _ in counts]
        if not singly:
            monkeypatch.setattr(c, "_step_plan", lambda *a, **kw: pytest.fail("planned on the device"))
        outs = []
        for ql in ([17, 30, 1], counts, counts):
            q, k, v = (torch.from_numpy(bf16(r, (sum(ql), h, d)).view(np.int16)).cuda() for h in (Hq, Hkv, Hkv))
            if singly:  # token by token of each sequence
                at, got = 0, []
                for s, n in zip(slots, ql):
                    for j in range(n):
                        got.append(be.forward(*(x[at + j:at + j + 1] for x in (q, k, v)), [s], [1])[0])
                    at += n
                outs.append(torch.cat(got))
            else:
                out, fl = be.forward(q, k, v, slots, ql)
                be.check_flags(fl)
                outs.append(out)
        return outs, c

    (a, ca), (b, cb) = run(False), run(True)
    for x, y in zip(a, b):
        assert torch.equal(x, y)
    assert ca.length == cb.length

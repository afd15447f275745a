"""ExactAttentionBackend.accept on a host-resident cache: paths that name no node are refused before anything
changes, with rotary positions too (where the rows are gathered on the cache's device)."""

from types import SimpleNamespace

import numpy as np
import pytest

from exactattention_amd.formats import default_alpha_bits
from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache
from gen import bf16


def _backend(rotary, axes=1):
    rng = np.random.default_rng(1)
    c = PagedKVCache(num_pages=8, page_size=8, num_kv_heads=2, head_dim=16, max_seqs=1, max_seq_len=40, digits=False, device="cpu")
    be = ExactAttentionBackend(c, 4, None, alpha_bits=default_alpha_bits(16),
                               rotary=SimpleNamespace(head_dim=16, axes=axes) if rotary else None)
    s = c.add_sequence()
    c.append(s, bf16(rng, (13, 2, 16)), bf16(rng, (13, 2, 16)))
    return be, c, s, bf16(rng, (3, 2, 16)), bf16(rng, (3, 2, 16))


@pytest.mark.parametrize("rotary", [False, True])
@pytest.mark.parametrize("path", [[3], [0, 1, 7], [-4], [[0, 1]], [0, 1 << 40]])
def test_paths_that_name_no_node(path, rotary):
    be, c, s, k, v = _backend(rotary)
    before = c.k.clone()
    with pytest.raises(IndexError):
        be.accept(s, 10, path, k, v)
    assert c.length[s] == 13 and len(c.pages[s]) == 2 and bool((c.k == before).all())


def test_positions_that_accept_does_not_have():
    be, c, s, k, v = _backend(True, axes=3)
    with pytest.raises(ValueError):
        be.accept(s, 10, [0], k, v)
    assert c.length[s] == 13


def test_accepted_path():
    be, c, s, k, v = _backend(False)
    be.accept(s, 10, [0, -1], k, v)
    assert c.length[s] == 12
    rows = [int(c.block_table[s, n // 8]) * 8 + n % 8 for n in (10, 11)]
    assert np.array_equal(c.k.view(-1, 2, 16)[rows].numpy().view(np.uint16), k[[0, 2]])
    assert np.array_equal(c.v.view(-1, 2, 16)[rows].numpy().view(np.uint16), v[[0, 2]])
    be.accept(s, 4, [], k, v)
    assert c.length[s] == 4

"""ExactAttentionBackend.verify_tree on a host-resident cache: parents that are no tree are refused before
anything changes (a cycle among them would be walked for ever)."""

import numpy as np
import pytest

from exactattention_amd.formats import default_alpha_bits
from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache
from gen import bf16


@pytest.mark.parametrize("parents", [[0, 0, 1], [-1, 1, 0], [-1, 2, 1], [1, -1, 0], [-1, 0, 5]])
def test_parents_after_their_nodes(parents):
    rng = np.random.default_rng(1)
    c = PagedKVCache(num_pages=8, page_size=8, num_kv_heads=2, head_dim=16, max_seqs=1, max_seq_len=40, digits=False, device="cpu")
    be = ExactAttentionBackend(c, 4, None, alpha_bits=default_alpha_bits(16))
    s = c.add_sequence()
    c.append(s, bf16(rng, (5, 2, 16)), bf16(rng, (5, 2, 16)))
    with pytest.raises(ValueError, match="parent"):
        be.verify_tree(s, bf16(rng, (3, 4, 16)), bf16(rng, (3, 2, 16)), bf16(rng, (3, 2, 16)), parents)
    assert c.length[s] == 5

"""Positions given to ExactAttentionBackend's calls from the host: whole numbers that fit 32 bits, or refused."""

from types import SimpleNamespace

import numpy as np
import pytest

from exactattention_amd.formats import default_alpha_bits
from exactattention_amd.serving import ExactAttentionBackend, PagedKVCache


def _backend(axes=1):
    c = PagedKVCache(num_pages=4, page_size=8, num_kv_heads=2, head_dim=16, max_seqs=1, max_seq_len=32, digits=False, device="cpu")
    return ExactAttentionBackend(c, 4, None, alpha_bits=default_alpha_bits(16), rotary=SimpleNamespace(head_dim=16, axes=axes))


@pytest.mark.parametrize("positions", [np.array([1, 2, 1 << 31]), np.array([0, -(1 << 31) - 1, 3]), np.array([0.0, 1.5, 2.0]),
                                       np.array([1, 2, (1 << 32) + 3], np.uint64), [0, 1, 1 << 40], [0, 1], 5, np.array([True, False, True])])
def test_refused(positions):
    with pytest.raises(ValueError):
        _backend()._positions(positions, 3)


@pytest.mark.parametrize("positions", [[4, 5, 6], np.array([4, 5, 6]), np.array([4, 5, 6], np.uint8), np.array([(1 << 31) - 1, -(1 << 31), 0])])
def test_taken(positions):
    p = _backend()._positions(positions, 3)
    assert p.dtype.itemsize == 4 and p.tolist() == list(positions)
    assert _backend()._positions([], 0).numel() == 0 and _backend()._positions(None, 3) is None
    assert _backend(2)._positions([[1, 2, 3], [4, 5, 6]], 3).shape == (2, 3)

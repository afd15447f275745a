"""Calls that a cache held in 4 bits refuses before anything runs or changes: no GPU."""

from types import SimpleNamespace

import pytest

from exactattention_amd import hip


def test_no_digit_tiles_of_a_4_bit_cache(monkeypatch):
    """Neither made for such a problem nor updated from one: the update reads rows of bf16."""
    def unreached():
        raise AssertionError("the library was called")

    monkeypatch.setattr(hip, "load", unreached)
    dp = SimpleNamespace(kv4=object(), geom=dict(num_seqs=1, num_kv_heads=1), out=None, torch=None)
    with pytest.raises(ValueError, match="4 bits"):
        hip.KVDigits(dp, 4)
    cache = hip.KVDigits.__new__(hip.KVDigits)  # as made for another problem
    cache.tiles, cache.buf = 4, None
    with pytest.raises(ValueError, match="4 bits"):
        cache.update(dp, None, None, 64)

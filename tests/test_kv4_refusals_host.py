"""Calls that a cache held in 4 bits refuses before anything runs or changes: no GPU."""

from types import SimpleNamespace

import numpy as np
import pytest

from exactattention_amd import hip
from exactattention_amd.kv4 import KV4Pool
from exactattention_amd.serving import PagedKVCache


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


@pytest.mark.parametrize("shape", [(3, 4, 64), (3, 1, 64), (3, 2, 32), (3, 2, 128)])
def test_keys_of_other_heads_change_nothing(shape):
    """Keys of other heads than the cache's are refused while lengths, pages and the table still are as they were (a 4-bit cache
    took the first rows of what they reshape to, or raised with the pages taken)."""
    c = PagedKVCache(4, 16, 2, 64, 2, 64, device="cpu")
    s = c.add_sequence()
    good, bad = np.zeros((3, 2, 64), np.uint16), np.zeros(shape, np.uint16)
    for k, v in ((bad, good), (good, bad), (bad, bad)):
        with pytest.raises(ValueError, match="bf16 bits"):
            c.append(s, k, v)
        assert c.length[s] == 0 and c.pages[s] == [] and len(c.free) == 4
    c.append(s, good, good)
    assert c.length[s] == 3 and len(c.free) == 3


def test_heads_that_attention_does_not_take():
    """Heads past 128: a pool may hold them, but a cache to be served from, and a problem, say so when they are made, not by an
    attention call's error code after the keys are in."""
    for d in (136, 256):
        with pytest.raises(ValueError, match="up to 128"):
            PagedKVCache(4, 16, 2, d, 1, 64, bits=4)
        pool = KV4Pool(1, 16, 1, d, device="cpu")
        with pytest.raises(ValueError, match="up to 128"):
            hip.DeviceProblem(dict(geom=dict(num_seqs=1, num_tokens=1, num_q_heads=1, max_seq_len=16, block_table_stride=1,
                                             **pool.geometry()), kv4=pool, q=np.zeros((1, 1, 1, d), np.uint16),
                                   seq_len=np.ones(1, np.int32), kv_len=np.ones(1, np.int32), block_table=np.zeros((1, 1), np.int32),
                                   out_shape=(1, 1, 1, d)), device="cpu")


@pytest.mark.parametrize("seqs, keys", [(3, 16), (2, 17), (1, 64)])
def test_no_block_table_and_no_page(seqs, keys):
    """Without a block table the kernels read page b for sequence b: more sequences than pages, or longer ones, would be read from
    behind the pool."""
    pool = KV4Pool(2, 16, 1, 64, device="cpu")
    with pytest.raises(ValueError, match="block table"):
        hip.DeviceProblem(dict(geom=dict(num_seqs=seqs, num_tokens=1, num_q_heads=1, max_seq_len=keys, block_table_stride=0,
                                         q_seq_stride=64, q_tok_stride=64, q_head_stride=64, o_seq_stride=64, o_tok_stride=64,
                                         o_head_stride=64, **pool.geometry()), kv4=pool, q=np.zeros((seqs, 1, 1, 64), np.uint16),
                               seq_len=np.full(seqs, keys, np.int32), kv_len=np.full(seqs, keys, np.int32),
                               out_shape=(seqs, 1, 1, 64)), device="cpu")

"""The step plan's arrays that share memory are refused, on the host (no device call is made)."""

import ctypes

import pytest

from exactattention_amd import hip

NAMES = ["seq_len", "counts", "slots", "free_pages", "num_free", "block_table", "dst_rows", "positions", "seq_of", "q_rows", "kv_len",
         "new_seq_len", "new_num_free", "status"]
SIZE = dict(seq_len=8, counts=8, slots=8, free_pages=12, num_free=4, block_table=4 * 4 * 8, dst_rows=32, positions=16, seq_of=16,
            q_rows=32, kv_len=16, new_seq_len=8, new_num_free=4, status=4)
WRITTEN = NAMES[5:]


def _plan(**kw):
    a = dict(num_seqs=2, page_size=16, table_rows=4, table_width=8, max_tokens=4, pad_tokens=2, max_seq_len=100, free_capacity=3)
    a.update({n: (i + 1) << 20 for i, n in enumerate(NAMES)})
    a.update(kw)
    return a


def _refused(a):
    return hip.load().ea_hip_step_plan(ctypes.byref(hip.StepPlanArgs(**a)), None) == -1


@pytest.mark.parametrize("written", WRITTEN)
def test_shared(written):
    for other in NAMES:
        if other == written:
            continue
        at = _plan()[other]
        for p in (at, at + SIZE[other] - 4, at - SIZE[written] + 4):
            assert _refused(_plan(**{written: p})), (written, other, p - at)


def test_optional_arrays_do_not_count():
    """An array that is left out shares nothing; the rest is still looked at."""
    for n in ("positions", "seq_of", "q_rows", "kv_len", "slots"):
        assert _refused(_plan(**{n: None, "dst_rows": _plan()["counts"]}))

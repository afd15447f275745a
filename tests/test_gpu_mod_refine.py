"""GPU: tier 2's double-double pass on rows with score modifications, against the definition: the rows that
tier 1 lists, of scores and biases that spread the weights over thousands of binades."""

import numpy as np
import pytest

from exactattention_amd import hip, problem
from exactattention_amd.formats import default_alpha_bits
from gen import bf16
import mod_oracle as mo

pytestmark = pytest.mark.gpu


def _steps(p, ab, m, kernel, out):
    """(tier 1's flags, the step's bits, flags and counters)."""
    import torch
    got = []
    for tier2 in (False, True):
        dp = hip.DeviceProblem(p, out, 0, "cuda:0", kernel, mods=hip.ScoreMods(**m))
        dp.out.fill_(-1)
        hip.launch_hip(dp, ab, tier2=tier2)
        torch.cuda.synchronize()
        got.append(dp)
    st = dict(zip(hip.STATS, got[1].stats.tolist()))
    return got[0].flags.cpu().numpy(), got[1].out.cpu().numpy().view(np.uint32 if out == "fp32" else np.uint16), got[1].flags.cpu().numpy(), st


@pytest.mark.parametrize("steep", [0.02, 1.0, 20.0])
@pytest.mark.parametrize("cap", [0.0, 30.0])
@pytest.mark.parametrize("T, d, S", [(40, 128, 300), (70, 96, 190)])
def test_rows_the_prefill_kernel_lists(gpu, T, d, S, cap, steep):
    """fp32 outputs under a bias: the int32 sums leave rows undecided, more of them the steeper it is. Positions
    past and before the prefix's end, so that the largest weights come first, last or in the middle of a row."""
    rng = np.random.default_rng(T + int(steep * 10))
    Hq = 4
    p = problem.contiguous(bf16(rng, (1, T, Hq, d), "normal", 3.0), bf16(rng, (1, 2, S, d)), bf16(rng, (1, 2, S, d)),
                           S - T + 1 + np.arange(T)[None])
    m = dict(slopes=np.float32(steep * 2.0 ** -np.arange(Hq)), softcap=cap, q_pos=rng.integers(-200, S + 200, (1, T)).astype(np.int32))
    ab = default_alpha_bits(d)
    listed, res, fl, st = _steps(p, ab, m, "prefill", "fp32")
    rows = np.flatnonzero(listed == 1)
    assert len(rows) == st["tier1_flagged"] > 0 and st["tier2_certified"] == len(rows) and (fl == 0).all(), st
    assert st["tier2_wide_rows"] < len(rows), st  # the pass decides rows itself
    for r in rng.permutation(rows)[:25].tolist():
        assert np.array_equal(res.reshape(-1, d)[r], mo.row(p, ab, r, "fp32", slopes=m["slopes"], q_pos=m["q_pos"], cap=cap)), r


@pytest.mark.parametrize("slope", [0.0, 3.0, 45.0])
@pytest.mark.parametrize("S", [60, 700])
def test_rows_that_cancel(gpu, S, slope):
    """Few rows, their keys in chunks: channels whose terms cancel to 2^-40 of their size fail tier 1's bound on
    every kernel. The bias (45 a key: 2^-900 within 20 keys) drops whole chunks below the others."""
    rng = np.random.default_rng(S)
    Hq, d = 2, 64
    p = problem.contiguous(bf16(rng, (1, 1, Hq, d)), bf16(rng, (1, 1, S, d)), bf16(rng, (1, 1, S, d)), np.array([[S]]))
    p["q"][0, 0, 0] = 0  # equal scores
    # positions in the middle of the keys, whose neighbours on both sides then weigh the same
    mid = S // 2
    col = np.zeros(S, np.uint16)
    for i in range(1, min(mid, S - mid - 1)):
        col[mid - i], col[mid + i] = 0x3FC0, 0xBFC0  # 1.5, -1.5
    col[mid] = 0x2C00  # about 2^-39
    p["v"][0, 0, :, 0] = col
    m = dict(slopes=np.full(Hq, slope, np.float32), q_pos=np.array([[mid]], np.int32))
    ab = default_alpha_bits(d)
    for out in ("bf16", "fp32"):
        for kernel in ("auto", "general"):
            listed, res, fl, st = _steps(p, ab, m, kernel, out)
            assert (fl == 0).all(), st
            if slope < 40:
                assert listed[0] == 1 and st["tier2_certified"] >= 1, st
            for r in range(Hq):
                assert np.array_equal(res.reshape(-1, d)[r], mo.row(p, ab, r, out, slopes=m["slopes"], q_pos=m["q_pos"])), (out, kernel, r)

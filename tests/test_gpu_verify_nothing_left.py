"""verify_drafts where a refused draft leaves no weight, over a large vocabulary."""
from __future__ import annotations

import math

import pytest
import torch

from test_gpu_verify import Step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("outright", [False, True])
def test_a_refusal_that_leaves_nothing_takes_no_longer(gpu_ops, dtype, outright):
    """Over a large vocabulary, beside rows that draw from what is left: the same
    tokens as the rule's, in a call no slower than that of an ordinary refusal
    but for the second search (four times its time, where summing the row
    thread by thread took hundreds)."""

    def step(nothing):
        s = Step(3, 2, 2**20 + 3, dtype, outright=outright, counts=False, seed=23)
        s.accept_u.fill_(1.0)  # outside [0, 1): refuses q = p
        if outright:
            s.target[:, :, 1000] = 0.0  # refused: no probability of its own
            s.tokens.fill_(1000)
            if nothing:  # and nothing but NaN and negative values beside it
                s.target[0] = math.nan
                s.target[2, :, ::2], s.target[2, :, 1::2] = -1.0, 0.0
        elif nothing:
            s.draft[0], s.draft[2] = s.target[0, :2], s.target[2, :2]
        else:
            s.tokens.fill_(1000)
            s.target[:, :, 1000] = 0.0
        return s

    def microseconds(s):
        call = gpu_ops.bind_verify_drafts(*s.args(gpu_ops))
        best = math.inf
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            call()
            b.record()
            torch.cuda.synchronize()
            best = min(best, 1e3 * a.elapsed_time(b))
        s.compare()
        return best

    ordinary, nothing = step(False), step(True)
    quick, slow = microseconds(ordinary), microseconds(nothing)
    assert nothing.acc.tolist()[0] == 0 and nothing.acc.tolist()[2] == 0
    print("ordinary %.1f us, nothing left %.1f us" % (quick, slow))
    assert slow <= 4 * quick

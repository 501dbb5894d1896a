"""token_logprobs over logits of any finite size: mask constants, ties and levels from a
hundred to the type's largest values.

The tolerances are test_gpu_logprobs's, which count what holds at any size (y = x - m in
fp32 is off by at most half a step of itself), and one term more for rows whose other
tokens all lie some 87 to 104 below the largest: an exponential below 2^-126, fp32's
least normal value, may count as zero.  Each of V such takes 2^-126 at most from S and
|y| 2^-126 < 2^-119 from the mean (|y e^y| falls with y there; 87.4 at the border), so a
row's results are off by V 2^-119 at most, 2^-101 for the largest V here.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

import test_gpu_logprobs as plain
from gpu_cases import DEV
from test_gpu_logprobs import CHAIN, STEP, logits_of

pytestmark = pytest.mark.gpu

SIZES = [100.0, 3000.0, 4095.0, 4097.0, 5000.0, 6.0e4, 1.0e5, 1.0e6, 1.0e7, 1.0e8, 1.0e9, 1.0e10, 1.0e20, 1.0e30,
         1.0e36, 1.0e37, 3.0e38]


class Rows(plain.Rows):
    def check(self):
        """In 64 bits on the GPU."""
        x = self.x.double().nan_to_num(-math.inf, math.inf, -math.inf)
        n, vocab = x.shape
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        m = x.amax(1, keepdim=True)
        some = m > -math.inf
        y = torch.where(x == m, 0.0, x - m)
        size = torch.where(y > -math.inf, y.abs(), 0.0)
        e = torch.where(some, y.exp(), 0.0)
        others = e.scatter(1, order[:, :1], 0.0)  # without one largest element
        under = vocab * 2.0**-119
        rest = others.sum(1, keepdim=True)
        dr = (others * 2 * STEP * (2 * size + 4)).sum(1, keepdim=True) + CHAIN * STEP * rest + under
        log_s = torch.log1p(rest)
        dlog = dr / (1 + rest) + 2 * STEP * log_s
        ye = torch.where(e > 0, y * e, 0.0)
        mean = ye.sum(1, keepdim=True)
        dmean = (ye.abs() * 2 * STEP * (2 * size + 5)).sum(1, keepdim=True) + CHAIN * STEP * mean.abs() + under
        h = torch.where(some, log_s - mean / (1 + rest), 0.0)
        dh = dlog + dmean / (1 + rest) + mean.abs() * dr / (1 + rest) ** 2 + 4 * STEP * (log_s + mean.abs() / (1 + rest))

        def near(name, got, want, dy):
            fine = torch.isfinite(want)
            assert torch.equal(got.double()[~fine], want[~fine]), name + ": infinities differ"
            err = (got.double() - want).abs()[fine]
            tol = (dy + STEP * want.abs())[fine]
            assert bool((err <= tol).all()), "%s: %.3g off, %.3g of the tolerance" % (name, err.max(), (err / tol).max())

        token = self.t.long()[:, None]
        inside = (token >= 0) & (token < vocab)
        at = token.clamp(0, vocab - 1)
        there = inside & (x.gather(1, at) > -math.inf)
        yt = torch.where(there, y.gather(1, at), 0.0)
        lp = torch.where(there, yt - log_s, -math.inf)
        near("logprobs", self.lp, lp[:, 0], (dlog + STEP * yt.abs())[:, 0])
        place = (order == token).int().argmax(1) + 1
        assert torch.equal(self.rank.long(), torch.where(there[:, 0], place, 0)), "ranks"
        near("entropy", self.h, h[:, 0], dh[:, 0])
        first = order[:, : self.top]
        live = x.gather(1, first) > -math.inf
        pad = (0, self.top - first.shape[1])
        ids = torch.nn.functional.pad(torch.where(live, first, -1), pad, value=-1)
        assert torch.equal(self.ids, ids), "ids"
        lps = torch.nn.functional.pad(torch.where(live, y.gather(1, first) - log_s, -math.inf), pad, value=-math.inf)
        dy = torch.nn.functional.pad(dlog + STEP * size.gather(1, first), pad, value=0.0)
        near("likeliest", self.lps, lps, dy)
        assert bool((self.ids_all[:, 0] == 99).all() and (self.ids_all[:, -1] == 99).all() and (self.lps_all[:, -1] == 99).all())


def rows_of_size(size, vocab, dtype, seed):
    """Rows: all equal; the first three fifths masked by -size; maxima tied at size;
    all masked but the last; every second one masked; a level of -size, and one of size."""
    x = logits_of(7, vocab, torch.float32, seed)
    gen = torch.Generator().manual_seed(seed)
    x[0] = -size
    x[1, : vocab * 3 // 5] = -size
    x[2, torch.randint(0, vocab, (3,), generator=gen).to(DEV)] = size
    x[3, :-1] = -size
    x[4, seed % 2 :: 2] = -size
    x[5] -= size
    x[6] += size
    return x.to(dtype)


def repeated(ops, patterns, tokens, top, rows):
    """``rows`` rows that repeat the patterns: each as the first of its kind, those checked."""
    n = patterns.shape[0]
    index = torch.arange(rows, device=DEV) % n
    st = Rows(patterns[index], (tokens * (rows // n + 1))[:rows], top).run(ops)
    outs = ("lp", "rank", "h", "ids_all", "lps_all")
    for name in outs:
        got = getattr(st, name)
        assert torch.equal(got, got[index]), name
    first = Rows(patterns, tokens, top)
    for name in outs:
        getattr(first, name).copy_(getattr(st, name)[:n])
    first.check()


# One work-group a row that holds it; one that streams it in fp32; slices that are held;
# rows streamed whole; rows streamed in slices.
@pytest.mark.parametrize("rows,vocab,sizes", [(0, 70, SIZES), (0, 5000, SIZES), (0, 40001, SIZES[::2]),
                                              (600, 20000, SIZES), (64, 300000, SIZES[1::4])])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_large_logits(gpu_ops, dtype, rows, vocab, sizes):
    sizes = [s for s in sizes if s <= torch.finfo(dtype).max]
    patterns = torch.cat([rows_of_size(s, vocab, dtype, 3 + i) for i, s in enumerate(sizes)])
    rng = random.Random(vocab)
    tokens = [rng.choice((0, vocab - 1, rng.randrange(vocab))) for _ in range(patterns.shape[0])]
    if rows:
        repeated(gpu_ops, patterns, tokens, 8, rows)
    else:
        Rows(patterns, tokens, 8).run(gpu_ops).check()


@pytest.mark.parametrize("vocab", [70, 5000, 70001])
def test_masked_rows_in_bf16(gpu_ops, vocab):
    """The type's lowest and largest values, equal and beside ordinary ones."""
    low, high = torch.finfo(torch.bfloat16).min, torch.finfo(torch.bfloat16).max
    x = logits_of(6, vocab, torch.bfloat16, 5)
    x[0] = low
    x[1] = low
    x[1, vocab // 2] = 1.0
    x[2, : vocab * 4 // 5] = low
    x[3] = high
    x[4, ::2] = low
    x[5, 2::3] = -float("inf")
    for tokens in ([0, vocab // 2, vocab - 1, 1, 0, 5], [vocab - 1, 0, 0, vocab - 1, 1, 0]):
        Rows(x, tokens, 20).run(gpu_ops).check()

"""token_logprobs against log-softmax in 64 bits.

Ranks and ids have to be equal.  With y = x - m in fp32 (half a step, 2^-24 |y|),
exp(y) is off by that and by the exponential's own few steps, 2^-23 (2 |y| + 4) of
it in all; a sum of n terms in fp32 adds 2^-24 of the sum for each of the additions
that one partial sum takes (a few hundred here, CHAIN), and sums of sums are exact
beside that.  S = 1 + r, so log S is off by dr / (1 + r) and two steps of itself, and a
log probability by that, y's half step and its own.
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from gpu_cases import DEV

pytestmark = pytest.mark.gpu

CHAIN = 640
STEP = 2.0**-24


class Rows:
    def __init__(self, logits, tokens, top, int64=True, entropy=True):
        n = logits.shape[0]
        self.x, self.top, self.n = logits, top, n
        self.t = torch.tensor(tokens, dtype=torch.int64 if int64 else torch.int32, device=DEV)
        self.lp = torch.full((n,), 99.0, device=DEV)
        self.rank = torch.full((n,), 99, dtype=torch.int32, device=DEV)
        self.h = torch.full((n,), 99.0, device=DEV) if entropy else None
        self.ids_all = torch.full((n, top + 2), 99, dtype=torch.int64, device=DEV)
        self.lps_all = torch.full((n, top + 1), 99.0, device=DEV)
        self.ids, self.lps = self.ids_all[:, 1 : top + 1], self.lps_all[:, :top]

    def bind(self, ops):
        nbytes = ops.token_logprobs_workspace_bytes(self.n, self.x.shape[1], self.top)
        self.ws = torch.full((max(16, nbytes),), 0xFF, dtype=torch.uint8, device=DEV)
        return ops.bind_token_logprobs(self.x, self.t, self.ws, self.lp, self.rank, self.h, self.ids, self.lps)

    def run(self, ops):
        self.bind(ops)()
        torch.cuda.synchronize()
        return self

    def check(self):
        x = self.x.double().cpu()
        x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
        vocab = x.shape[1]
        order = torch.sort(x, dim=1, descending=True, stable=True).indices
        m = x.amax(1, keepdim=True)
        some = m > -math.inf
        y = torch.where(x == m, 0.0, x - m)
        e = torch.where(some, y.exp(), torch.zeros_like(y))
        rest = (e.sum(1, keepdim=True) - some.double()).clamp_min(0)
        # Without the largest element by value, not by subtraction.
        first = torch.zeros_like(e).scatter_(1, order[:, :1], 1.0)
        rest = (e * (1 - first)).sum(1, keepdim=True)
        dr = (e * (1 - first) * 2 * STEP * (2 * y.abs().nan_to_num(0, 0, 0) + 4)).sum(1, keepdim=True) + CHAIN * STEP * rest
        log_s = torch.log1p(rest)
        dlog = dr / (1 + rest) + 2 * STEP * log_s
        ye = torch.where(e > 0, y * e, torch.zeros_like(e))
        mean = ye.sum(1, keepdim=True)
        dmean = (ye.abs() * 2 * STEP * (2 * y.abs().nan_to_num(0, 0, 0) + 5)).sum(1, keepdim=True) + CHAIN * STEP * mean.abs()
        h = torch.where(some, log_s - mean / (1 + rest), torch.zeros_like(mean))
        dh = dlog + dmean / (1 + rest) + mean.abs() * dr / (1 + rest) ** 2 + 4 * STEP * (log_s + mean.abs() / (1 + rest))

        def near(got, want, dy):
            got, want = got.cpu().double(), want
            fine = torch.isfinite(want)
            assert torch.equal(got[~fine], want[~fine]), "infinities differ"
            err = (got - want).abs()[fine]
            tol = (dy + STEP * want.abs() + 2.0**-140)[fine]
            assert bool((err <= tol).all()), "%.3g off, %.3g of the tolerance" % (float(err.max()), float((err / tol).max()))

        tokens = self.t.cpu().long()
        inside = (tokens >= 0) & (tokens < vocab)
        at = tokens.clamp(0, vocab - 1)[:, None]
        xt = x.gather(1, at)[:, 0]
        there = inside & (xt > -math.inf)
        yt = torch.where(there, y.gather(1, at)[:, 0], torch.zeros_like(xt))
        near(self.lp, torch.where(there, yt - log_s[:, 0], torch.full_like(xt, -math.inf)), dlog[:, 0] + STEP * yt.abs().nan_to_num(0, 0, 0))
        place = (order == tokens[:, None]).int().argmax(1) + 1
        assert torch.equal(self.rank.cpu().long(), torch.where(there, place, torch.zeros_like(place)))
        if self.h is not None:
            near(self.h, h[:, 0], dh[:, 0])
        w = min(self.top, vocab)
        ids = torch.full((self.n, self.top), -1, dtype=torch.int64)
        lps = torch.full((self.n, self.top), -math.inf, dtype=torch.float64)
        ids[:, :w] = order[:, :w]
        live = x.gather(1, order[:, :w]) > -math.inf
        lps[:, :w] = torch.where(live, y.gather(1, order[:, :w]) - log_s, lps[:, :w])
        ids[:, :w][~live] = -1
        assert torch.equal(self.ids.cpu(), ids)
        near(self.lps, lps, dlog + STEP * y.gather(1, order[:, :1]).abs() + STEP * lps.abs().nan_to_num(0, 0, 0))
        assert bool((self.ids_all[:, 0] == 99).all() and (self.ids_all[:, -1] == 99).all() and (self.lps_all[:, -1] == 99).all())


def logits_of(n, vocab, dtype, seed, spread=2.5, pad=0):
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn((n, vocab), generator=gen) * spread
    x[::3, seed % vocab] += 20.0
    x = x.to(dtype)
    if pad:  # rows of a padded vocabulary
        buf = torch.full((n, vocab + pad), math.nan, dtype=dtype)
        buf[:, :vocab] = x
        return buf.to(DEV)[:, :vocab]
    return x.to(DEV)


VOCABS = [1, 2, 63, 64, 65, 100, 255, 1000, 1024, 2049, 4097, 32000, 65537, 152000]


@pytest.mark.parametrize("vocab", VOCABS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_vocabularies(gpu_ops, vocab, dtype):
    rng = random.Random(vocab)
    for n, top in ((1, 8), (7, 20), (3, 0), (2, 64)):
        tokens = [rng.choice((rng.randrange(vocab), rng.randrange(vocab), -1, vocab)) for _ in range(n)]
        Rows(logits_of(n, vocab, dtype, vocab + n, pad=n % 3), tokens, top, int64=n % 2 == 1, entropy=n != 3).run(gpu_ops).check()


@pytest.mark.parametrize("rows", [16, 64, 257, 1000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_many_rows(gpu_ops, rows, dtype):
    rng = random.Random(rows)
    vocab = 5003 if rows > 64 else 40001
    Rows(logits_of(rows, vocab, dtype, rows), [rng.randrange(vocab) for _ in range(rows)], 5).run(gpu_ops).check()


@pytest.mark.parametrize("vocab", [70, 5000, 70001])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_masked_rows(gpu_ops, vocab, dtype):
    """Rows with no token, one, fewer than asked for; NaN; the type's lowest value; infinities."""
    x = logits_of(12, vocab, dtype, 5)
    x[0] = -math.inf
    x[1] = -math.inf
    x[1, vocab - 1] = -3.0
    x[2, 5:] = -math.inf
    x[3] = torch.finfo(dtype).min
    x[4] = torch.finfo(dtype).min
    x[4, vocab // 2] = 1.0
    x[5, ::2] = math.nan
    x[6] = math.nan
    x[7, 3], x[7, vocab - 2] = math.inf, math.inf
    x[8] = 0.0  # all equal: the lowest indices
    x[9] = torch.finfo(dtype).max
    x[10, :] = -math.inf
    x[10, ::7] = 2.0
    x[11, 1:] = -30.0
    x[11, 0] = 30.0
    for tokens in ([0, vocab - 1, 4, 1, vocab // 2, 1, 0, vocab - 2, 63, 9, 14, 0], [1, 0, 5, vocab - 1, 0, 2, 3, 4, vocab - 1, 0, 1, 7]):
        Rows(x, tokens, 20).run(gpu_ops).check()


@pytest.mark.parametrize("dtype,bits", [(torch.bfloat16, 0x7F81), (torch.float16, 0x7C01), (torch.float32, 0x7F800001)])
@pytest.mark.parametrize("vocab", [90, 20000])
def test_signalling_nan(gpu_ops, dtype, bits, vocab):
    """Beside the row's largest values, in the first batch of elements and in later ones."""
    x = logits_of(4, vocab, dtype, 8)
    whole = x.view(torch.int32 if dtype == torch.float32 else torch.int16)
    for row, at in ((0, [0, 1, 2]), (1, [vocab - 1, vocab - 2, 5]), (2, list(range(1, 80, 2)))):
        whole[row, torch.tensor(at, device=DEV)] = bits
    x[0, 3], x[1, vocab - 3], x[2, 0] = 25.0, 25.0, 25.0
    Rows(x, [3, vocab - 1, 0, 5], 9).run(gpu_ops).check()


@pytest.mark.parametrize("vocab", [300, 9000, 152000])
def test_sorted_and_equal_rows(gpu_ops, vocab):
    """Rows in ascending and descending order (the likeliest last or first), few distinct values."""
    up = torch.arange(vocab, dtype=torch.float32) / vocab * 8
    x = torch.stack((up, up.flip(0), torch.arange(vocab) % 3 * 1.0, (torch.arange(vocab) // 100 % 7) * 0.5)).to(DEV)
    for dtype in (torch.float32, torch.bfloat16):
        Rows(x.to(dtype), [vocab - 1, vocab // 2, 2, vocab - 1], 64).run(gpu_ops).check()


def test_only_what_is_asked_for(gpu_ops):
    x = logits_of(5, 3000, torch.float32, 9)
    st = Rows(x, [1, 2, 3, 4, 5], 6)
    ws = torch.empty((max(16, gpu_ops.token_logprobs_workspace_bytes(5, 3000, 6)),), dtype=torch.uint8, device=DEV)
    gpu_ops.token_logprobs(x, None, ws, None, None, None, st.ids, st.lps)
    whole = Rows(x, [1, 2, 3, 4, 5], 6).run(gpu_ops)
    assert torch.equal(st.ids, whole.ids) and torch.equal(st.lps, whole.lps) and bool((st.lp == 99).all())
    gpu_ops.token_logprobs(x, st.t, ws, st.lp, st.rank, None, None, None)
    assert torch.equal(st.lp, whole.lp) and torch.equal(st.rank, whole.rank)
    assert gpu_ops.bind_token_logprobs(x[:0], None, None, None, None, None, None, None) is None


@pytest.mark.parametrize("rows,vocab", [(2, 40000), (300, 700)])
def test_replayed_with_other_logits(gpu_ops, rows, vocab):
    st = Rows(logits_of(rows, vocab, torch.bfloat16, 11), [3] * rows, 10)
    call = st.bind(gpu_ops)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(3):
        st.x.copy_(logits_of(rows, vocab, torch.bfloat16, 30 + seed, spread=1.0 + seed))
        st.t.random_(0, vocab)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        st.check()


def test_rows_beyond_32_bits(gpu_ops):
    """The last rows of a tensor whose elements pass 2^31."""
    vocab, n = 152001, 14200
    x = torch.zeros((n, vocab), dtype=torch.float16, device=DEV)
    last = logits_of(3, vocab, torch.float16, 13)
    x[-3:] = last
    st = Rows(x, [n % 7] * n, 3)
    st.bind(gpu_ops)()
    small = Rows(last, [n % 7] * 3, 3).run(gpu_ops)
    small.check()
    assert torch.equal(st.lp[-3:], small.lp) and torch.equal(st.ids[-3:], small.ids) and torch.equal(st.rank[-3:], small.rank)

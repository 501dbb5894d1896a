"""verify_drafts against the acceptance and sampling rule in 64 bits, token by token.

Every output is a whole number and has to be equal: the random numbers are
inputs, products are exact in float64, and the sums' order moves a border by
about 2^-50 of the sum, which these inputs do not meet."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
BELOW_ONE = 1.0 - 2.0**-24


def verify64(target, draft, tokens, counts, accept_u, sample_u, lens):
    """The rule on the CPU."""
    target, tokens = target.cpu().double(), tokens.cpu()
    draft = None if draft is None else draft.cpu().double()
    batch, k = tokens.shape
    vocab = target.shape[2]
    out = torch.full((batch, k + 1), -1, dtype=torch.int64)
    acc = torch.zeros(batch, dtype=torch.int32)
    for b in range(batch):
        n = k if counts is None else min(max(int(counts[b]), 0), k)
        a = 0
        while a < n:
            x = int(tokens[b, a])
            if not 0 <= x < vocab:
                break
            q = 1.0 if draft is None else float(draft[b, a, x])
            if not float(accept_u[b, a]) * q < float(target[b, a, x]):
                break
            out[b, a] = x
            a += 1
        w = target[b, a].clone()
        if a < n:
            if draft is not None:
                w = w - draft[b, a]
            elif 0 <= int(tokens[b, a]) < vocab:
                w[int(tokens[b, a])] = 0.0
        w = torch.where(w > 0, w, torch.zeros_like(w))
        if float(w.sum()) == 0.0:
            w = torch.where(target[b, a] > 0, target[b, a], torch.zeros_like(w))
        c = w.cumsum(0)
        if float(c[-1]) > 0:
            past = (c > float(sample_u[b]) * float(c[-1])).nonzero()
            out[b, a] = int(past[0]) if len(past) else int((w > 0).nonzero()[-1])
        acc[b] = a
    return out, acc, lens.cpu() + acc + 1


class Step:
    """One step's inputs on the GPU."""

    def __init__(self, batch, k, vocab, dtype=torch.float32, outright=False, counts=True, seed=0, int64=False):
        gen = torch.Generator().manual_seed(seed)
        logits = 2.0 * torch.randn((batch, k + 1, vocab), generator=gen)
        guess = torch.softmax(logits[:, :k] + 0.5 * torch.randn((batch, k, vocab), generator=gen), -1)
        self.target = torch.softmax(logits, -1).to(dtype).to(DEV)
        pick = (guess / torch.empty(guess.shape).exponential_(generator=gen)).argmax(-1) if k else guess[..., 0]
        self.tokens = (guess.argmax(-1) if outright else pick).to(torch.int64 if int64 else torch.int32).to(DEV)
        self.draft = None if outright else guess.to(dtype).to(DEV)
        self.counts = torch.randint(0, k + 1, (batch,), generator=gen, dtype=torch.int32).to(DEV) if counts else None
        self.accept_u = torch.rand((batch, k), generator=gen).to(DEV)
        self.sample_u = torch.rand((batch,), generator=gen).to(DEV)
        self.lens = torch.randint(1, 1000, (batch,), generator=gen, dtype=torch.int32).to(DEV)
        self.out = torch.full((batch, k + 1), -7, dtype=torch.int64, device=DEV)
        self.acc = torch.full((batch,), -7, dtype=torch.int32, device=DEV)
        self.next = torch.full((batch,), -7, dtype=torch.int32, device=DEV)

    def args(self, ops):
        batch, _, vocab = self.target.shape
        nbytes = ops.verify_drafts_workspace_bytes(batch, vocab)
        self.ws = torch.full((max(1, nbytes),), 0x5A, dtype=torch.uint8, device=DEV)
        return (self.target, self.draft, self.tokens, self.counts, self.accept_u, self.sample_u, self.lens, self.ws,
                self.out, self.acc, self.next)

    def check(self, ops):
        ops.verify_drafts(*self.args(ops))
        self.compare()

    def compare(self):
        torch.cuda.synchronize()
        out, acc, nxt = verify64(self.target, self.draft, self.tokens, self.counts, self.accept_u, self.sample_u,
                                 self.lens)
        assert torch.equal(self.acc.cpu(), acc)
        assert torch.equal(self.out.cpu(), out)
        assert torch.equal(self.next.cpu(), nxt)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("batch,k,vocab", [(1, 3, 1), (3, 1, 5), (5, 4, 1023), (4, 6, 1024), (7, 2, 1025),
                                           (2, 9, 4097), (33, 3, 2000), (2, 3, 65537)])
def test_matches_the_rule(gpu_ops, dtype, batch, k, vocab):
    Step(batch, k, vocab, dtype, seed=batch * 100 + k).check(gpu_ops)
    Step(batch, k, vocab, dtype, outright=True, seed=batch * 100 + k + 1, int64=True).check(gpu_ops)
    Step(batch, k, vocab, dtype, counts=False, seed=batch * 100 + k + 2).check(gpu_ops)


def test_many_pieces(gpu_ops):
    """A vocabulary of more pieces than threads of the second launch."""
    Step(2, 2, 300 * 1024 + 17, seed=3).check(gpu_ops)


def test_no_drafts_at_all(gpu_ops):
    Step(5, 0, 777, counts=False, seed=4).check(gpu_ops)
    s = Step(5, 3, 777, seed=4)
    s.counts.zero_()
    s.check(gpu_ops)
    assert s.acc.tolist() == [0] * 5


def test_63_drafts(gpu_ops):
    s = Step(2, 63, 50, counts=False, seed=5)
    s.accept_u.zero_()  # all accepted: every p is positive
    s.check(gpu_ops)
    assert s.acc.tolist() == [63, 63]


def test_counts_outside_the_range_are_clamped(gpu_ops):
    s = Step(4, 3, 100, seed=6)
    s.counts.copy_(torch.tensor([-5, 99, 2**31 - 1, -2**31]))
    s.check(gpu_ops)


@pytest.mark.parametrize("outright", [False, True])
@pytest.mark.parametrize("bad", [-1, 500, 2**31 - 1, -2**31])
def test_tokens_outside_the_vocabulary_are_refused(gpu_ops, outright, bad):
    s = Step(3, 3, 500, outright=outright, counts=False, seed=7)
    s.accept_u.zero_()
    s.tokens[1, 1] = bad
    s.check(gpu_ops)
    assert s.acc.tolist() == [3, 1, 3]


@pytest.mark.parametrize("u", [0.0, 0.5, BELOW_ONE])
def test_the_ends_of_the_unit_interval(gpu_ops, u):
    s = Step(6, 3, 3001, seed=8)
    s.target[:, :, :10] = 0.0
    s.target[:, :, -10:] = 0.0
    s.accept_u.fill_(u)
    s.sample_u.fill_(u)
    s.check(gpu_ops)


def test_ties_go_to_the_lowest_index(gpu_ops):
    """Four equal weights: a uniform on a border belongs to the next token."""
    s = Step(5, 1, 4, counts=False, seed=9)
    s.counts = torch.zeros(5, dtype=torch.int32, device=DEV)
    s.target.fill_(0.25)
    s.sample_u.copy_(torch.tensor([0.0, 0.25, 0.5, 0.75, BELOW_ONE]))
    s.check(gpu_ops)
    assert s.out[:, 0].tolist() == [0, 1, 2, 3, 3]


def test_a_refusal_that_leaves_nothing_draws_from_the_target(gpu_ops):
    s = Step(3, 2, 3000, counts=False, seed=10)
    s.draft.copy_(s.target[:, :2])  # p = q: nothing left
    s.accept_u.fill_(1.0)  # outside [0, 1): refuses q = p
    s.check(gpu_ops)
    assert s.acc.tolist() == [0, 0, 0] and bool((s.out[:, 0] >= 0).all())
    # Drafts chosen outright whose probability rounded to just under one.
    s = Step(2, 1, 40, outright=True, counts=False, seed=11)
    s.target.zero_()
    s.target[:, 0, 7] = BELOW_ONE
    s.tokens.fill_(7)
    s.accept_u.fill_(BELOW_ONE)
    s.check(gpu_ops)
    assert s.acc.tolist() == [0, 0] and s.out[:, 0].tolist() == [7, 7]


def test_rows_without_probability(gpu_ops):
    s = Step(4, 2, 2050, counts=False, seed=12)
    s.target[0] = 0.0
    s.target[1] = math.nan
    s.target[2, 0, ::2] = math.nan
    s.target[3] = -1.0
    s.check(gpu_ops)
    assert s.out[[0, 1, 3], 0].tolist() == [-1, -1, -1] and s.acc.tolist()[:2] == [0, 0]


def test_an_infinite_weight_is_drawn(gpu_ops):
    s = Step(1, 0, 2050, counts=False, seed=13)
    s.target[0, 0, 1500] = math.inf
    gpu_ops.verify_drafts(*s.args(gpu_ops))
    assert 1500 <= int(s.out[0, 0]) < 2050


def test_strided_inputs(gpu_ops):
    s = Step(4, 3, 999, seed=14)

    def spread(x, pads):
        big = torch.full([n + p for n, p in zip(x.shape, pads)], 9, dtype=x.dtype, device=DEV)
        view = big[tuple(slice(0, n) for n in x.shape)]
        view.copy_(x)
        return view

    s.target, s.draft = spread(s.target, (0, 2, 5)), spread(s.draft, (0, 1, 3))
    s.tokens, s.accept_u = spread(s.tokens, (0, 4)), spread(s.accept_u, (0, 2))
    s.out = spread(s.out, (0, 3))
    s.check(gpu_ops)


def test_lengths_move_in_place(gpu_ops):
    s = Step(4, 3, 300, seed=15)
    before = s.lens.clone()
    args = list(s.args(gpu_ops))
    args[10] = s.lens
    gpu_ops.verify_drafts(*args)
    torch.cuda.synchronize()
    assert torch.equal(s.lens, before + s.acc + 1)
    args[6] = args[10] = None  # lengths not wanted
    gpu_ops.verify_drafts(*args)


def test_the_tokens_follow_the_target(gpu_ops):
    """Many sequences with one p and q: the first token's frequencies are p's.

    A frequency of n draws is off its p by more than 5 sqrt(p (1 - p) / n) once
    in 1.7 million; ten of them stay inside."""
    n, vocab = 60000, 10
    gen = torch.Generator().manual_seed(16)
    p = torch.softmax(1.2 * torch.randn(vocab, generator=gen), 0)
    q = torch.softmax(1.2 * torch.randn(vocab, generator=gen), 0)
    s = Step(1, 1, vocab)
    s.target = p.expand(n, 2, vocab).contiguous().to(DEV)
    s.draft = q.expand(n, 1, vocab).contiguous().to(DEV)
    s.tokens = torch.multinomial(q, n, replacement=True, generator=gen).to(torch.int32)[:, None].to(DEV)
    s.counts = None
    s.accept_u, s.sample_u = torch.rand((n, 1), generator=gen).to(DEV), torch.rand((n,), generator=gen).to(DEV)
    s.lens = torch.zeros(n, dtype=torch.int32, device=DEV)
    s.out = torch.empty((n, 2), dtype=torch.int64, device=DEV)
    s.acc, s.next = torch.empty_like(s.lens), torch.empty_like(s.lens)
    gpu_ops.verify_drafts(*s.args(gpu_ops))
    got = torch.bincount(s.out[:, 0].cpu(), minlength=vocab).double() / n
    want = p.double()
    assert bool(((got - want).abs() <= 5 * (want * (1 - want) / n).sqrt()).all())


def test_on_another_stream_and_in_a_graph(gpu_ops):
    s = Step(6, 4, 5000, seed=17)
    call = gpu_ops.bind_verify_drafts(*s.args(gpu_ops))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    s.compare()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in (18, 19, 20):
        t = Step(6, 4, 5000, seed=seed)
        for name in ("target", "draft", "tokens", "counts", "accept_u", "sample_u", "lens"):
            getattr(s, name).copy_(getattr(t, name))
        s.out.fill_(-7)
        graph.replay()
        s.compare()
        t.check(gpu_ops)  # an eager call between the replays


def test_two_calls_share_nothing(gpu_ops):
    """Two calls on two streams at once, each with its own workspace."""
    a, b = Step(16, 3, 70001, seed=21), Step(16, 3, 70001, seed=22)
    ca, cb = gpu_ops.bind_verify_drafts(*a.args(gpu_ops)), gpu_ops.bind_verify_drafts(*b.args(gpu_ops))
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(5):
        with torch.cuda.stream(sa):
            ca()
        with torch.cuda.stream(sb):
            cb()
    torch.cuda.synchronize()
    a.compare()
    b.compare()

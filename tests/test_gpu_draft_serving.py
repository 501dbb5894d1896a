"""Serving steps with drafted tokens over a shared prompt, the operators together:
each step stores its tokens, attends over the shared prefix, turns the result into
probabilities, verifies the drafts and goes on from the lengths that gives; at the
end the cache is read back.  Every step's attention and verification are checked
against 64 bits, and the same steps replayed from one graph give the same."""
from __future__ import annotations

import pytest
import torch

from gpu_cases import DEV
from k8v4_v030.layout import GQA, PAGE
from test_gpu_kv_load import assert_rounded, rows64
from test_gpu_shared import Batch
from test_gpu_verify import verify64

pytestmark = pytest.mark.gpu

VOCAB, STEPS = 301, 5


class Serve:
    def __init__(self, ops, hkv, d, batch, k, prefix, ppb, seed=0):
        self.ops, self.k, self.q_len, self.ppb = ops, k, k + 1, ppb
        room = prefix % PAGE + 9 + STEPS * (k + 1)
        self.b = Batch(ops, hkv, d, k + 1, prefix, [room + 11 * i for i in range(batch)], ppb=ppb, seed=seed)
        self.start = [n - STEPS * (k + 1) for n in self.b.lens]  # the rest of each table is for the steps
        gen = torch.Generator().manual_seed(seed + 1)
        rand = lambda *s: torch.randn(s, generator=gen).to(DEV)  # noqa: E731
        self.embed_q, self.embed_k, self.embed_v = (rand(VOCAB, h, d).half() for h in (GQA * hkv, hkv, hkv))
        self.head = rand(7 * d, VOCAB) * 0.2  # of seven of the query heads
        self.guess = torch.softmax(3.0 * rand(VOCAB, VOCAB), -1)
        self.accept_u = torch.rand((STEPS, batch, k), generator=gen).to(DEV)
        self.sample_u = torch.rand((STEPS, batch), generator=gen).to(DEV)
        self.raw0 = self.b.cache.raw.clone()
        self.verify_ws = torch.empty(ops.verify_drafts_workspace_bytes(batch, VOCAB) or 1, dtype=torch.uint8, device=DEV)
        new = lambda *s, t=torch.int32: torch.zeros(s, dtype=t, device=DEV)  # noqa: E731
        self.lens, self.next_lens, self.accepted = new(batch), new(batch), new(batch)
        self.step_lens, self.last = new(batch), new(batch, t=torch.int64)
        self.out_tokens, self.tokens = new(batch, k + 1, t=torch.int64), new(batch, k + 1, t=torch.int64)
        self.u, self.su = new(batch, k, t=torch.float32), new(batch, t=torch.float32)
        self.attn = torch.empty((batch * (k + 1), GQA * hkv, d), dtype=torch.float32, device=DEV)
        self.q = torch.empty(self.attn.shape, dtype=torch.float16, device=DEV)
        self.draft = torch.empty((batch, k, VOCAB), device=DEV)
        self.target = torch.empty((batch, k + 1, VOCAB), device=DEV)

    def reset(self):
        self.b.cache.raw.copy_(self.raw0)
        self.lens.copy_(torch.tensor(self.start, dtype=torch.int32))
        self.last.copy_(torch.arange(self.b.batch) * 7 % VOCAB)

    def step(self):
        b, ops = self.b, self.ops
        chain = [self.last]
        for j in range(self.k):  # the draft model: one table row per token
            self.draft[:, j] = self.guess[chain[-1]]
            chain.append(self.draft[:, j].argmax(-1))
        self.tokens.copy_(torch.stack(chain, 1))
        at = self.lens.long()[:, None] + torch.arange(self.q_len, device=DEV)
        page = at // PAGE
        slots = (b.table_dev.long().gather(1, page // self.ppb) * self.ppb + page % self.ppb) * PAGE + at % PAGE
        flat = self.tokens.flatten()
        b.cache.store(ops, self.embed_k[flat], self.embed_v[flat], slots.flatten())
        self.q.copy_(self.embed_q[flat])
        torch.add(self.lens, self.q_len, out=self.step_lens)
        ops.int8k_int4v_attn_shared(self.q, *b.cache.region_args(), b.prefix_dev, b.prefix, b.table_dev,
                                    self.step_lens, b.ws, self.attn, self.q_len, self.ppb)
        # The draft model is near the target: its logits and the attention's.
        logits = self.attn[:, :7].flatten(1) @ self.head + self.guess[flat].log()
        self.target.copy_(torch.softmax(logits, -1).view(self.target.shape))
        ops.verify_drafts(self.target, self.draft, self.tokens[:, 1:].contiguous(), None, self.u, self.su, self.lens,
                          self.verify_ws, self.out_tokens, self.accepted, self.next_lens)
        self.last.copy_(self.out_tokens.gather(1, self.accepted.long()[:, None]).flatten())
        self.lens.copy_(self.next_lens)

    def run(self, go, after):
        """``go()`` once per step; ``after(lens before)`` checks it.  The tokens each sequence kept."""
        self.reset()
        kept = [[] for _ in range(self.b.batch)]
        states = []
        for s in range(STEPS):
            self.u.copy_(self.accept_u[s])
            self.su.copy_(self.sample_u[s])
            lens = self.lens.clone()
            go()
            torch.cuda.synchronize()
            after(lens)
            for i, a in enumerate(self.accepted.tolist()):
                kept[i] += self.tokens[i, : a + 1].tolist()
            states.append([x.clone() for x in (self.attn, self.target, self.out_tokens, self.accepted, self.lens)])
        return kept, states

    def check(self, lens):
        b = self.b
        b.q, b.lens = self.q, (lens + self.q_len).tolist()
        b.check(self.attn)
        out, acc, nxt = verify64(self.target, self.draft, self.tokens[:, 1:], None, self.u, self.su, lens)
        assert torch.equal(self.out_tokens.cpu(), out)
        assert torch.equal(self.accepted.cpu(), acc) and torch.equal(self.lens.cpu(), nxt.to(torch.int32))

    def read_back(self, kept):
        """Every sequence's tokens behind the start, loaded: what the formula gives, and the kept tokens' own rows."""
        b = self.b
        counts = [len(t) for t in kept]
        assert [s + n for s, n in zip(self.start, counts)] == self.lens.tolist()
        rows = torch.tensor([0, *torch.tensor(counts).cumsum(0).tolist()], dtype=torch.int32, device=DEV)
        shape = (sum(counts), b.hkv, b.d)
        k_out, v_out = (torch.empty(shape, dtype=torch.float32, device=DEV) for _ in range(2))
        self.ops.kv_load_paged(*b.cache.region_args(), b.table_dev, torch.tensor(self.start, dtype=torch.int32, device=DEV),
                               rows, self.ppb, k_out, v_out)
        torch.cuda.synchronize()
        k64, v64 = rows64(b.cache, b.table, self.ppb, self.start, counts)
        assert_rounded(k_out, k64, 1)
        flat = torch.tensor([t for seq in kept for t in seq], device=DEV)
        stored = self.embed_k[flat].double()
        # Half a step of the int8 code (amax / 127) and the fp32 roundings of scale, quotient and product.
        step = stored.abs().amax(-1, keepdim=True) / 127.0
        assert bool(((k_out.double() - stored).abs() <= step * (0.5 + 127 * 4 * 2.0**-24)).all())
        stored = self.embed_v[flat].double()
        # Half a step of 15, and half of one for the rounded zero point.
        step = (stored.amax(-1, keepdim=True) - stored.amin(-1, keepdim=True)) / 15.0
        assert bool(((v_out.double() - stored).abs() <= step * (1 + 2.0**-10)).all())
        assert bool(((v_out.cpu().double() - v64).abs() <= 2.0**-22 * (v64.abs() + 16 * step.cpu())).all())


@pytest.mark.parametrize("hkv,d,batch,k,prefix,ppb", [(2, 128, 5, 3, 200, 1), (4, 256, 3, 1, 64 * 6, 2), (4, 128, 40, 4, 700, 1)])
def test_steps_together(gpu_ops, hkv, d, batch, k, prefix, ppb):
    s = Serve(gpu_ops, hkv, d, batch, k, prefix, ppb)
    kept, eager = s.run(s.step, s.check)
    assert any(len(t) > STEPS for t in kept)  # drafts were accepted somewhere
    s.read_back(kept)

    s.reset()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        s.step()  # warm-up outside the graph
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.step()
    kept2, replayed = s.run(graph.replay, s.check)
    assert kept2 == kept
    for a, b in zip(eager, replayed):
        for x, y in zip(a[2:], b[2:]):
            assert torch.equal(x, y)
        assert torch.equal(a[0], b[0])
    s.read_back(kept2)

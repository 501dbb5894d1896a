"""Decode steps of the vLLM backend whose requests share a prefix, on the GPU: the
step reads it once and matches softmax attention in 64 bits (tolerances:
test_gpu_shared.py), beside prefills and captured too."""
from __future__ import annotations

import pytest
import torch

from backend_cases import common_metadata, make_builder, make_impl
from gpu_cases import DEV
from k8v4_v030 import plan
from k8v4_v030.layout import PAGE
from k8v4_v030.scratch import clear_scratch
from test_gpu_shared import Batch

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def own_scratch():
    clear_scratch()
    yield
    clear_scratch()


@pytest.fixture
def calls(gpu_ops, monkeypatch):
    """Which of the two decode ops ran, with the query length."""
    seen = []
    for name in ("int8k_int4v_attn_shared", "int8k_int4v_attn_batch"):
        real = getattr(type(gpu_ops), name)

        def spy(self, *a, _real=real, _name=name, **kw):
            seen.append(_name)
            return _real(self, *a, **kw)

        monkeypatch.setattr(type(gpu_ops), name, spy)
    return seen


class Served(Batch):
    """A Batch the way the engine serves it: every request's table begins with the prefix."""

    def __init__(self, *args, **kw):
        super().__init__(*args, **kw)
        same = self.shared // (PAGE * self.ppb)
        assert same * PAGE * self.ppb == self.prefix  # the engine's prefixes are whole blocks
        self.table[:, :same] = self.prefix_table[:same]
        self.table_dev = self.table.to(DEV)
        lay = self.cache.layout
        self.kv = self.cache.raw.view(-1, lay.hkv, PAGE * self.ppb, lay.slot_bytes_per_head)
        self.impl = make_impl(self.hkv, self.d)
        self.builder = make_builder(self.hkv, self.d, block_size=PAGE * self.ppb, kernel_block=None, device=DEV,
                                    max_model_len=self.table.shape[1] * self.ppb * PAGE, max_seqs=self.batch)

    def meta(self, prefix, q_lens=None):
        q_lens = q_lens or [self.q_len] * self.batch
        return self.builder.build(prefix, common_metadata(q_lens, self.lens, self.table,
                                                          torch.zeros(sum(q_lens), dtype=torch.int64), DEV))

    def forward(self, meta, out_dtype=torch.float32):
        out = torch.full(self.q.shape, float("nan"), dtype=out_dtype, device=DEV)
        self.impl.forward(None, self.q, None, None, self.kv, meta, out)
        torch.cuda.synchronize()
        return out


@pytest.mark.parametrize("hkv,d,q_len,ppb,batch,prefix_blocks", [
    (4, 128, 1, 1, 5, 9), (4, 128, 7, 2, 3, 4), (2, 128, 10, 1, 6, 3), (4, 256, 2, 33, 3, 1), (2, 256, 4, 1, 26, 5),
    (4, 128, 3, 1, 70, 2)])
def test_step_over_a_shared_prefix(gpu_ops, calls, monkeypatch, hkv, d, q_len, ppb, batch, prefix_blocks):
    monkeypatch.setattr(plan, "SHARED_PREFIX_MIN_SAVED", 1)
    own = [q_len + (37 * i) % 150 for i in range(batch)]
    b = Served(gpu_ops, hkv, d, q_len, prefix_blocks * ppb * PAGE, own, ppb=ppb, dtype=torch.bfloat16, seed=batch)
    meta = b.meta(b.prefix)
    for dtype in (torch.float32, torch.bfloat16):
        b.check(b.forward(meta, dtype))
    assert calls == ["int8k_int4v_attn_shared"] * 2
    b.check(b.forward(b.meta(0)))  # the same step without it
    assert calls[2:] == ["int8k_int4v_attn_batch"]


def test_the_shapes_that_pay_use_it_by_themselves(gpu_ops, calls):
    b = Served(gpu_ops, 2, 128, 1, 280 * PAGE, [1 + i for i in range(32)], seed=1)
    assert b.builder.use_cascade_attention(b.prefix, [1] * 32)
    b.check(b.forward(b.meta(b.prefix)))
    assert calls == ["int8k_int4v_attn_shared"]
    b = Served(gpu_ops, 2, 128, 1, 10 * PAGE, [1 + i for i in range(32)], seed=1)
    assert not b.builder.use_cascade_attention(b.prefix, [1] * 32)
    b.check(b.forward(b.meta(b.prefix)))
    assert calls[1:] == ["int8k_int4v_attn_batch"]


def test_prefills_and_other_runs_beside_it(gpu_ops, calls, monkeypatch):
    """Runs of 1 and of 3 query tokens and two prefills, all behind one prefix: the
    decode rows agree with 64 bits, the prefill rows are those of a step without a prefix."""
    monkeypatch.setattr(plan, "SHARED_PREFIX_MIN_SAVED", 1)
    q_lens = [1, 1, 1, 3, 3, 40, 25]
    first = sum(q_lens[:5])
    b = Served(gpu_ops, 4, 128, 1, 5 * PAGE, [50 + 3 * n for n in q_lens], seed=3)
    b.q = torch.randn((sum(q_lens), 24, 128), generator=torch.Generator().manual_seed(4)).half().to(DEV)
    got, plain = b.forward(b.meta(b.prefix, q_lens)), b.forward(b.meta(0, q_lens))
    assert calls == ["int8k_int4v_attn_shared"] * 2 + ["int8k_int4v_attn_batch"] * 2
    assert torch.equal(got[first:], plain[first:])
    rows, lens, table = b.q, b.lens, b.table_dev
    for out in (got, plain):
        for q_len, lo, hi, row in ((1, 0, 3, 0), (3, 3, 5, 3)):
            n = (hi - lo) * q_len
            b.q, b.q_len, b.batch = rows[row : row + n], q_len, hi - lo
            b.lens, b.table_dev = lens[lo:hi], table[lo:hi]
            b.check(out[row : row + n])


def test_a_captured_step_reads_each_requests_own_table(gpu_ops, calls, monkeypatch):
    """A graph's replays may be steps of other prefixes, or none."""
    monkeypatch.setattr(plan, "SHARED_PREFIX_MIN_SAVED", 1)
    b = Served(gpu_ops, 4, 128, 2, 4 * PAGE, [70, 5, 200], seed=5)
    meta = b.meta(b.prefix)
    b.forward(meta)
    out = torch.zeros(b.q.shape, dtype=torch.float32, device=DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        b.impl.forward(None, b.q, None, None, b.kv, meta, out)
    assert calls == ["int8k_int4v_attn_shared", "int8k_int4v_attn_batch"]
    spare = next(p for p in range(b.cache.num_pages) if p not in set(b.table.flatten().tolist()))
    for step in range(3):
        if step == 1:  # the second request leaves the prefix
            b.cache.raw.view(b.cache.num_pages, -1)[spare] = b.cache.raw.view(b.cache.num_pages, -1)[int(b.table[1, 4])]
            meta.block_table[1, 0] = spare
        graph.replay()
        torch.cuda.synchronize()
        table = meta.block_table.clone()
        want = b.forward(b.builder.build(0, common_metadata([2] * 3, b.lens, table, torch.zeros(6), DEV)))
        assert torch.equal(out, want)


def test_the_workspace_is_not_made_inside_a_capture(gpu_ops):
    from k8v4_v030.scratch import get_scratch

    b = Served(gpu_ops, 4, 128, 1, PAGE, [3, 4], seed=6)
    b.meta(0)  # the first step makes the scratch
    scratch = get_scratch(torch.device(DEV), b.builder.layout)
    x = torch.zeros(8, device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x.add_(1)
        with pytest.raises(RuntimeError, match="not allocated before capture"):
            scratch.shared_ws()
    graph.replay()
    torch.cuda.synchronize()
    assert float(x[0]) == 1.0

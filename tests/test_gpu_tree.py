"""int8k_int4v_attn_tree against softmax attention in 64 bits.

Tolerance, per output element with a = sum of p |v| over the row's keys and o
the result: the kernels round to fp16 a key's probability, its V scale and their
product, or its dequantized V (2^-11 each, on a); the row sum's probabilities (2^-11,
on o); and a page run's output (2^-11, on a); scores are off by at most 0.75 q_scale
k_scale / sqrt(D), 1e-4 of a probability here, which a quarter of 2^-11 covers; the
output rounds by half a step of its type.  Where the matrix products sum whole V bytes
(at most 255 of a V step) the zero point's share comes off at the end: each chunk of
32 keys rounds the running sum once, by at most 2^-24 of it, and c such roundings of
either sign add up to at most 4 sqrt(c) of one (four standard deviations).
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from gpu_cases import Cache, DEV, decode, fill_sequence
from k8v4_v030.layout import GQA, PAGE, PageLayout
from k8v4_v030.plan import tree_masks

pytestmark = pytest.mark.gpu


def random_parents(rng, nodes):
    return [-1] + [rng.randrange(max(0, i - 7), i) for i in range(1, nodes)]


class Trees:
    """``contexts``: tokens ahead of each sequence's tree (negative: the sequence is that
    much shorter than its tree; None: no tokens at all)."""

    def __init__(self, ops, hkv, d, nodes, contexts, ppb=1, dtype=torch.float16, seed=0, fused=False, masks=None):
        self.ops, self.hkv, self.d, self.nodes, self.ppb, self.batch = ops, hkv, d, nodes, ppb, len(contexts)
        self.lens = [0 if c is None else max(0, c + nodes) for c in contexts]
        gen, rng = torch.Generator().manual_seed(seed), random.Random(seed)
        need = [max(1, -(-n // (PAGE * ppb))) for n in self.lens]
        perm = torch.randperm(sum(need) + 3, generator=gen).to(torch.int32)
        self.cache = Cache(perm.shape[0] * ppb, PageLayout(hkv, d))
        self.cache.raw.fill_(-1)  # what is not stored holds NaN planes
        self.table = torch.full((self.batch, max(need)), -1, dtype=torch.int32)
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at : at + n]
            at += n
            fill_sequence(ops, self.cache, gen, self.table[b], self.lens[b], ppb)
        if masks is None:
            masks = [tree_masks(random_parents(rng, nodes)) for _ in contexts]
        self.masks = torch.tensor(masks, dtype=torch.int64)
        rows = torch.randn((self.batch * nodes, GQA * hkv, d), generator=gen).to(dtype).to(DEV)
        if fused:
            buf = torch.zeros((rows.shape[0], (GQA + 2) * hkv * d), dtype=dtype, device=DEV)
            buf[:, : GQA * hkv * d] = rows.flatten(1)
            rows = buf[:, : GQA * hkv * d].unflatten(1, (GQA * hkv, d))
        self.q = rows
        nbytes = ops.attn_tree_workspace_bytes(self.batch, nodes, hkv, d)
        self.ws = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=DEV)  # NaN patterns
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        self.table_dev, self.masks_dev = self.table.to(DEV), self.masks.to(DEV)

    def bind(self, out):
        return self.ops.bind_int8k_int4v_attn_tree(self.q, *self.cache.region_args(), self.table_dev, self.lens_dev,
                                                   self.masks_dev, self.ws, out, self.nodes, self.ppb)

    def run(self, out_dtype=torch.float16):
        out = torch.full(self.q.shape, math.nan, dtype=out_dtype, device=DEV)
        self.bind(out)()
        torch.cuda.synchronize()
        return out

    def rows64(self, b):
        """float64 K and V rows of sequence b and which of them exist (their page is in the cache)."""
        n = min(self.lens[b], self.table.shape[1] * self.ppb * PAGE)
        t = torch.arange(n, device=DEV)
        page = t // PAGE
        phys = self.table_dev[b][page // self.ppb].long() * self.ppb + page % self.ppb
        there = (phys >= 0) & (phys < self.cache.num_pages)
        phys, r = torch.where(there, phys, 0), t % PAGE
        v_ = self.cache.views
        k = v_["k"][phys, r].double() * v_["k_scale"][phys, r].double()[..., None]
        byte = v_["v"][phys, r]
        nib = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).double()
        v = (nib - v_["v_zero"][phys, r].double()[..., None]) * v_["v_scale"][phys, r].double()[..., None]
        return torch.where(there[:, None, None], k, 0), torch.where(there[:, None, None], v, 0), there

    def want(self):
        """(o, a, r): the result, the sums of p |v| and the fp32 sums' roundings, float64."""
        q = self.q.double()
        # By a tensor: torch multiplies by the reciprocal of a Python number, an ulp off.
        scale = q.abs().amax(-1, keepdim=True) / torch.full((), 127.0, dtype=torch.float64, device=DEV)
        inv = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
        q = torch.sign(q) * torch.floor(q.abs() * inv + 0.5) * scale
        o, a = torch.zeros_like(q), torch.zeros_like(q)
        r = torch.zeros(q.shape[0], 1, 1, dtype=torch.float64, device=DEV)
        n = self.nodes
        for b in range(self.batch):
            if self.lens[b] == 0:
                continue
            k, v, there = self.rows64(b)
            node = torch.arange(k.shape[0], device=DEV) - (self.lens[b] - n)
            bits = (self.masks_dev[b][:, None] >> node.clamp(0, 63)[None]) & 1
            hidden = ((node[None] >= 0) & (bits == 0)) | ~there[None]
            hidden = hidden.repeat_interleave(GQA, 0)
            rows = slice(b * n, (b + 1) * n)
            step = max(float(self.cache.views["v_scale"].nan_to_num(0.0).max()), 1e-30)
            r[rows] = 4 * math.sqrt(-(-k.shape[0] // 32)) * 255 * step * 2.0**-24
            for h in range(self.hkv):
                heads = slice(h * GQA, (h + 1) * GQA)
                s = torch.mm(q[rows, heads].reshape(-1, self.d), k[:, h].t().contiguous()) / math.sqrt(self.d)
                p = torch.softmax(s.masked_fill(hidden, -math.inf), 1).nan_to_num(0.0)
                o[rows, heads] = torch.mm(p, v[:, h].contiguous()).view(n, GQA, self.d)
                a[rows, heads] = torch.mm(p, v[:, h].abs().contiguous()).view(n, GQA, self.d)
        return o, a, r

    def check(self, out, want=None):
        o, a, r = want or self.want()
        got = out.double()
        assert bool(torch.isfinite(got).all())
        eps = torch.finfo(out.dtype).eps / 2
        tol = 4.25 * 2.0**-11 * a + (2.0**-11 + eps) * o.abs() + r
        err = (got - o).abs()
        assert bool((err <= tol).all()), "max error %.3g, %.3g of the tolerance" % (
            float(err.max()), float((err / tol).nan_to_num(0.0).max()))


SHAPES = [(4, 128), (2, 128), (2, 256), (4, 256)]


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes,contexts", [
    (1, [0, 1, 63, 64, 500]), (3, [0, 200, None, 61, 62]), (7, [5, 4000, 57, 58, 60]), (8, [56, 900, None, 0, 55]),
    (9, [2048, None, 55, 1]), (16, [640, 0, 3000]), (17, [47, 48, 1000, 4097]), (21, [2048, 43]), (22, [2048, 42, 0]),
    (42, [300, 22, 0, 700]), (43, [5000]), (64, [0, 1, 64, 1500, None]),
])
def test_trees(gpu_ops, hkv, d, nodes, contexts):
    st = Trees(gpu_ops, hkv, d, nodes, contexts, seed=nodes)
    st.check(st.run())


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes", [4, 13, 30, 64])
def test_types_blocks_and_fused_rows(gpu_ops, hkv, d, nodes):
    st = Trees(gpu_ops, hkv, d, nodes, [3000, 17, 2112, 6000 - nodes], ppb=33, dtype=torch.bfloat16, seed=nodes + 1, fused=True)
    for out_dtype in (torch.bfloat16, torch.float32, torch.float16):
        st.check(st.run(out_dtype))


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes", [6, 25, 50])
def test_shorter_than_their_trees(gpu_ops, hkv, d, nodes):
    """Nodes before the first token do not exist: a row may see nothing."""
    st = Trees(gpu_ops, hkv, d, nodes, [-1, 1 - nodes, 2 - nodes, -nodes // 2, 100], seed=nodes + 2)
    st.check(st.run())


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes", [5, 19, 64])
def test_masks_of_any_bits(gpu_ops, hkv, d, nodes):
    """Empty words, words with every bit (those from `nodes` on are ignored), random ones
    without the node's own bit."""
    rng = random.Random(nodes)
    signed = lambda w: w - (1 << 64) if w >> 63 else w  # noqa: E731
    contexts = [0, 0, 30, 700, 63]
    masks = [[0] * nodes, [-1] * nodes, [0] * nodes, [signed(rng.getrandbits(64)) for _ in range(nodes)],
             [signed(rng.getrandbits(64) & ~(1 << j)) for j in range(nodes)]]
    st = Trees(gpu_ops, hkv, d, nodes, contexts, seed=nodes + 3, masks=masks)
    out = st.run()
    st.check(out)
    assert not out[:nodes].any()  # no context, no nodes


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes", [1, 7, 10])
def test_a_chain_is_the_batch_op(gpu_ops, hkv, d, nodes):
    """The chain's masks against the batch op's causal rule, both within the tolerance."""
    st = Trees(gpu_ops, hkv, d, nodes, [700, 64, 0, 3000], seed=nodes + 4,
               masks=[[(2 << j) - 1 for j in range(nodes)]] * 4)
    out = st.run(torch.float32)
    st.check(out)
    st.check(decode(gpu_ops, st.cache, st.q, st.table, st.lens_dev, nodes, out_dtype=torch.float32))


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 256)])
def test_one_tree_for_all_and_pages_outside(gpu_ops, hkv, d):
    rng = random.Random(1)
    words = tree_masks(random_parents(rng, 27))
    st = Trees(gpu_ops, hkv, d, 27, [900, 400, 64, 2000], seed=5, masks=[words] * 4)
    st.masks_dev = st.masks_dev[:1].expand(4, 27)
    st.check(st.run())
    for entry, bad in ((0, -1), (1, st.cache.num_pages), (3, 2**31 - 1), (0, -2**31), (14, -5)):
        st.table[rng.randrange(4), min(entry, st.table.shape[1] - 1)] = bad
    st.table_dev = st.table.to(DEV)
    st.check(st.run())


def test_a_table_shorter_than_the_sequence(gpu_ops):
    """Tokens behind the table's last page are not attended to."""
    st = Trees(gpu_ops, 4, 128, 12, [300, 500], seed=6)
    st.table_dev = st.table_dev[:, :5].contiguous()
    st.table = st.table[:, :5]
    st.check(st.run())


def test_a_padding_sequence_may_hold_anything(gpu_ops):
    st = Trees(gpu_ops, 4, 128, 20, [600, None, 70], seed=7)
    st.q[20:40] = math.nan
    st.masks_dev[1] = -1
    out = st.run()
    assert not out[20:40].any()
    st.q[20:40] = 0
    st.check(out)


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes", [6, 20, 50, 64])
def test_nodes_that_nobody_sees_need_not_be_stored(gpu_ops, hkv, d, nodes):
    """Trees of fewer nodes than the call's: the cache may hold NaN at the others."""
    rng = random.Random(nodes)
    real = [nodes // 2, 1, nodes - 1, nodes]
    masks = [tree_masks(random_parents(rng, n)) + [0] * (nodes - n) for n in real]
    for words in masks:
        words[-1] = words[0] if words[-1] == 0 else words[-1]  # an absent node's row may see stored ones
    st = Trees(gpu_ops, hkv, d, nodes, [500, 64 - real[1], 0, 3000], seed=nodes + 5, masks=masks)
    want = st.want()
    for b, n in enumerate(real):
        t = torch.arange(st.lens[b] - nodes + n, st.lens[b])
        page, row = st.table[b][t // PAGE].long().to(DEV), (t % PAGE).to(DEV)
        for name in ("k_scale", "v_scale", "v_zero"):
            st.cache.views[name][page, row] = math.nan
    st.check(st.run(), want)


def test_large_values(gpu_ops):
    """V rows of the whole fp16 range stay finite."""
    st = Trees(gpu_ops, 4, 128, 24, [200, 0], seed=8)
    for b in range(2):
        t = torch.arange(st.lens[b])
        slots = (st.table[b][t // PAGE].long() * PAGE + t % PAGE).to(DEV)
        k = torch.randn((st.lens[b], 4, 128), device=DEV, dtype=torch.float16)
        v = torch.where(torch.rand((st.lens[b], 4, 128), device=DEV) < 0.5, -65504.0, 65504.0).half()
        st.cache.store(gpu_ops, k, v, slots)
    st.check(st.run(torch.float32))


@pytest.mark.parametrize("nodes", [6, 26, 64])
def test_captured_and_replayed(gpu_ops, nodes):
    """Lengths, tables, masks and queries change between replays; eager work in between."""
    st = Trees(gpu_ops, 4, 128, nodes, [1500, 800, 2000], seed=9)
    out = torch.full(st.q.shape, math.nan, dtype=torch.float16, device=DEV)
    call = st.bind(out)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    rng = random.Random(2)
    for k in range(4):
        st.lens = [rng.randrange(nodes, n + 1) for n in (1500 + nodes, 800 + nodes, 2000 + nodes)]
        if k == 2:
            st.lens[1] = 0
        st.lens_dev.copy_(torch.tensor(st.lens, dtype=torch.int32))
        st.masks_dev.copy_(torch.tensor([tree_masks(random_parents(rng, nodes)) for _ in range(3)]))
        st.q.normal_()
        out.fill_(math.nan)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        st.check(out)
        eager = st.run()
        assert torch.equal(eager, out)


def test_two_streams_with_their_own_workspaces(gpu_ops):
    a = Trees(gpu_ops, 4, 128, 33, [4000, 100], seed=10)
    b = Trees(gpu_ops, 2, 256, 9, [3000, 700, 50], seed=11)
    outs = [torch.full(x.q.shape, math.nan, dtype=torch.float32, device=DEV) for x in (a, b)]
    calls = [a.bind(outs[0]), b.bind(outs[1])]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for call, stream in zip(calls, streams):
            with torch.cuda.stream(stream):
                call()
    torch.cuda.synchronize()
    a.check(outs[0])
    b.check(outs[1])


@pytest.mark.parametrize("seed", range(24))
def test_random_shapes(gpu_ops, seed):
    rng = random.Random(1000 + seed)
    hkv, d = rng.choice(SHAPES)
    nodes = rng.randint(1, 64)
    contexts = [None if rng.random() < 0.1 else int(10 ** rng.uniform(0, 3.6)) - 1 for _ in range(rng.randint(1, 9))]
    st = Trees(gpu_ops, hkv, d, nodes, contexts, ppb=rng.choice((1, 1, 3, 33)), seed=seed,
               dtype=rng.choice((torch.float16, torch.bfloat16)), fused=rng.random() < 0.5)
    st.check(st.run(rng.choice((torch.float16, torch.bfloat16, torch.float32))))

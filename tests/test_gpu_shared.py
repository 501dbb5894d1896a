"""int8k_int4v_attn_shared against softmax attention in 64 bits.

Tolerance, per output element with a = sum of p |v| over the row's keys and o
the result: the kernel rounds to fp16 a key's probability, its V scale and
their product (2^-11 each, on a), the row sum's probabilities (2^-11, on o) and
a page run's output (2^-11, on a); scores are off by at most 0.75 q_scale
k_scale / sqrt(D), 1e-4 of a probability here, which a quarter of 2^-11
covers; the output rounds by half a step of its type.

The matrix products sum whole V bytes (16 high + low nibble, at most 255 of a V
step) in fp32 and take the zero point's share off at the end, so a value near
zero is the difference of two sums of up to 255 s, s the row's largest V scale:
each chunk of 32 keys rounds the running sum once, by at most 2^-24 of it, and c
such roundings of either sign add up to at most 4 sqrt(c) of one (four standard
deviations).  (A head's row of two keys whose nibble is the zero point gives
-7.4e-6 for 0, through this op and the batch op alike: 255 * 0.35 * 2^-24 is
5.3e-6.)
"""
from __future__ import annotations

import math
import random

import pytest
import torch

from gpu_cases import Cache, DEV, decode, fill_sequence
from k8v4_v030.layout import GQA, PAGE, PageLayout

pytestmark = pytest.mark.gpu


class Batch:
    """A cache whose sequences share their first pages, and one step's queries.

    ``own`` are the tokens of each sequence behind the prefix's whole pages (a
    negative number takes tokens off the prefix, None is an empty sequence)."""

    def __init__(self, ops, hkv, d, q_len, prefix, own, ppb=1, dtype=torch.float16, seed=0, fused=False):
        self.ops, self.hkv, self.d, self.q_len, self.ppb = ops, hkv, d, q_len, ppb
        self.prefix, self.batch = prefix, len(own)
        self.shared = prefix // PAGE * PAGE
        self.lens = [0 if n is None else max(0, self.shared + n) for n in own]
        gen = torch.Generator().manual_seed(seed)
        blk = PAGE * ppb
        head = -(-max(prefix, 1) // blk)
        same = self.shared // blk
        need = [max(1, -(-n // blk)) for n in self.lens]
        pool = head + sum(max(0, n - same) for n in need) + 3
        perm = torch.randperm(pool, generator=gen).to(torch.int32)
        self.cache = Cache(pool * ppb, PageLayout(hkv, d))
        self.prefix_table = perm[:head].clone()
        self.table = torch.full((self.batch, max(need)), -1, dtype=torch.int32)
        at = head
        fill_sequence(ops, self.cache, gen, self.prefix_table, max(prefix, 1), ppb)
        for b, n in enumerate(need):
            fresh = max(0, n - same)
            self.table[b, same:n] = perm[at : at + fresh]
            at += fresh
            if self.lens[b] > self.shared:
                # A block that the prefix ends inside: the shared pages of it are the sequence's own copy,
                # which the op does not read; other tokens than the prefix's are stored there.
                fill_sequence(ops, self.cache, gen, self.table[b], self.lens[b], ppb, start=same * blk)
        rows = torch.randn((self.batch * q_len, GQA * hkv, d), generator=gen).to(dtype).to(DEV)
        if fused:
            buf = torch.zeros((rows.shape[0], (GQA + 2) * hkv * d), dtype=dtype, device=DEV)
            buf[:, : GQA * hkv * d] = rows.flatten(1)
            rows = buf[:, : GQA * hkv * d].unflatten(1, (GQA * hkv, d))
        self.q = rows
        nbytes = ops.attn_shared_workspace_bytes(self.batch, q_len, hkv, d)
        self.ws = torch.full((nbytes,), 0xFF, dtype=torch.uint8, device=DEV)  # NaN patterns
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        self.table_dev, self.prefix_dev = self.table.to(DEV), self.prefix_table.to(DEV)

    def bind(self, out, q=None):
        return self.ops.bind_int8k_int4v_attn_shared(
            self.q if q is None else q, *self.cache.region_args(), self.prefix_dev, self.prefix, self.table_dev,
            self.lens_dev, self.ws, out, self.q_len, self.ppb)

    def run(self, out_dtype=torch.float16):
        out = torch.full(self.q.shape, math.nan, dtype=out_dtype, device=DEV)
        self.bind(out)()
        torch.cuda.synchronize()
        return out

    def rows64(self, b):
        """float64 K and V rows of sequence b and which of them exist (their page is in the cache)."""
        n = min(self.lens[b], max(self.shared, self.table.shape[1] * self.ppb * PAGE))
        t = torch.arange(n, device=DEV)
        page = t // PAGE
        entry = page // self.ppb
        own = self.table_dev[b][entry.clamp(max=self.table.shape[1] - 1)]
        pre = self.prefix_dev[entry.clamp(max=self.prefix_dev.shape[0] - 1)]
        phys = torch.where(t < self.shared, pre, own).long() * self.ppb + page % self.ppb
        there = (phys >= 0) & (phys < self.cache.num_pages)
        phys, r = torch.where(there, phys, 0), t % PAGE
        v_ = self.cache.views
        k = v_["k"][phys, r].double() * v_["k_scale"][phys, r].double()[..., None]
        byte = v_["v"][phys, r]
        nib = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).double()
        v = (nib - v_["v_zero"][phys, r].double()[..., None]) * v_["v_scale"][phys, r].double()[..., None]
        return k, v, there

    def want(self):
        """(o, a, r): the result, the sums of p |v| and the fp32 sums' roundings, float64."""
        q = self.q.double()
        # By a tensor: torch multiplies by the reciprocal of a Python number, an ulp off, and a
        # query value on a rounding tie (bf16 with amax 127 / 64, say) gets the other code.
        scale = q.abs().amax(-1, keepdim=True) / torch.full((), 127.0, dtype=torch.float64, device=DEV)
        inv = torch.where(scale == 0, torch.zeros_like(scale), 1.0 / scale)
        q = torch.sign(q) * torch.floor(q.abs() * inv + 0.5) * scale
        o, a = torch.zeros_like(q), torch.zeros_like(q)
        r = torch.zeros(q.shape[0], 1, 1, dtype=torch.float64, device=DEV)
        for b in range(self.batch):
            if self.lens[b] == 0:
                continue
            k, v, there = self.rows64(b)
            t = torch.arange(k.shape[0], device=DEV)
            end = self.lens[b] - self.q_len + 1 + torch.arange(self.q_len, device=DEV).repeat_interleave(GQA)
            hidden = (t[None] >= end[:, None]) | ~there[None]
            rows = slice(b * self.q_len, (b + 1) * self.q_len)
            step = max(float(self.cache.views["v_scale"].nan_to_num(0.0).max()), 1e-30)
            r[rows] = 4 * math.sqrt(-(-k.shape[0] // 32)) * 255 * step * 2.0**-24
            for h in range(self.hkv):
                heads = slice(h * GQA, (h + 1) * GQA)
                s = torch.mm(q[rows, heads].reshape(-1, self.d), k[:, h].t().contiguous()) / math.sqrt(self.d)
                p = torch.softmax(s.masked_fill(hidden, -math.inf), 1).nan_to_num(0.0)
                o[rows, heads] = torch.mm(p, v[:, h].contiguous()).view(self.q_len, GQA, self.d)
                a[rows, heads] = torch.mm(p, v[:, h].abs().contiguous()).view(self.q_len, GQA, self.d)
        return o, a, r

    def check(self, out):
        o, a, r = self.want()
        got = out.double()
        assert bool(torch.isfinite(got).all())
        eps = torch.finfo(out.dtype).eps / 2
        tol = 4.25 * 2.0**-11 * a + (2.0**-11 + eps) * o.abs() + r
        err = (got - o).abs()
        assert bool((err <= tol).all()), "max error %.3g, %.3g of the tolerance" % (
            float(err.max()), float((err / tol).max()))
        empty = torch.tensor([[n - self.q_len + j + 1 <= 0 for j in range(self.q_len)] for n in self.lens]).flatten()
        assert not bool(got[empty.to(DEV)].any())


CASES = [
    # hkv, D, q_len, prefix, own tokens, pages per entry
    (4, 128, 1, 2048, [1, 17, 40, 64, 65, 128, 200, 300], 1),
    (4, 128, 1, 64, [1, 2], 1),
    (2, 128, 1, 640, [5] * 17, 1),
    (4, 128, 7, 500, [7, 100, 64], 1),
    (2, 256, 2, 8011, [2, 93, 214, 377, 65], 33),
    (4, 256, 4, 1000, [4, 30, 500, 64, 128, 129], 1),
    (2, 256, 1, 4096, [3, 700], 1),
    (2, 128, 8, 3000, [8, 9, 1000], 2),
    (4, 128, 9, 700, [9, 130], 1),
    (2, 256, 10, 1300, [10, 200, 64], 3),
    (4, 256, 10, 200, [10], 1),
    (4, 128, 3, 0, [3, 70, 1000], 1),
    (4, 128, 2, 63, [2, 66, 500], 1),
    (2, 128, 1, 10000, [1], 1),
    (4, 128, 1, 320, [1000, 2000, 1, 3, 555], 1),
]


@pytest.mark.parametrize("hkv,d,q_len,prefix,own,ppb", CASES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_matches_the_formula(gpu_ops, hkv, d, q_len, prefix, own, ppb, dtype):
    x = Batch(gpu_ops, hkv, d, q_len, prefix, own, ppb, dtype, seed=q_len + prefix)
    x.check(x.run(dtype))


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 128), (4, 256), (2, 256)])
@pytest.mark.parametrize("tokens", [(1, 1), (2, 1), (1, 5), (7, 1), (9, 1), (3, 5), (4, 6), (65, 1), (130, 2)])
def test_groups_of_every_size(gpu_ops, hkv, d, tokens):
    """Batches that fill one, two and three query tiles, groups that end inside
    a sequence, and more sequences than lanes of a wave."""
    batch, q_len = tokens
    gen = random.Random(batch * 100 + q_len)
    x = Batch(gpu_ops, hkv, d, q_len, 450, [gen.randint(q_len, 90) for _ in range(batch)], seed=batch)
    x.check(x.run())


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 256)])
def test_sequences_that_end_inside_the_prefix(gpu_ops, hkv, d):
    """Lengths below the prefix, a query longer than its sequence, and empty ones."""
    x = Batch(gpu_ops, hkv, d, 3, 512, [5, -1, -64, -500, -509, -510, -511, None, 100, None], seed=1)
    x.check(x.run(torch.float32))
    x = Batch(gpu_ops, hkv, d, 10, 512, [-503, -504, -511, None, 12], seed=2)
    x.check(x.run())
    x = Batch(gpu_ops, hkv, d, 10, 0, [1, 2, 3, 9, 10, None], seed=2)
    x.check(x.run())


def test_nothing_to_see(gpu_ops):
    x = Batch(gpu_ops, 4, 128, 2, 300, [None, None, None], seed=3)
    x.check(x.run())
    x = Batch(gpu_ops, 4, 128, 2, 0, [None], seed=3)
    x.check(x.run())


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 256)])
def test_padding_rows_may_hold_anything(gpu_ops, hkv, d, bad):
    """A padding sequence's queries are NaN or infinite: it gives zeros, the others of its group are unmoved."""
    x = Batch(gpu_ops, hkv, d, 2, 400, [5, None, 70, 2, None], seed=4)
    clean = x.run()
    for b in (1, 4):
        x.q[2 * b : 2 * b + 2] = bad
    out = x.run()
    assert torch.equal(out, clean)
    assert not bool(out[2:4].any()) and not bool(out[8:].any())


def test_rows_that_see_no_token_of_a_written_page(gpu_ops):
    """Nine query tokens over a sequence of one: its first eight see nothing, and
    the page behind token 0 holds NaN planes."""
    x = Batch(gpu_ops, 4, 128, 9, 0, [1, 30], seed=5)
    for name in ("k_scale", "v_scale", "v_zero"):
        x.cache.views[name][int(x.table[0, 0]), 1:] = math.nan
    x.check(x.run())


def test_unwritten_tails_are_not_used(gpu_ops):
    """Rows of a sequence's last page behind its length hold NaN planes and codes."""
    x = Batch(gpu_ops, 2, 128, 2, 256, [2, 33, 64, 95, 130], seed=6)
    for b, n in enumerate(x.lens):
        page, row = int(x.table[b, (n - 1) // PAGE]), n % PAGE
        if row:
            for name in ("k_scale", "v_scale", "v_zero"):
                x.cache.views[name][page, row:] = math.nan
    x.check(x.run())


def test_pages_outside_the_cache_hold_no_keys(gpu_ops):
    x = Batch(gpu_ops, 4, 128, 2, 640, [2, 200, 300], seed=7)
    x.prefix_table[3], x.prefix_table[7] = -1, x.cache.num_pages
    x.table[1, 11], x.table[2, 12] = 2**31 - 1, -2**31
    x.prefix_dev, x.table_dev = x.prefix_table.to(DEV), x.table.to(DEV)
    x.check(x.run())


def test_lengths_past_the_table_are_cut_off(gpu_ops):
    x = Batch(gpu_ops, 4, 128, 1, 128, [300, 10], seed=8)
    x.lens_dev[0] = 2**31 - 1
    out = x.run()
    full = x.table.shape[1] * PAGE
    x.lens[0] = full
    fill_sequence(gpu_ops, x.cache, torch.Generator().manual_seed(9), x.table[0], full, start=(full // PAGE - 1) * PAGE)
    out = x.run()
    x.check(out)


def test_long_runs_of_pages(gpu_ops):
    """More than 128 pages in a work-group's piece: entries are looked up as it goes."""
    x = Batch(gpu_ops, 2, 128, 10, 64 * 900, [10 + (7 * i) % 90 for i in range(64)], seed=10)
    x.check(x.run())


@pytest.mark.parametrize("d,ppb", [(128, 33), (256, 33), (128, 5)])
def test_prefixes_that_end_inside_a_block(gpu_ops, d, ppb):
    x = Batch(gpu_ops, 2, d, 2, PAGE * ppb * 2 + 130, [2, 64 * ppb, 50], ppb, seed=11)
    x.check(x.run())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_strided_queries_and_outputs(gpu_ops, dtype):
    x = Batch(gpu_ops, 2, 128, 3, 300, [3, 60, 90], seed=12, fused=True)
    wide = torch.full((x.q.shape[0], 3 * 12 * 128), 5.0, dtype=dtype, device=DEV)
    out = wide[:, 12 * 128 : 2 * 12 * 128].unflatten(1, (12, 128))
    x.bind(out)()
    x.check(out)
    assert bool((wide[:, : 12 * 128] == 5).all()) and bool((wide[:, 2 * 12 * 128 :] == 5).all())
    flat = torch.full((x.q.numel() + 9 * 3 + 8,), 5.0, dtype=dtype, device=DEV)
    out = flat.as_strided(x.q.shape, (12 * 128 + 3, 128, 1), 1)  # rows at odd elements
    x.bind(out)()
    x.check(out)


def test_agrees_with_the_batch_op(gpu_ops):
    """The same step through int8k_int4v_attn_batch, the prefix written into every table row."""
    x = Batch(gpu_ops, 4, 128, 4, 1024, [4, 70, 500, 129], seed=13)
    table = x.table.clone()
    table[:, :16] = x.prefix_table[:16]
    same = decode(gpu_ops, x.cache, x.q, table, torch.tensor(x.lens, dtype=torch.int32), 4)
    out = x.run()
    x.check(out)
    x.check(same)


def test_the_same_call_gives_the_same_bits(gpu_ops):
    x = Batch(gpu_ops, 4, 256, 3, 2000, [3, 300, 40, 64, 1000], seed=14)
    first = x.run()
    for _ in range(3):
        x.ws.fill_(0x7F)
        assert torch.equal(x.run(), first)


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 256)])
def test_a_captured_call_follows_lengths_and_tables(gpu_ops, hkv, d):
    x = Batch(gpu_ops, hkv, d, 2, 700, [900, 900, 900, 900], seed=15)
    out = torch.empty_like(x.q)
    call = x.bind(out)
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    base = x.table.clone()
    for lens, order in (([1500, 702, 641, 642], [0, 1, 2, 3]), ([0, 2, 1, 1200], [3, 2, 1, 0]),
                        ([1540, 1540, 1540, 1540], [1, 0, 3, 2])):
        x.lens, x.table = lens, base[order]
        x.lens_dev.copy_(torch.tensor(lens, dtype=torch.int32))
        x.table_dev.copy_(x.table)
        x.q.copy_(torch.randn(x.q.shape, generator=torch.Generator().manual_seed(sum(lens))).to(x.q.dtype))
        out.fill_(math.nan)
        graph.replay()
        torch.cuda.synchronize()
        x.check(out)
        eager = x.run()  # an eager call between the replays, on the graph's own workspace
        assert torch.equal(eager, out)


def test_two_streams(gpu_ops):
    """Two calls at once, each with its own workspace; the tensors made on the default stream."""
    a = Batch(gpu_ops, 4, 128, 1, 5000, [40] * 20, seed=16)
    b = Batch(gpu_ops, 2, 256, 4, 3000, [60] * 9, seed=17)
    oa, ob = torch.empty_like(a.q), torch.empty_like(b.q)
    ca, cb = a.bind(oa), b.bind(ob)
    torch.cuda.synchronize()
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(4):
        with torch.cuda.stream(sa):
            ca()
        with torch.cuda.stream(sb):
            cb()
    torch.cuda.synchronize()
    a.check(oa)
    b.check(ob)


@pytest.mark.parametrize("case", range(16))
def test_random_shapes(gpu_ops, case):
    rng = random.Random(900 + case)
    hkv, d, ppb = rng.choice([2, 4]), rng.choice([128, 256]), rng.choice([1, 1, 2, 33])
    q_len, batch = rng.randint(1, 10), rng.randint(1, 40)
    prefix = rng.choice([rng.randint(0, 300), rng.randint(300, 9000)])
    own = [None if rng.random() < 0.1 else rng.choice([rng.randint(q_len, 100), rng.randint(q_len, 900)])
           for _ in range(batch)]
    print("case %d: hkv %d d %d ppb %d q_len %d prefix %d own %s" % (case, hkv, d, ppb, q_len, prefix, own), flush=True)
    x = Batch(gpu_ops, hkv, d, q_len, prefix, own, ppb, rng.choice([torch.float16, torch.bfloat16]), seed=case,
              fused=rng.random() < 0.5)
    x.check(x.run(rng.choice([torch.float16, torch.bfloat16, torch.float32])))


@pytest.mark.parametrize("hkv,d,batch,prefix", [(4, 128, 3, 130), (2, 256, 5, 64), (4, 128, 40, 17000), (4, 256, 30, 640)])
def test_query_values_on_rounding_ties(gpu_ops, hkv, d, batch, prefix):
    """Every query value halfway between two codes of its row (bf16, the largest 127 / 64): the rule's codes, in both forms."""
    x = Batch(gpu_ops, hkv, d, 2, prefix, [2 + 3 * i for i in range(batch)], dtype=torch.bfloat16, seed=batch)
    gen = torch.Generator().manual_seed(batch)
    rows = (torch.randint(-127, 127, x.q.shape, generator=gen) + 0.5) / 64
    rows[..., 5] = 127 / 64
    x.q = rows.to(torch.bfloat16).to(DEV)
    assert torch.equal(x.q.float().cpu(), rows)
    x.check(x.run(torch.float32))


def test_wide_value_range(gpu_ops):
    """V rows over the whole fp16 range stay finite in the states (as in the batch op)."""
    x = Batch(gpu_ops, 2, 128, 1, 256, [40, 70], seed=18)
    x.cache.views["v_scale"].mul_(20000.0)
    x.check(x.run(torch.float32))


def test_offsets_past_32_bits(gpu_ops):
    """Pages behind the first 4 GiB of a pool."""
    x = Batch(gpu_ops, 4, 128, 1, 200, [30, 100], seed=19)
    lay = PageLayout(4, 128)
    pages = (2**32 + 2**28) // lay.page_bytes
    big = Cache(pages, lay)
    shift = pages - x.cache.num_pages
    big.raw[shift * lay.page_bytes :] = x.cache.raw
    x.cache = big
    x.prefix_table, x.table = x.prefix_table + shift, torch.where(x.table >= 0, x.table + shift, x.table)
    x.prefix_dev, x.table_dev = x.prefix_table.to(DEV), x.table.to(DEV)
    x.check(x.run())

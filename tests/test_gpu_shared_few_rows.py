"""int8k_int4v_attn_shared where it takes eight tokens at a time over a long prefix.

The library's rule serves most batches by the kernel that holds many query rows;
each case here asks it first that the other form is the one taken, and the cases
of long page runs that a work-group's run is as long as they are meant to test.
Reference and tolerances: test_gpu_shared.py.
"""
from __future__ import annotations

import math

import pytest
import torch

from gpu_cases import DEV
from k8v4_v030.layout import GQA, PAGE
from test_gpu_shared import Batch

pytestmark = pytest.mark.gpu

# (sequences, query tokens, pages of the prefix): one, two and three row tiles, one and more groups of eight tokens.
SMALL = [(1, 1, 300), (2, 1, 300), (1, 3, 260), (3, 1, 300), (5, 1, 300), (1, 5, 257), (8, 1, 400), (13, 1, 640), (2, 6, 600)]
CASES = [(hkv, d, *s) for hkv in (2, 4) for d in (128, 256) for s in SMALL]
CASES += [(hkv, 128, *s) for hkv in (2, 4) for s in ((15, 1, 730), (3, 5, 730), (2, 10, 970))]
CASES += [(4, 128, 5, 7, 240), (4, 128, 50, 1, 210), (2, 128, 5, 7, 400), (2, 128, 64, 2, 300), (2, 256, 5, 7, 300),
          (2, 256, 10, 2, 370)]


@pytest.mark.parametrize("hkv,d,batch,q_len,pages", CASES)
def test_long_prefix_by_eight_tokens_at_a_time(gpu_ops, hkv, d, batch, q_len, pages):
    prefix = pages * PAGE
    assert not gpu_ops.attn_shared_many_rows(batch, q_len, hkv, d, prefix)
    own = [q_len + (29 * i) % 150 for i in range(batch)]
    dtype = (torch.float16, torch.bfloat16)[batch & 1]
    x = Batch(gpu_ops, hkv, d, q_len, prefix, own, dtype=dtype, seed=batch + pages)
    x.check(x.run(dtype))
    x.lens[0] = prefix - 100  # a sequence that ends inside the prefix
    x.lens_dev[0] = x.lens[0]
    x.check(x.run(torch.float32))


class Repeated(Batch):
    """Sequences of many pages that are few physical ones, each many times over.

    A key that occurs c times weighs c exp(score): the reference adds log(c) to the
    score of one."""

    def __init__(self, ops, hkv, d, q_len, batch, prefix_pages, own_pages, cut, seed):
        super().__init__(ops, hkv, d, q_len, 12 * PAGE, [q_len] * batch, seed=seed)
        gen = torch.Generator().manual_seed(seed)
        stored = self.prefix_table[:12]
        width = prefix_pages + own_pages
        pick = lambda shape: stored[torch.randint(0, 12, shape, generator=gen)].contiguous()
        self.prefix_table, self.table = pick((max(prefix_pages, 1),)), pick((batch, width))
        self.prefix = self.shared = prefix_pages * PAGE
        self.lens = [width * PAGE - cut - 3 * b for b in range(batch)]
        self.lens_dev = torch.tensor(self.lens, dtype=torch.int32, device=DEV)
        self.table_dev, self.prefix_dev = self.table.to(DEV), self.prefix_table.to(DEV)

    def want(self):
        v_ = self.cache.views
        byte = v_["v"].flatten(0, 1)
        nib = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).double()
        k = v_["k"].flatten(0, 1).double() * v_["k_scale"].flatten(0, 1).double()[..., None]
        v = (nib - v_["v_zero"].flatten(0, 1).double()[..., None]) * v_["v_scale"].flatten(0, 1).double()[..., None]
        q = self.q.double()
        scale = q.abs().amax(-1, keepdim=True) / torch.full((), 127.0, dtype=torch.float64, device=DEV)
        q = torch.sign(q) * torch.floor(q.abs() * (1.0 / scale) + 0.5) * scale
        o, a = torch.zeros_like(q), torch.zeros_like(q)
        r = torch.zeros(q.shape[0], 1, 1, dtype=torch.float64, device=DEV)
        step = float(v_["v_scale"].max())
        pages = torch.arange(self.table.shape[1], device=DEV)
        for b in range(self.batch):
            entry = torch.where(pages < self.shared // PAGE, self.prefix_dev[pages.clamp(max=self.prefix_dev.shape[0] - 1)],
                                self.table_dev[b]).long()
            slots = (entry[:, None] * PAGE + torch.arange(PAGE, device=DEV)).flatten()
            for j in range(self.q_len):
                row, end = b * self.q_len + j, self.lens[b] - self.q_len + j + 1
                many = torch.bincount(slots[:end], minlength=k.shape[0]).double()
                r[row] = 4 * math.sqrt(-(-end // 32)) * 255 * step * 2.0**-24
                for h in range(self.hkv):
                    heads = slice(h * GQA, (h + 1) * GQA)
                    s = torch.mm(q[row, heads], k[:, h].t().contiguous()) / math.sqrt(self.d)
                    p = torch.softmax(torch.where(many > 0, s + many.log(), -math.inf), 1)
                    p = torch.where(many > 0, p, 0.0)
                    there = torch.where(many[:, None] > 0, v[:, h], 0.0)
                    o[row, heads] = torch.mm(p, there)
                    a[row, heads] = torch.mm(p, there.abs())
        return o, a, r


def groups_on_the_chip(hkv, d):
    """Work-groups of the launch: one per CU, two of two 128-dim heads."""
    return torch.cuda.get_device_properties(DEV).multi_processor_count * (2 if (hkv, d) == (2, 128) else 1)


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 128), (4, 256), (2, 256)])
@pytest.mark.parametrize("batch,q_len", [(2, 1), (3, 4)])
def test_prefix_runs_of_more_than_128_pages(gpu_ops, hkv, d, batch, q_len):
    """A work-group's run of the prefix is longer than the table entries it keeps: it looks them up as it goes."""
    groups = -(-batch * q_len // 8)
    pages = 140 * groups_on_the_chip(hkv, d) // groups
    assert not gpu_ops.attn_shared_many_rows(batch, q_len, hkv, d, pages * PAGE)
    x = Repeated(gpu_ops, hkv, d, q_len, batch, pages, 2, 5, seed=batch)
    x.check(x.run())


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 128), (4, 256), (2, 256)])
@pytest.mark.parametrize("q_len", [1, 3, 9])
def test_own_runs_of_more_than_128_pages(gpu_ops, hkv, d, q_len):
    """The same of the sequences' own pages, with nothing shared and behind a page of prefix."""
    segments = 2 if q_len > 8 else 1  # of a sequence
    batch = 24
    pages = 140 * groups_on_the_chip(hkv, d) // (batch * segments)
    x = Repeated(gpu_ops, hkv, d, q_len, batch, 0, pages, 70, seed=q_len)
    assert not gpu_ops.attn_shared_many_rows(batch, q_len, hkv, d, x.prefix)
    x.check(x.run())
    x = Repeated(gpu_ops, hkv, d, q_len, batch, 1, pages, 33, seed=q_len + 1)  # either form
    x.check(x.run())

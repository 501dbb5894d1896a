"""rope_kv_store_paged against the rotation and the cache's rules in 64 bits.

The cache's bytes are compared bit for bit: the rule applies to the rotated rows in
float64, which the products (of 24 and 11 bits) and one sum define.  Queries are
two fp32 products and an fp32 sum, 2^-24 each of the products' magnitudes, and one
rounding to their type, half a step.
"""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from gpu_cases import Cache, DEV
from k8v4_v030.layout import GQA, PAGE, PageLayout
from oracle import paged

pytestmark = pytest.mark.gpu

F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def angles(rows, rot, dtype, gen):
    """A table as a model makes it, with a few rows of other values."""
    inv = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat((a.cos(), a.sin()), 1).to(dtype)


def rotated(x, cos_sin, neox):
    x = x.double().cpu()
    half = cos_sin.shape[1] // 2
    c, s = cos_sin[:, None, :half].double(), cos_sin[:, None, half:].double()
    first = torch.arange(half) if neox else 2 * torch.arange(half)
    second = first + (half if neox else 1)
    u, v = x[..., first], x[..., second]
    y = x.clone()
    y[..., first], y[..., second] = u * c - v * s, v * c + u * s
    size = x.abs()
    size[..., first] = size[..., second] = 0.0
    size[..., first], size[..., second] = (u * c).abs() + (v * s).abs(), (v * c).abs() + (u * s).abs()
    return y, size


class Step:
    def __init__(self, hkv, d, dtype, table, rot, neox, tokens, seed, table_rows=5000, fused=True, index=torch.int64):
        gen = torch.Generator().manual_seed(seed)
        self.hkv, self.d, self.neox = hkv, d, neox
        self.cache = Cache(tokens // PAGE + 3, PageLayout(hkv, d))
        heads = (GQA + 2) * hkv
        rows = torch.randn((tokens, heads, d), generator=gen).to(dtype)
        if fused:  # views of a projection's rows
            q, k, v = rows.to(DEV).split([GQA * hkv, hkv, hkv], 1)
        else:
            q, k, v = (x.contiguous().to(DEV) for x in rows.split([GQA * hkv, hkv, hkv], 1))
        self.q, self.k, self.v = q, k, v
        self.table = angles(table_rows, rot, table, gen)
        self.positions = torch.randint(0, table_rows, (tokens,), generator=gen).to(index)
        self.slots = torch.randperm(self.cache.num_pages * PAGE, generator=gen)[:tokens]
        self.q_out = torch.full(q.shape, math.nan, dtype=dtype, device=DEV)

    def args(self, q="q", q_out="q_out"):
        pick = lambda x: getattr(self, x) if isinstance(x, str) else x  # noqa: E731
        return (pick(q), self.k, self.v, self.positions.to(DEV), self.table.to(DEV), self.neox, self.slots.to(DEV),
                *self.cache.region_args(), pick(q_out))

    def want_blob(self, before=None):
        there = (self.positions >= 0) & (self.positions < self.table.shape[0])
        k, _ = rotated(self.k, self.table[self.positions.clamp(0, self.table.shape[0] - 1).long()], self.neox)
        blob = paged.new_blob(self.cache.num_pages, self.cache.geom) if before is None else before.copy()
        slots = torch.where(there, self.slots, torch.full_like(self.slots, -1))
        paged.store(blob, self.cache.geom, k.numpy(), self.v.cpu().double().numpy(), slots.numpy())
        return blob

    def check_queries(self, q, got):
        there = (self.positions >= 0) & (self.positions < self.table.shape[0])
        want, size = rotated(q, self.table[self.positions.clamp(0, self.table.shape[0] - 1).long()], self.neox)
        want, size = want * there[:, None, None], size * there[:, None, None]
        eps = torch.finfo(got.dtype).eps / 2
        low = 2.0**-25 if got.dtype == F16 else 0.0  # half of fp16's subnormal step
        tol = (eps * want.abs() + 2 * 2.0**-24 * size) * (1 + 2.0**-7) + low
        err = (got.double().cpu() - want).abs()
        assert bool((err <= tol).all()), float((err - tol).max())


CASES = [
    (4, 128, F16, F32, 128, True, 130), (4, 128, BF16, BF16, 128, True, 1), (2, 128, BF16, F32, 64, False, 67),
    (4, 128, F16, F16, 16, True, 5), (4, 128, F16, F32, 112, False, 33), (2, 128, F16, F32, 48, True, 9),
    (4, 256, BF16, F32, 256, True, 70), (2, 256, F16, BF16, 64, True, 65), (2, 256, BF16, F32, 256, False, 3),
    (4, 256, F16, F32, 16, False, 2), (2, 256, BF16, BF16, 240, True, 1),
]


@pytest.mark.parametrize("hkv,d,dtype,table,rot,neox,tokens", CASES)
@pytest.mark.parametrize("fused", [True, False])
def test_rows_and_bytes(gpu_ops, hkv, d, dtype, table, rot, neox, tokens, fused):
    st = Step(hkv, d, dtype, table, rot, neox, tokens, seed=rot + tokens, fused=fused)
    gpu_ops.rope_kv_store_paged(*st.args())
    assert np.array_equal(st.cache.blob(), st.want_blob())
    st.check_queries(st.q, st.q_out)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
def test_skipped_tokens_and_positions_outside(gpu_ops, index):
    st = Step(4, 128, BF16, F32, 128, True, 40, seed=3, table_rows=100, index=index)
    st.slots[5], st.slots[17], st.slots[18] = -1, -(2**40), st.cache.num_pages * PAGE
    st.positions[3], st.positions[9] = 100, -1
    st.cache.raw.random_(0, 127)
    before = st.cache.blob().copy()
    gpu_ops.rope_kv_store_paged(*st.args())
    assert np.array_equal(st.cache.blob(), st.want_blob(before))
    st.check_queries(st.q, st.q_out)
    assert not st.q_out[[3, 9]].any() and st.q_out[5].any()


def test_in_place_and_without_queries(gpu_ops):
    st = Step(2, 256, F16, F32, 128, True, 21, seed=5)
    before = st.q.clone()
    gpu_ops.rope_kv_store_paged(*st.args(q_out="q"))  # a view of the projection's rows
    st.check_queries(before, st.q)
    assert np.array_equal(st.cache.blob(), st.want_blob())
    st.cache.raw.zero_()
    gpu_ops.rope_kv_store_paged(*st.args(None, None))
    assert np.array_equal(st.cache.blob(), st.want_blob())


def test_rows_at_any_element(gpu_ops):
    """Query, key, value, output and table rows that start at odd elements."""
    st = Step(4, 128, F16, F16, 64, False, 11, seed=6, fused=False)

    def odd(x):
        width = x[0].numel()
        buf = torch.zeros(x.shape[0] * (width + 3) + 1, dtype=x.dtype, device=DEV)
        view = buf[1:].as_strided(x.shape, (width + 3, *x.stride()[1:]), 1)
        view.copy_(x)
        return view, buf

    (st.q, _), (st.k, _), (st.v, _) = odd(st.q), odd(st.k), odd(st.v)
    st.q_out, whole = odd(st.q_out)
    table, _ = odd(st.table.to(DEV))
    args = list(st.args())
    args[4] = table
    whole.fill_(7.0)
    gpu_ops.rope_kv_store_paged(*args)
    assert np.array_equal(st.cache.blob(), st.want_blob())
    st.check_queries(st.q, st.q_out)
    st.q_out.fill_(7.0)
    assert bool((whole == 7.0).all())  # nothing between the rows was written


def test_zero_rows_ties_and_large_values(gpu_ops):
    """All-zero rows, position 0 (the identity: codes on ties), rows whose rotation leaves
    the type's range."""
    st = Step(4, 128, BF16, F32, 128, True, 12, seed=7, fused=False)
    st.k[0], st.v[0] = 0.0, 0.0
    st.positions[:4] = 0
    st.k[1] = (torch.arange(512, device=DEV).view(4, 128) % 255 - 127) / 128.0  # amax 127 / 128: ties at .5
    st.k[2, :, 0], st.v[2] = 127 / 64, 1.0
    st.k[3] = torch.randint(-254, 255, (4, 128), device=DEV) / 128.0
    st.k[4] = 3.0e38
    st.k[5] = 1.0e-38
    st.k[6] = 1.0e-40
    gpu_ops.rope_kv_store_paged(*st.args())
    assert np.array_equal(st.cache.blob(), st.want_blob())


def test_no_tokens(gpu_ops):
    st = Step(4, 128, F16, F32, 128, True, 2, seed=8)
    st.q, st.k, st.v, st.q_out = st.q[:0], st.k[:0], st.v[:0], st.q_out[:0]
    st.positions, st.slots = st.positions[:0], st.slots[:0]
    assert gpu_ops.bind_rope_kv_store_paged(*st.args()) is None
    gpu_ops.rope_kv_store_paged(*st.args())
    assert not st.cache.raw.any()


def test_captured_and_replayed(gpu_ops):
    """One captured store, replayed with other keys, positions and slots."""
    st = Step(4, 128, BF16, F32, 128, True, 30, seed=9)
    args = st.args()
    call = gpu_ops.bind_rope_kv_store_paged(*args)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(3):
        new = Step(4, 128, BF16, F32, 128, True, 30, seed=20 + seed)
        for old, x in ((st.q, new.q), (st.k, new.k), (st.v, new.v)):
            old.copy_(x)
        st.positions, st.slots = new.positions, new.slots
        args[3].copy_(st.positions)
        args[6].copy_(st.slots)
        st.cache.raw.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(st.cache.blob(), st.want_blob())
        st.check_queries(st.q, st.q_out)

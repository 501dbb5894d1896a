"""The tree-drafting operators where sizes choose another kernel or pass 32 bits.

Which kernel int8k_int4v_attn_tree takes depends on the nodes and on the pages that
the tables have room for: eight nodes at a time up to 16 nodes over more than 64 pages
a node, and from 22 (256 dims) or 33 on over up to 384 pages (but for four heads of 256
dims, and some of 42 nodes and fewer), all rows of a KV head otherwise.  Here tables are widened by entries that no length reaches, so
that short sequences take either.  Tolerances are test_gpu_tree's and, for bytes, none.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from gpu_cases import Cache, DEV
from k8v4_v030.layout import PAGE, PageLayout
from oracle import paged
from test_gpu_rope_store import Step
from test_gpu_tree import SHAPES, Trees

pytestmark = pytest.mark.gpu

CONTEXTS = [300, 0, None, 1000, 61, -3]


def widened(st, pages):
    """The same tables, wide enough for more than ``pages`` pages in all."""
    width = pages // (st.batch * st.ppb) + 1
    if width > st.table.shape[1]:
        more = torch.full((st.batch, width - st.table.shape[1]), -1, dtype=torch.int32)
        st.table = torch.cat((st.table, more), 1)
        st.table_dev = st.table.to(DEV)
    return st


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes", [1, 2, 5, 8, 9, 13, 16])
def test_few_nodes_over_wide_tables(gpu_ops, hkv, d, nodes):
    st = widened(Trees(gpu_ops, hkv, d, nodes, CONTEXTS, seed=nodes, dtype=torch.bfloat16), 64 * nodes)
    st.check(st.run(torch.float32))


@pytest.mark.parametrize("hkv,d", SHAPES)
@pytest.mark.parametrize("nodes", [17, 22, 26, 32, 37, 43, 50, 57, 63, 64])
def test_many_nodes_over_wide_tables(gpu_ops, hkv, d, nodes):
    st = widened(Trees(gpu_ops, hkv, d, nodes, CONTEXTS, seed=nodes), 384)
    st.check(st.run(torch.float32))


def test_both_forms_agree(gpu_ops):
    """On the rows that the padding of a table does not concern, within both tolerances."""
    st = Trees(gpu_ops, 4, 128, 40, CONTEXTS, seed=5)
    want = st.want()
    a = st.run(torch.float32)
    b = widened(st, 384).run(torch.float32)
    st.check(a, want)
    st.check(b, want)


def far(cache, lay):
    """A cache whose last pages, behind its first 4 GiB, are those of ``cache``, and the first of them."""
    pages = (2**32 + 2**28) // lay.page_bytes
    big = Cache(pages, lay)
    first = pages - cache.num_pages
    big.raw[first * lay.page_bytes :] = cache.raw
    return big, first


@pytest.mark.parametrize("hkv,d,nodes,pages", [(4, 128, 13, 0), (4, 128, 13, 64 * 13), (2, 256, 30, 0), (2, 256, 30, 384)])
def test_tree_offsets_past_32_bits(gpu_ops, hkv, d, nodes, pages):
    st = Trees(gpu_ops, hkv, d, nodes, [200, 0, 70], seed=3)
    st.cache, first = far(st.cache, PageLayout(hkv, d))
    st.table = torch.where(st.table >= 0, st.table + first, st.table)
    st.table_dev = st.table.to(DEV)
    widened(st, pages)
    st.check(st.run())


def test_store_and_moves_past_32_bits(gpu_ops):
    lay = PageLayout(4, 128)
    st = Step(4, 128, torch.bfloat16, torch.float32, 128, True, 150, 4)
    want = st.want_blob()
    small = st.cache
    st.cache, first = far(small, lay)
    st.slots = st.slots + first * PAGE
    gpu_ops.rope_kv_store_paged(*st.args())
    torch.cuda.synchronize()
    tail = st.cache.raw[first * lay.page_bytes :].view(torch.uint8)
    assert np.array_equal(tail.cpu().numpy(), want)
    assert not bool(st.cache.raw[: lay.page_bytes * small.num_pages].any())
    # Page 1's tokens moved among themselves: rows 10, 40 and 63 to rows 1, 2 and 3.
    table = torch.tensor([[first + 1]], dtype=torch.int32, device=DEV)
    path = torch.tensor([[0, 10, 40, 63]], dtype=torch.int32, device=DEV)
    index = lambda *x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    gpu_ops.kv_keep_paged(*st.cache.region_args(), table, index(0), path, index(3), 1)
    regions = paged.regions(want, small.geom)
    for region in regions.values():
        for to, node in ((1, 10), (2, 40), (3, 63)):
            region[1, to] = region[1, node]
    torch.cuda.synchronize()
    assert np.array_equal(tail.cpu().numpy(), want)

"""kv_keep_paged: cache rows moved byte for byte, nothing else touched."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from gpu_cases import Cache, DEV
from k8v4_v030.layout import PAGE, PageLayout
from oracle import paged

pytestmark = pytest.mark.gpu


def index(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def moved(cache, before, table, ppb, starts, path, accepted):
    """The bytes after the moves: everything read from ``before``."""
    blob = before.copy()
    src, dst = paged.regions(before, cache.geom), paged.regions(blob, cache.geom)
    reach = table.shape[1] * ppb * PAGE

    def place(b, t):
        if not 0 <= t < reach:
            return None
        page = int(table[b, t // PAGE // ppb]) * ppb + t // PAGE % ppb
        return (page, t % PAGE) if 0 <= page < cache.num_pages else None

    for b, row in enumerate(path):
        for i, node in enumerate(row[: accepted[b] + 1]):
            if node > i:
                x, y = place(b, starts[b] + node), place(b, starts[b] + i)
                if x and y:
                    for name in src:
                        dst[name][y] = src[name][x]
    return blob


def run(ops, hkv, d, ppb, table, starts, path, accepted, pages):
    cache = Cache(pages, PageLayout(hkv, d))
    cache.raw.copy_(torch.randint(-128, 128, cache.raw.shape, generator=torch.Generator().manual_seed(hkv * d), dtype=torch.int8))
    before = cache.blob().copy()
    table = torch.tensor(table, dtype=torch.int32)
    ops.kv_keep_paged(*cache.region_args(), table.to(DEV), index(starts), index(path), index(accepted), ppb)
    assert np.array_equal(cache.blob(), moved(cache, before, table, ppb, starts, path, accepted))


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 128), (2, 256), (4, 256)])
@pytest.mark.parametrize("ppb", [1, 3])
def test_branches(gpu_ops, hkv, d, ppb):
    wide = list(range(0, 40, 2))
    path = [[0, 2, 5, 6, 63] + [-1] * 15, wide, list(range(20)), [0, 1, 2] + [-1] * 17, [63] + [-1] * 19, [3] * 20]
    starts, accepted = [60, 0, 5, 64, 127, 191], [4, 19, 19, 2, 0, 19]
    table = [[6 * i + j for j in range(6)] for i in range(6)]
    run(gpu_ops, hkv, d, ppb, table, starts, path, accepted, pages=36 * ppb)


def test_what_moves_nothing(gpu_ops):
    """Entries behind `accepted`, below their place, outside the table, on pages outside the cache."""
    path = [[0, 5, -1, 1, 9], [0, 4, 5, 6, 7], [0, 3, 2**31 - 1, -2**31, 8], [0, 60, 61, 62, 63], [1, 2, 3, 4, 5],
            [0, 5, 6, 7, 8]]
    starts, accepted = [10, 10, 10, 64, -3, 2**31 - 4], [4, -1, 100, 4, 4, 4]
    table = [[0, 1], [2, 3], [4, 5], [6, 99], [7, -1], [8, 9]]
    run(gpu_ops, 4, 128, 1, table, starts, path, accepted, pages=12)
    run(gpu_ops, 4, 128, 1, [r[:1] for r in table], starts, path, [-2**31, 2**31 - 1, 4, 4, 4, 4], pages=7)


def test_of_nothing(gpu_ops):
    cache = Cache(2, PageLayout(4, 128))
    none = torch.empty((0, 3), dtype=torch.int32, device=DEV)
    empty = torch.empty((0,), dtype=torch.int32, device=DEV)
    assert gpu_ops.bind_kv_keep_paged(*cache.region_args(), none, empty, none, empty, 1) is None
    one = index([0])
    assert gpu_ops.bind_kv_keep_paged(*cache.region_args(), index([[0]]), one, none[:, :0].expand(0, 0).reshape(1, 0), one, 1) is None


def test_on_another_stream_and_replayed(gpu_ops):
    cache = Cache(8, PageLayout(2, 256))
    table, starts = torch.arange(8, dtype=torch.int32).view(2, 4), [30, 70]
    path, accepted = index([[0, 3, 4, 9], [0, 2, 40, 41]]), index([3, 3])
    call = gpu_ops.bind_kv_keep_paged(*cache.region_args(), table.to(DEV), index(starts), path, accepted, 1)
    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        call()
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    gen = torch.Generator().manual_seed(1)
    for rows, kept in (([[0, 1, 7, 8], [0, 5, 6, 7]], [3, 2]), ([[0, 2, 3, 30], [0, 1, 3, 4]], [1, 3]), ([[0, 3, 4, 9]] * 2, [-1, 3])):
        cache.raw.copy_(torch.randint(-128, 128, cache.raw.shape, generator=gen, dtype=torch.int8))
        before = cache.blob().copy()
        path.copy_(torch.tensor(rows, dtype=torch.int32))
        accepted.copy_(torch.tensor(kept, dtype=torch.int32))
        torch.cuda.synchronize()
        graph.replay()
        assert np.array_equal(cache.blob(), moved(cache, before, table, 1, starts, rows, kept))

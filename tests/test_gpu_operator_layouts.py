"""int8k_int4v_attn_shared and kv_load_paged over caches that are not one packed buffer:
regions in buffers of their own, pages padded by different amounts, planes far
apart or in another order, V rows that are only 4-byte aligned."""
from __future__ import annotations

import pytest
import torch

from gpu_cases import DEV
from k8v4_v030.layout import PAGE
from test_gpu_shared import Batch

pytestmark = pytest.mark.gpu

NAMES = ("k", "k_scale", "v", "v_scale", "v_zero")


def moved(view, buf, start, page_bytes):
    """``view`` copied into the bytes of ``buf`` from ``start`` on, its pages ``page_bytes`` apart."""
    size = view.element_size()
    assert start % size == 0 and page_bytes % size == 0
    shape = tuple(view.shape)
    inner = [1]
    for n in reversed(shape[2:]):
        inner.insert(0, inner[0] * n)
    assert start + (shape[0] - 1) * page_bytes + shape[1] * inner[0] * size <= buf.numel()
    out = buf.view(view.dtype).as_strided(shape, (page_bytes // size, *inner), start // size)
    out.copy_(view)
    return out


def page_of(view):
    return view[0].numel() * view.element_size()


def own_buffers(views, pad):
    """Every region in a buffer of its own, its pages ``pad[name]`` bytes apart."""
    out = {}
    for name in NAMES:
        view = views[name]
        step = page_of(view) + pad[name]
        buf = torch.full((view.shape[0] * step + 64,), -1, dtype=torch.int8, device=DEV)  # NaN planes, code -1
        out[name] = moved(view, buf, 0, step)
    return out


def far_planes(views, order):
    """Planes of one page stride in one buffer, their starts 1.1 GiB apart in the given order."""
    step = page_of(views["k_scale"])
    gap = (1 << 30) + (1 << 27)
    buf = torch.empty(2 * gap + step * views["k_scale"].shape[0] + 64, dtype=torch.int8, device=DEV)
    return {**views, **{name: moved(views[name], buf, i * gap, step) for i, name in enumerate(order)}}


def near_planes(views, order):
    """The same side by side: within the reach of one base address, v_zero's before v_scale's and so on."""
    step = page_of(views["k_scale"])
    room = -(-step * views["k_scale"].shape[0] // 64) * 64 + 192
    buf = torch.empty(3 * room, dtype=torch.int8, device=DEV)
    return {**views, **{name: moved(views[name], buf, i * room, step) for i, name in enumerate(order)}}


def shifted_v(views):
    """V rows that start 4 bytes off a 16-byte line, pages a multiple of 4 apart."""
    view = views["v"]
    step = page_of(view) + 12
    buf = torch.empty(view.shape[0] * step + 64, dtype=torch.int8, device=DEV)
    return {**views, "v": moved(view, buf, 4, step)}


LAYOUTS = {
    "padded": lambda v: own_buffers(v, dict(k=48, k_scale=8, v=24, v_scale=16, v_zero=40)),
    "own": lambda v: own_buffers(v, dict(k=0, k_scale=0, v=0, v_scale=0, v_zero=0)),
    "far": lambda v: far_planes(v, ("k_scale", "v_scale", "v_zero")),
    "far_back": lambda v: far_planes(v, ("v_zero", "v_scale", "k_scale")),
    "turned": lambda v: near_planes(v, ("v_zero", "k_scale", "v_scale")),
    "back": lambda v: near_planes(v, ("v_zero", "v_scale", "k_scale")),
    "shifted_v": shifted_v,
}

# hkv, D, sequences, query tokens, pages of the prefix, whether many rows are served together
SHAPES = [(4, 128, 3, 2, 20, True), (4, 128, 5, 7, 5, False), (2, 128, 30, 1, 9, True), (2, 128, 5, 9, 4, False),
          (2, 256, 3, 2, 6, True), (2, 256, 5, 7, 7, False), (4, 256, 40, 1, 11, True), (4, 256, 1, 1, 50, False)]


@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("hkv,d,batch,q_len,pages,many", SHAPES)
def test_shared_prefix(gpu_ops, layout, hkv, d, batch, q_len, pages, many):
    assert gpu_ops.attn_shared_many_rows(batch, q_len, hkv, d, pages * PAGE) == many
    x = Batch(gpu_ops, hkv, d, q_len, pages * PAGE + 7, [q_len + 7 + (31 * i) % 200 for i in range(batch)], seed=pages)
    packed = x.run(torch.float32)
    x.check(packed)
    x.cache.views = LAYOUTS[layout](x.cache.views)
    assert torch.equal(x.run(torch.float32), packed)


@pytest.mark.parametrize("layout", [n for n in LAYOUTS if n != "shifted_v"])
@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 256)])
def test_read_back(gpu_ops, layout, hkv, d):
    x = Batch(gpu_ops, hkv, d, 1, 0, [300, 77, 1, 64], seed=hkv)
    starts = torch.tensor([0, 300, 377, 378, 442], dtype=torch.int32, device=DEV)

    def load():
        k = torch.full((442, hkv, d), 7.0, device=DEV)
        v = torch.full_like(k, 7.0)
        gpu_ops.kv_load_paged(*x.cache.region_args(), x.table_dev, None, starts, 1, k, v)
        torch.cuda.synchronize()
        return k, v

    packed = load()
    for b in range(4):
        k64, v64, _ = x.rows64(b)
        rows = slice(int(starts[b]), int(starts[b + 1]))
        assert torch.equal(packed[0][rows].double(), k64.float().double())
        err = (packed[1][rows].double() - v64).abs()
        assert bool((err <= 2.0**-23 * (1 + 2.0**-20) * v64.abs()).all())  # the difference and the product, half a step of fp32 each
    x.cache.views = LAYOUTS[layout](x.cache.views)
    got = load()
    assert torch.equal(got[0], packed[0]) and torch.equal(got[1], packed[1])

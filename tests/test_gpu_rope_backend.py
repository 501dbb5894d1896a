"""The vLLM backend's rotation and store in one call, in vLLM's tensor shapes, and a
decode step over what it stored."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from backend_cases import common_metadata, make_builder, make_impl, slots_for, vllm_cache
from gpu_cases import DEV, assert_close
from k8v4_v030.layout import PageLayout
from oracle import attention, paged

pytestmark = pytest.mark.gpu


def table_of(rows, rot, dtype):
    inv = 10000.0 ** (-torch.arange(rot // 2, dtype=torch.float64) / (rot // 2))
    a = torch.arange(rows, dtype=torch.float64)[:, None] * inv
    return torch.cat((a.cos(), a.sin()), 1).to(dtype)


def rotated(x, angles, neox):
    x = x.double().cpu()
    half = angles.shape[1] // 2
    c, s = angles[:, None, :half].double(), angles[:, None, half:].double()
    first = torch.arange(half) if neox else 2 * torch.arange(half)
    second = first + (half if neox else 1)
    y = x.clone()
    y[..., first], y[..., second] = x[..., first] * c - x[..., second] * s, x[..., second] * c + x[..., first] * s
    return y


@pytest.mark.parametrize("hkv,d,dtype,rot,neox,flat", [(4, 128, torch.bfloat16, 128, True, True),
                                                       (2, 256, torch.float16, 64, False, False)])
def test_steps(hkv, d, dtype, rot, neox, flat):
    """A chunk, then single tokens, with padding rows behind the slot map's; every step's
    attention against the oracle over the stored bytes."""
    lay = PageLayout(hkv, d)
    impl, builder = make_impl(hkv, d), make_builder(hkv, d, device=DEV)
    cache, geom = vllm_cache(8, 64, lay, DEV), paged.Geometry(hkv, d)
    table = torch.tensor([[5, 2, 7, 0]], dtype=torch.int32)
    angles = table_of(300, rot, dtype)
    gen = torch.Generator().manual_seed(hkv)
    want, at = paged.new_blob(8, geom), 0
    for n in (100, 1, 1, 3):
        rows = torch.randn((n + 2, (lay.hq + 2 * hkv) * d), generator=gen).to(dtype).to(DEV)
        q, k, v = rows.split([lay.hq * d, hkv * d, hkv * d], 1)
        if not flat:
            q, k, v = (x.unflatten(1, (-1, d)) for x in (q, k, v))
        before = rows.clone()
        pos = torch.arange(at, at + n + 2)
        slots = slots_for(table[0], range(at, at + n), 64)
        assert impl.fused_rope_kvcache_supported()
        impl.do_rope_and_kv_cache_update(None, q, k, v, pos.to(DEV), angles.to(DEV), neox, cache, slots.to(DEV))
        at += n
        torch.cuda.synchronize()
        heads = before[:n].unflatten(1, (-1, d))
        turned = rotated(heads[:, : lay.hq + hkv], angles[pos[:n]], neox)
        paged.store(want, geom, turned[:, lay.hq :].numpy(), heads[:, lay.hq + hkv :].double().cpu().numpy(), slots.numpy())
        assert np.array_equal(cache.view(torch.uint8).reshape(-1).cpu().numpy(), want)
        got = rows.unflatten(1, (-1, d))
        assert_close(got[:n, : lay.hq].double().cpu().numpy(), turned[:, : lay.hq].numpy(), atol=1e-5,
                     rtol=torch.finfo(dtype).eps / 2 * 1.01)
        assert torch.equal(rows[n:], before[n:]) and torch.equal(rows[:, lay.hq * d :], before[:, lay.hq * d :])
        meta = builder.build(0, common_metadata([n], [at], table, slots, DEV))
        out = torch.full((n, lay.hq * d), math.nan, dtype=dtype, device=DEV)
        impl.forward(None, q[:n], k[:n], v[:n], cache, meta, out)
        torch.cuda.synchronize()
        if n <= 10:
            ref = attention.decode_attention(got[:n, : lay.hq].float().cpu().numpy(), want, geom, table.numpy(), [at], n)
            assert_close(out.view(n, lay.hq, d).double().cpu().numpy(), ref)


def test_refusals():
    lay = PageLayout(4, 128)
    impl, cache = make_impl(), vllm_cache(2, 64, lay, DEV)
    rows = torch.zeros((4, 32 * 128), dtype=torch.float16, device=DEV)
    q, k, v = rows.split([24 * 128, 512, 512], 1)
    pos, table = torch.zeros(4, dtype=torch.int64, device=DEV), torch.ones((9, 128), device=DEV)
    slots = torch.zeros(5, dtype=torch.int64, device=DEV)
    with pytest.raises(RuntimeError, match="shorter than slot_mapping"):
        impl.do_rope_and_kv_cache_update(None, q, k, v, pos, table, True, cache, slots)
    with pytest.raises(RuntimeError, match="slot_mapping rank 2"):
        impl.do_rope_and_kv_cache_update(None, q, k, v, pos, table, True, cache, slots[None, :4])
    with pytest.raises(RuntimeError, match="multiple of 16"):
        impl.do_rope_and_kv_cache_update(None, q, k, v, pos, table[:, :24], True, cache, slots[:4])
    impl.do_rope_and_kv_cache_update(None, q, k, v, pos, table, True, cache, slots[:0])
    assert not cache.any()

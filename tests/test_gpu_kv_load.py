"""kv_load_paged against the dequantization formula in 64 bits.

K = code * k_scale is one fp32 product, V = (nibble - v_zero) * v_scale an fp32
difference and a product; a 16-bit output rounds once more.  Each rounding is
off by at most half a step of its type.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from gpu_cases import Cache, DEV, fill_sequence, random_tables
from k8v4_v030.layout import PAGE, PageLayout

pytestmark = pytest.mark.gpu

SENTINEL = 777.0


def build(ops, hkv, d, lens, ppb=1, seed=0):
    gen = torch.Generator().manual_seed(seed)
    blocks = sum(-(-n // (PAGE * ppb)) for n in lens)
    cache = Cache((blocks + 3) * ppb, PageLayout(hkv, d))
    table = random_tables(gen, lens, cache.num_pages, ppb)
    for b, n in enumerate(lens):
        fill_sequence(ops, cache, gen, table[b], n, ppb)
    torch.cuda.synchronize()
    return cache, table


def rows64(cache, table, ppb, firsts, counts):
    """float64 K and V rows on the CPU; a token outside the table or the cache is zeros."""
    v = {name: x.cpu() for name, x in cache.views.items()}
    hkv, d = cache.layout.hkv, cache.layout.head_dim
    ks, vs = [], []
    for b, (f, n) in enumerate(zip(firsts, counts)):
        for t in range(f, f + n):
            page = t // PAGE
            phys = -1
            if 0 <= t < table.shape[1] * ppb * PAGE:
                phys = int(table[b, page // ppb]) * ppb + page % ppb
            if not 0 <= phys < cache.num_pages:
                ks.append(torch.zeros(hkv, d, dtype=torch.float64))
                vs.append(torch.zeros(hkv, d, dtype=torch.float64))
                continue
            r = t % PAGE
            ks.append(v["k"][phys, r].double() * v["k_scale"][phys, r].double()[:, None])
            byte = v["v"][phys, r]
            nib = torch.stack((byte & 15, byte >> 4), -1).flatten(-2).double()
            vs.append((nib - v["v_zero"][phys, r].double()[:, None]) * v["v_scale"][phys, r].double()[:, None])
    if not ks:
        return torch.zeros(0, hkv, d, dtype=torch.float64), torch.zeros(0, hkv, d, dtype=torch.float64)
    return torch.stack(ks), torch.stack(vs)


def assert_rounded(got, want, roundings32):
    """|got - want| within half a step of the output type and of ``roundings32`` fp32 roundings."""
    rel = roundings32 * 2.0**-24
    low = 0.0
    if got.dtype != torch.float32:
        rel += torch.finfo(got.dtype).eps / 2
        low = 2.0**-25 if got.dtype == torch.float16 else 0.0  # half of fp16's subnormal step
    err = (got.cpu().double() - want).abs()
    assert bool((err <= rel * (1 + 2.0**-20) * want.abs() + low).all()), float((err - rel * want.abs()).max())


def index(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def starts_of(counts, first=0):
    return index(list(np.cumsum([first, *counts])))


CASES = [
    # hkv, D, out type, pages per entry, sequence lengths, first tokens, counts
    (4, 128, torch.float16, 1, [500], [0], [500]),
    (4, 128, torch.bfloat16, 1, [130, 1, 64, 700], [0, 0, 0, 300], [130, 1, 64, 400]),
    (2, 256, torch.bfloat16, 33, [2113, 90, 5000], [2000, 0, 63], [113, 0, 129]),
    (2, 128, torch.float32, 2, [65, 200, 3, 129], [0, 64, 2, 128], [65, 65, 1, 1]),
    (4, 256, torch.float16, 1, [33, 64, 65], [31, 0, 1], [1, 64, 64]),
    (4, 256, torch.float32, 3, [400], [100], [257]),
]


@pytest.mark.parametrize("hkv,d,dtype,ppb,lens,firsts,counts", CASES)
def test_rows_match_the_formula(gpu_ops, hkv, d, dtype, ppb, lens, firsts, counts):
    cache, table = build(gpu_ops, hkv, d, lens, ppb)
    n = sum(counts)
    k = torch.full((n, hkv, d), SENTINEL, dtype=dtype, device=DEV)
    v = torch.full_like(k, SENTINEL)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), index(firsts), starts_of(counts), ppb, k, v)
    kw, vw = rows64(cache, table, ppb, firsts, counts)
    assert_rounded(k, kw, 1)
    assert_rounded(v, vw, 2)


def test_round_trip_of_a_store(gpu_ops):
    """A store of the rows read back writes the same K codes again (V: values half a step away at most)."""
    cache, table = build(gpu_ops, 4, 128, [200, 77])
    counts = [200, 77]
    k = torch.empty((277, 4, 128), dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, starts_of(counts), 1, k, v)
    other = Cache(cache.num_pages, cache.layout)
    t = torch.cat([torch.arange(200), torch.arange(77)])
    b = torch.cat([torch.zeros(200, dtype=torch.long), torch.ones(77, dtype=torch.long)])
    slots = table[b, t // PAGE].long() * PAGE + t % PAGE
    other.store(gpu_ops, k, v, slots.to(DEV))
    torch.cuda.synchronize()
    p, r = slots // PAGE, slots % PAGE
    assert torch.equal(other.views["k"].cpu()[p, r], cache.views["k"].cpu()[p, r])
    k2, v2 = torch.empty_like(k), torch.empty_like(v)
    gpu_ops.kv_load_paged(*other.region_args(), table.to(DEV), None, starts_of(counts), 1, k2, v2)
    # A row read back spans (M - m) steps s, m and M its lowest and highest code:
    # 0 and 15, or less where the first store's zero point was rounded, which
    # leaves an end code unused.  Stored again its step is s' = s (M - m) / 15 <=
    # s; a code is within half of s' of its value, the end values too: lo / s' and
    # hi / s' are 15 apart, so with the zero point z' within half of -lo / s'
    # neither end passes the codes 0 .. 15 by more than a half, all a clamp takes
    # away.  The fp16 roundings of the two reads add 2^-11 of at most 16 steps
    # each.  Proof that s / 2 + 16 s 2^-9 holds: s' / 2 + 2 * 16 s 2^-11 <= it.
    step = cache.views["v_scale"].cpu()[p, r].double()[..., None]
    off = (v2.cpu().double() - v.cpu().double()).abs()
    assert bool((off <= step * (0.5 + 16 * 2.0**-9)).all())
    # Where the codes 0 and 15 are both used the step is the same, and so are the values.
    packed = cache.views["v"].cpu()[p, r]
    nib = torch.stack((packed & 15, packed >> 4), -1).flatten(-2)
    full = (nib.amin(-1) == 0) & (nib.amax(-1) == 15)
    assert bool(full.any()) and bool((off[full] <= (step * 16 * 2.0**-9).expand_as(off)[full]).all())


def test_rows_of_no_sequence_stay(gpu_ops):
    cache, table = build(gpu_ops, 4, 128, [100, 40])
    k = torch.full((150, 4, 128), SENTINEL, dtype=torch.bfloat16, device=DEV)
    v = torch.full_like(k, SENTINEL)
    # Rows 0..4 lie before the first sequence, 95.. behind the last.
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), index([10, 0]), index([5, 65, 95]), 1, k, v)
    kw, vw = rows64(cache, table, 1, [10, 0], [60, 30])
    assert_rounded(k[5:95], kw, 1)
    assert_rounded(v[5:95], vw, 2)
    for x in (k, v):
        assert bool((x[:5] == SENTINEL).all()) and bool((x[95:] == SENTINEL).all())


def test_row_starts_past_the_outputs_write_nothing_there(gpu_ops):
    """Counts that do not fit the outputs are cut off at their end."""
    cache, table = build(gpu_ops, 2, 128, [300])
    whole = torch.full((128, 2, 128), SENTINEL, dtype=torch.float16, device=DEV)
    k, v = whole[:70], torch.empty((70, 2, 128), dtype=torch.float16, device=DEV)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([0, 300]), 1, k, v)
    kw, _ = rows64(cache, table, 1, [0], [70])
    assert_rounded(k, kw, 1)
    assert bool((whole[70:] == SENTINEL).all())


def test_tokens_outside_the_table_and_the_cache_are_zeros(gpu_ops):
    cache, table = build(gpu_ops, 4, 128, [300, 300])
    table[0, 1] = -1
    table[0, 3] = cache.num_pages
    table[1, 0] = 2**31 - 1
    firsts, counts = [0, 250], [300, 200]  # row 1 runs past its table
    k = torch.full((500, 4, 128), SENTINEL, dtype=torch.float32, device=DEV)
    v = torch.full_like(k, SENTINEL)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), index(firsts), starts_of(counts), 1, k, v)
    kw, vw = rows64(cache, table, 1, firsts, counts)
    assert bool((kw[64:128] == 0).all()) and bool((kw[-100:] == 0).all())
    assert_rounded(k, kw, 1)
    assert_rounded(v, vw, 2)
    # A first token below zero reads zeros up to token 0.
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), index([-5, 0]), index([0, 20, 20]), 1, k, v)
    kw, _ = rows64(cache, table, 1, [-5], [20])
    assert bool((kw[:5] == 0).all())
    assert_rounded(k[:20], kw, 1)


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_strided_and_misaligned_outputs(gpu_ops, dtype):
    cache, table = build(gpu_ops, 2, 128, [100])
    kw, vw = rows64(cache, table, 1, [0], [100])
    fused = torch.full((100, 5 * 256), SENTINEL, dtype=dtype, device=DEV)
    k, v = fused[:, 256:512].unflatten(1, (2, 128)), fused[:, 768:1024].unflatten(1, (2, 128))
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([0, 100]), 1, k, v)
    assert_rounded(k, kw, 1)
    assert_rounded(v, vw, 2)
    for cols in (slice(0, 256), slice(512, 768), slice(1024, 1280)):
        assert bool((fused[:, cols] == SENTINEL).all())
    flat = torch.full((100 * 259 + 8,), SENTINEL, dtype=dtype, device=DEV)
    k = flat[1:].as_strided((100, 2, 128), (259, 128, 1), 1)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([0, 100]), 1, k, None)
    assert_rounded(k, kw, 1)
    rest = flat[: 1 + 100 * 259][1:].view(100, 259)[:, 256:]
    assert bool((rest == SENTINEL).all()) and float(flat[0]) == SENTINEL


def test_one_side_alone(gpu_ops):
    cache, table = build(gpu_ops, 2, 256, [70])
    both = [torch.empty((70, 2, 256), dtype=torch.bfloat16, device=DEV) for _ in range(2)]
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([0, 70]), 1, *both)
    k, v = torch.empty_like(both[0]), torch.empty_like(both[1])
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([0, 70]), 1, k, None)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([0, 70]), 1, None, v)
    assert torch.equal(k, both[0]) and torch.equal(v, both[1])


def test_many_short_sequences(gpu_ops):
    """More sequences than rows of a work-group, empty ones among them."""
    gen = torch.Generator().manual_seed(5)
    lens = [int(x) for x in torch.randint(1, 12, (200,), generator=gen)]
    cache, table = build(gpu_ops, 2, 128, lens)
    counts = [0 if i % 7 == 3 else n for i, n in enumerate(lens)]
    n = sum(counts)
    k = torch.empty((n, 2, 128), dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, starts_of(counts), 1, k, v)
    kw, vw = rows64(cache, table, 1, [0] * len(lens), counts)
    assert_rounded(k, kw, 1)
    assert_rounded(v, vw, 2)


def test_large_values_round_as_a_conversion_does(gpu_ops):
    """Planes that take V past fp16's range give infinities, as .to(float16) does."""
    cache, table = build(gpu_ops, 2, 128, [64])
    cache.views["v_scale"].fill_(131008.0 / 15)
    cache.views["k_scale"].fill_(600.0)
    k = torch.empty((64, 2, 128), dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([0, 64]), 1, k, v)
    kw, vw = rows64(cache, table, 1, [0], [64])
    assert torch.equal(k.cpu(), kw.float().half()) and torch.equal(v.cpu(), vw.float().half())
    assert bool(torch.isinf(k).any()) and bool(torch.isinf(v).any())


def test_on_another_stream_and_in_a_graph(gpu_ops):
    cache, table = build(gpu_ops, 4, 128, [400, 300])
    table = table.to(DEV)
    firsts, rows = index([0, 100]), index([0, 200, 300])
    k = torch.empty((300, 4, 128), dtype=torch.float16, device=DEV)
    v = torch.empty_like(k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    call = gpu_ops.bind_kv_load_paged(*cache.region_args(), table, firsts, rows, 1, k, v)
    with torch.cuda.stream(side):
        call()
    side.synchronize()
    kw, vw = rows64(cache, table.cpu(), 1, [0, 100], [200, 100])
    assert_rounded(k, kw, 1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for f, (a, b) in (([3, 0], (120, 130)), ([0, 299], (299, 300)), ([64, 64], (0, 64))):
        firsts.copy_(index(f))
        rows.copy_(index([0, a, b]))
        k.fill_(SENTINEL)
        v.fill_(SENTINEL)
        graph.replay()
        torch.cuda.synchronize()
        kw, vw = rows64(cache, table.cpu(), 1, f, [a, b - a])
        assert_rounded(k[:b], kw, 1)
        assert_rounded(v[:b], vw, 2)
        assert bool((k[b:] == SENTINEL).all()) and bool((v[b:] == SENTINEL).all())


def test_offsets_past_32_bits(gpu_ops):
    """Pages behind the first 4 GiB of a pool and rows behind the first 2^31 output elements."""
    lay = PageLayout(4, 256)
    pages = (2**32 + 2**28) // lay.page_bytes
    cache = Cache(pages, lay)
    gen = torch.Generator().manual_seed(7)
    table = torch.tensor([[pages - 1, pages - 2]], dtype=torch.int32)
    fill_sequence(gpu_ops, cache, gen, table[0], 100)
    views = {name: x[-2:].cpu() for name, x in cache.views.items()}
    n = 2**31 // (4 * 256) + 1000
    k = torch.zeros((n, 4, 256), dtype=torch.float16, device=DEV)
    gpu_ops.kv_load_paged(*cache.region_args(), table.to(DEV), None, index([n - 100, n]), 1, k, None)
    t = torch.arange(100)
    page = 1 - t // PAGE
    want = views["k"][page, t % PAGE].double() * views["k_scale"][page, t % PAGE].double()[..., None]
    assert_rounded(k[-100:], want, 1)
    assert not bool(k[-101].any()) and not bool(k[:1000].any())


@pytest.mark.parametrize("batch", [1, 2, 255, 256, 257, 512, 513, 1000])
def test_every_row_finds_its_sequence(gpu_ops, batch):
    """Ragged and empty sequences around the number the kernel's first search covers
    (256): every row holds its own sequence's token, found by the codes alone."""
    hkv, d = 2, 128
    counts = [(7 * i + i // 5) % 4 for i in range(batch)]
    counts[-1] = 3
    cache = Cache(batch, PageLayout(hkv, d))
    cache.views["k_scale"].fill_(1.0)
    cache.views["v_scale"].fill_(1.0)
    # Page p's token r: K codes hold p % 100 and r, V nibbles p // 100.
    page = torch.arange(batch, device=DEV, dtype=torch.int8) if batch < 100 else (
        torch.arange(batch, device=DEV) % 100).to(torch.int8)
    cache.views["k"][..., 0] = page[:, None, None]
    cache.views["k"][..., 1] = torch.arange(PAGE, device=DEV, dtype=torch.int8)[None, :, None]
    cache.views["v"][..., 0] = (torch.arange(batch, device=DEV) // 100).to(torch.uint8)[:, None, None]
    table = torch.randperm(batch, generator=torch.Generator().manual_seed(batch)).to(torch.int32)
    firsts = [(3 * i) % 60 for i in range(batch)]
    k = torch.full((sum(counts) + 2, hkv, d), SENTINEL, device=DEV)
    v = torch.full_like(k, SENTINEL)
    gpu_ops.kv_load_paged(*cache.region_args(), table[:, None].to(DEV), index(firsts), starts_of(counts, 1), 1, k, v)
    torch.cuda.synchronize()
    want = torch.tensor([(int(table[b]) % 100, firsts[b] + j, int(table[b]) // 100)
                         for b, n in enumerate(counts) for j in range(n)], dtype=torch.float32)
    got = torch.cat((k[1:-1, 0, :2], v[1:-1, 0, :1]), 1).cpu()
    assert torch.equal(got, want)
    for x in (k, v):
        assert bool((x[0] == SENTINEL).all()) and bool((x[-1] == SENTINEL).all())

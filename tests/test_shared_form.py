"""Which of its two forms int8k_int4v_attn_shared takes (the library's rule, no GPU)."""
from __future__ import annotations

import pytest

from k8v4_v030.layout import PAGE
from k8v4_v030.ops_api import ops

# (KV heads, head dim, sequences, query tokens): pages at which eight tokens at a time
# were measured the faster form by 4 % or more, and pages at which many rows were.
MEASURED = [
    (4, 128, 8, 1, (625, 1024, 2048), (8, 16, 32, 64, 96, 128, 192)),
    (4, 128, 16, 1, (1024, 2048), (8, 64, 128, 192, 256, 384)),
    (4, 128, 32, 1, (), (8, 64, 256, 625, 2048)),
    (4, 128, 5, 7, (8, 16), (384, 625, 1024, 2048)),
    (4, 128, 64, 1, (8, 16, 32), (384, 625, 1024, 2048)),
    (4, 128, 16, 4, (8, 16, 32, 64, 96, 128), (384, 625, 1024, 2048)),
    (4, 128, 128, 1, (8, 16, 32), (128, 192, 256, 625, 2048)),
    (4, 128, 64, 4, (), (8, 16, 32, 64, 96, 128, 192, 256, 625, 2048)),
    (2, 128, 8, 1, (1024, 2048), (8, 16, 32, 64, 256, 384)),
    (2, 128, 48, 1, (8, 64, 128, 192, 256), (625, 1024, 2048)),
    (2, 128, 64, 1, (8, 64, 128), (625, 1024, 2048)),
    (2, 128, 128, 1, (8, 64, 128, 192), (625, 1024, 2048)),
    (2, 128, 256, 1, (8, 64, 128), (384, 625, 2048)),
    (2, 128, 64, 4, (8, 16, 32, 64), (192, 256, 384, 625, 2048)),
    (2, 256, 8, 1, (625, 1024, 2048), (8, 16, 32, 64)),
    (2, 256, 16, 1, (), (8, 32, 64, 256, 625, 2048)),
    (2, 256, 24, 1, (8, 64, 128, 192, 256), (625, 1024, 2048)),
    (2, 256, 64, 1, (8, 32, 64, 128), (384, 625, 2048)),
    (2, 256, 128, 1, (8, 16, 32), (128, 192, 256, 384, 625, 2048)),
    (2, 256, 64, 4, (8, 16), (64, 96, 128, 192, 256, 2048)),
    (4, 256, 8, 1, (625, 1024, 2048), (8, 64, 128, 192, 256)),
    (4, 256, 16, 1, (), (8, 64, 256, 1024)),
    (4, 256, 128, 1, (), (8, 64, 256, 1024, 2048)),
]


@pytest.mark.parametrize("hkv,d,batch,q_len,few,many", MEASURED)
def test_the_form_measured_faster_is_taken(hkv, d, batch, q_len, few, many):
    takes = ops().attn_shared_many_rows
    for pages in few:
        assert not takes(batch, q_len, hkv, d, pages * PAGE), pages
    for pages in many:
        assert takes(batch, q_len, hkv, d, pages * PAGE), pages


@pytest.mark.parametrize("hkv,d", [(2, 128), (4, 128), (2, 256), (4, 256)])
def test_the_form_counts_whole_pages(hkv, d):
    takes = ops().attn_shared_many_rows
    for prefix in (0, 1, PAGE - 1):
        assert not takes(16, 1, hkv, d, prefix)
    for batch in (8, 48, 300):
        for pages in (1, 31, 384, 1000):
            assert takes(batch, 1, hkv, d, pages * PAGE) == takes(batch, 1, hkv, d, pages * PAGE + PAGE - 1)


def test_the_form_of_bad_shapes():
    lib = ops()._lib
    for bad in ((0, 1, 4, 128, 64), (1, 0, 4, 128, 64), (1, 11, 4, 128, 64), (1, 1, 3, 128, 64), (1, 1, 4, 64, 64),
                (2**21, 1, 4, 128, 64), (1, 1, 4, 128, -1), (1, 2**30, 4, 128, 64), (1, 1, 4, 128, 2**31)):
        assert lib.k8v4_attn_shared_many_rows(*bad) == -1
    with pytest.raises(RuntimeError, match="shared-prefix plan"):
        ops().attn_shared_many_rows(0, 1, 4, 128, 64)

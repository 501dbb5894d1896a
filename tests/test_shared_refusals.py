"""Arguments that int8k_int4v_attn_shared refuses with a message (host checks, no GPU)."""
from __future__ import annotations

import pytest
import torch

from k8v4_v030.cache_views import bind_regions
from k8v4_v030.layout import PageLayout
from k8v4_v030.ops_api import ops
from test_operator_checks import lib, refused, shared  # noqa: F401


@pytest.mark.parametrize("q_len", [2**30, 715827883, 2**31 - 1, -2**31])
def test_query_lengths_whose_rows_overflow(lib, q_len):  # noqa: F811
    """6 x 715,827,883 is 2 in 32 bits."""
    refused(lib, shared, "q_len*GQA exceeds BM", q_len=q_len)
    assert lib.k8v4_attn_shared_workspace_bytes(4, q_len, 4, 128) == -1
    assert lib.k8v4_attn_shared_many_rows(4, q_len, 4, 128, 640) == -1


def test_a_prefix_without_its_table():
    lay = PageLayout(2, 128)
    regions = [bind_regions(torch.zeros(3 * lay.page_bytes, dtype=torch.int8), lay)[n]
               for n in ("k", "k_scale", "v", "v_scale", "v_zero")]
    q = torch.zeros(4, 12, 128, dtype=torch.float16)
    rest = (torch.zeros((2, 3), dtype=torch.int32), torch.zeros(2, dtype=torch.int32), torch.zeros(64), q.clone(), 2, 1)
    with pytest.raises(RuntimeError, match="prefix_table must be a contiguous int32 row"):
        ops().int8k_int4v_attn_shared(q, *regions, None, 64, *rest)
    with pytest.raises(RuntimeError, match="GPU tensors"):  # no whole page: not needed
        ops().int8k_int4v_attn_shared(q, *regions, None, 63, *rest)

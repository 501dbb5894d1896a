"""What the vLLM backend decides about a prefix that all requests share (no GPU)."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from backend_cases import backend, common_metadata, make_builder
from k8v4_v030 import plan
from k8v4_v030.layout import PAGE, PageLayout
from k8v4_v030.ops_api import ops
from k8v4_v030.scratch import clear_scratch, get_scratch


@pytest.fixture(autouse=True)
def no_scratch():
    clear_scratch()
    yield
    clear_scratch()


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 256)])
def test_the_rule_counts_the_bytes_not_read_again(hkv, d):
    lay = PageLayout(hkv, d)
    pages = -(-plan.SHARED_PREFIX_MIN_SAVED // (31 * lay.page_bytes))
    assert plan.shared_prefix_pays(32, pages * PAGE, lay)
    assert plan.shared_prefix_pays(32, pages * PAGE + PAGE - 1, lay)
    assert not plan.shared_prefix_pays(32, pages * PAGE - 1, lay)  # the last page is not whole
    assert not plan.shared_prefix_pays(31, pages * PAGE - 1, lay)
    for few in (0, 1):
        assert not plan.shared_prefix_pays(few, 1 << 30, lay)
    for none in (0, -64, 63):
        assert not plan.shared_prefix_pays(1 << 10, none, lay)


def test_the_engine_is_told_when_it_pays():
    b = make_builder(hkv=4, head=128, max_model_len=131072, max_seqs=64)
    long = 65536
    assert b.use_cascade_attention(long, np.ones(48, dtype=np.int32), num_query_heads=24, num_kv_heads=4,
                                   use_alibi=False, use_sliding_window=False, use_local_attention=False,
                                   num_sms=256, dcp_world_size=1)
    assert b.use_cascade_attention(long, [1] * 16 + [400])  # a prefill beside the decodes
    assert not b.use_cascade_attention(long, [400] * 16)  # nothing but prefills
    assert not b.use_cascade_attention(long, [1, 2] * 16)  # runs of one request each
    assert not b.use_cascade_attention(0, [1] * 48)
    assert not b.use_cascade_attention(long, [])
    for other in ("use_alibi", "use_sliding_window", "use_local_attention"):
        assert not b.use_cascade_attention(long, [1] * 48, **{other: True})
    assert not b.use_cascade_attention(long, [1] * 48, dcp_world_size=2)


@pytest.mark.parametrize("common,kept", [(65536, True), (0, False), (64, False)])
def test_the_builder_keeps_the_prefix_and_makes_its_workspace(common, kept):
    b = make_builder(hkv=4, head=128, max_model_len=131072, max_seqs=16)
    scratch = get_scratch(torch.device("cpu"), b.layout)
    before = scratch.nbytes
    table = torch.zeros((16, 1030), dtype=torch.int32)
    meta = b.build(common, common_metadata([2] * 16, [65600] * 16, table, torch.zeros(32, dtype=torch.int64), "cpu"))
    assert meta.common_prefix_len == common
    assert (scratch.nbytes > before) is kept
    if kept:
        ws = scratch.shared_ws()
        assert ws is scratch.shared_ws()  # one for all steps
        for q_len in range(1, 11):
            assert ws.numel() * 4 >= ops().attn_shared_workspace_bytes(16, q_len, 4, 128)
        assert scratch.nbytes == before + 4 * ws.numel()


def test_metadata_made_without_a_prefix_has_none():
    b = make_builder()
    cam = common_metadata([1, 1], [10, 20], torch.zeros((2, 4)), torch.zeros(2), "cpu")
    meta = backend.Xe2K8V4Metadata(cam.seq_lens, cam.slot_mapping, cam.block_table_tensor, cam.query_start_loc,
                                   (0, 1, 2), cam.seq_lens_cpu_upper_bound, 2, 1, 20, 1, 1, b.layout)
    assert meta.common_prefix_len == 0

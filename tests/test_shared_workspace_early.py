"""When the workspace of the shared-prefix decode is made (no GPU)."""
from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

from backend_cases import common_metadata, make_builder
from k8v4_v030.ops_api import ops
from k8v4_v030.scratch import clear_scratch, get_scratch


@pytest.fixture(autouse=True)
def no_scratch():
    clear_scratch()
    yield
    clear_scratch()


def builder(caching, disabled, hkv=4, d=128, **cfg):
    b = make_builder(hkv, d, kernel_block=None, max_model_len=131072, **cfg)
    if caching is not None:
        b.vllm_config.cache_config = SimpleNamespace(enable_prefix_caching=caching)
    if disabled is not None:
        b.vllm_config.model_config.disable_cascade_attn = disabled
    b.set_kernel_block_size(64)
    return b


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 256)])
@pytest.mark.parametrize("disabled", [None, False])
def test_made_with_the_others_where_the_engine_shares_prefixes(hkv, d, disabled):
    """No step has to allocate it: the scratch holds what a step over a prefix needs before the first one."""
    b = builder(True, disabled, hkv, d, max_seqs=16)
    scratch = get_scratch(torch.device("cpu"), b.layout)
    before = scratch.nbytes
    ws = scratch.shared_ws()
    assert scratch.nbytes == before  # it was there
    for q_len in range(1, 11):
        assert ws.numel() * 4 >= ops().attn_shared_workspace_bytes(16, q_len, hkv, d)
    table = torch.zeros((16, 1030), dtype=torch.int32)
    b.build(65536, common_metadata([2] * 16, [65600] * 16, table, torch.zeros(32, dtype=torch.int64), "cpu"))
    assert get_scratch(torch.device("cpu"), b.layout).shared_ws() is ws


def test_a_larger_scratch_has_one_too():
    builder(True, False, max_seqs=4)
    b = builder(True, False, max_seqs=64, max_batched=4096)
    scratch = get_scratch(torch.device("cpu"), b.layout)
    before = scratch.nbytes
    assert scratch.shared_ws().numel() * 4 >= ops().attn_shared_workspace_bytes(64, 1, 4, 128)
    assert scratch.nbytes == before


@pytest.mark.parametrize("caching,disabled", [(None, None), (False, False), (True, True)])
def test_not_made_for_engines_without_common_prefixes(caching, disabled):
    b = builder(caching, disabled)
    scratch = get_scratch(torch.device("cpu"), b.layout)
    before = scratch.nbytes
    scratch.shared_ws()
    assert scratch.nbytes > before

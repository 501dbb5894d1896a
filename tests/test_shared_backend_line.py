"""Which steps the backend takes out of the engine's captured graphs for a shared prefix (no GPU)."""
from __future__ import annotations

import enum

import pytest
import torch

from backend_cases import backend, common_metadata, make_builder
from k8v4_v030 import plan
from k8v4_v030.layout import PAGE, PageLayout
from k8v4_v030.scratch import clear_scratch

MIB = 1 << 20


class GraphMode(enum.Enum):
    """The names of the engine's graph modes."""

    NONE = 0
    PIECEWISE = 1
    FULL = 2
    FULL_DECODE_ONLY = (2, 0)
    FULL_AND_PIECEWISE = (2, 1)


@pytest.fixture(autouse=True)
def no_scratch():
    clear_scratch()
    yield
    clear_scratch()


def prefix_saving(mib, sequences, layout):
    """The shortest prefix of whole pages by which ``sequences`` save ``mib`` MiB."""
    return -(-mib * MIB // ((sequences - 1) * layout.page_bytes)) * PAGE


def builder(mode, hkv=4, d=128, capture=(1, 2, 4, 8, 16, 32, 64, 128, 256, 512)):
    b = make_builder(hkv, d, max_model_len=131072, max_seqs=256, capture=capture)
    if mode is not None:
        b.vllm_config.compilation_config.cudagraph_mode = mode
    return b


@pytest.mark.parametrize("mode,line", [(GraphMode.NONE, 192), (GraphMode.PIECEWISE, 192), (GraphMode.FULL, 768),
                                       (GraphMode.FULL_DECODE_ONLY, 768), (GraphMode.FULL_AND_PIECEWISE, 384),
                                       (None, 768)])
@pytest.mark.parametrize("hkv,d,count,q_len", [(4, 128, 64, 1), (2, 256, 32, 4), (2, 128, 32, 10), (4, 256, 256, 1)])
def test_a_step_leaves_its_graph_only_where_that_pays(mode, line, hkv, d, count, q_len):
    b = builder(mode, hkv, d)
    lay = PageLayout(hkv, d)
    prefix = prefix_saving(line, count, lay)
    assert b.use_cascade_attention(prefix, [q_len] * count)
    assert not b.use_cascade_attention(prefix - 1, [q_len] * count)


@pytest.mark.parametrize("mode", [GraphMode.FULL, GraphMode.FULL_AND_PIECEWISE, None])
def test_steps_that_no_graph_serves_keep_the_ops_own_line(mode):
    lay = PageLayout(4, 128)
    prefix = prefix_saving(192, 64, lay)
    b = builder(mode)
    assert not b.use_cascade_attention(prefix, [1] * 64)
    assert b.use_cascade_attention(prefix, [1] * 64 + [400])  # a prefill beside the decodes
    assert b.use_cascade_attention(prefix, [1] * 64 + [3] * 2)  # two runs
    assert b.use_cascade_attention(prefix, [9] * 64)  # 576 tokens: more than any graph holds
    assert not b.use_cascade_attention(prefix, [8] * 64)
    assert builder(mode, capture=()).use_cascade_attention(prefix, [1] * 64)  # no graphs at all
    assert not b.use_cascade_attention(prefix - 1, [1] * 64 + [400])


def test_an_accepted_step_reads_the_prefix_once(monkeypatch):
    """The step's metadata follow the op's line: what the engine was told of runs over the prefix."""
    b = builder(GraphMode.FULL)
    prefix = prefix_saving(192, 64, b.layout)
    table = torch.zeros((65, 40), dtype=torch.int32)
    meta = b.build(prefix, common_metadata([1] * 64 + [400], [prefix + 500] * 65, table,
                                           torch.zeros(464, dtype=torch.int64), "cpu"))
    assert [backend._reads_prefix_once(meta, run) for run in meta.decode_runs] == [True]


@pytest.mark.parametrize("prefix", [0, -64, 63, 64])
def test_steps_without_a_prefix_are_not_planned(monkeypatch, prefix):
    b = builder(GraphMode.FULL)

    def fail(*args):
        raise AssertionError("planned a step that shares nothing")

    monkeypatch.setattr(backend, "plan_step", fail)
    assert not b.use_cascade_attention(prefix, [1] * 200)


def test_the_lines_are_in_order():
    assert plan.SHARED_PREFIX_MIN_SAVED < plan.SHARED_PREFIX_MIN_SAVED_PIECES < plan.SHARED_PREFIX_MIN_SAVED_EAGER

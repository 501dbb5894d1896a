"""What the operators of drafted trees refuse (host checks, no GPU)."""
from __future__ import annotations

from pathlib import Path

import pytest
import torch

from k8v4_v030 import ops_api
from k8v4_v030.cache_views import bind_regions
from k8v4_v030.layout import PageLayout

P = 0x10000  # a pointer that is never dereferenced
CACHE = dict(k=P, ks=P, v=P, vs=P, vz=P, pages=64, k_ps=52224, ks_ps=52224, v_ps=52224, vs_ps=52224, vz_ps=52224)


@pytest.fixture(scope="module")
def lib():
    if not Path(ops_api.library_path()).is_file():
        pytest.skip("library not built (run __graft_entry__.build())")
    return ops_api.load_library()


def refused(lib, call, text, code=1, **over):
    assert call(lib, **over) == code
    assert text in lib.k8v4_last_error().decode()


def rope(lib, **over):
    a = dict(q=P, k_rows=P, v_rows=P, dtype=1, q_stride=4096, k_stride=4096, v_stride=4096, pos=P, pos64=1, table=P,
             table_dtype=2, rows=100, table_stride=128, rot=128, neox=1, slots=P, ntok=5, hkv=4, d=128, **CACHE,
             q_out=P, q_out_stride=4096, stream=None)
    a.update(over)
    return lib.k8v4_rope_kv_store_paged(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(hkv=3), "KV head count 3"), (dict(d=64), "head dim 64"), (dict(dtype=2), "fp16 or bf16"),
    (dict(table_dtype=3), "cos_sin must be"), (dict(rot=0), "rotary dim 0"), (dict(rot=24), "rotary dim 24"),
    (dict(rot=144), "rotary dim 144"), (dict(rot=256, d=256, table_stride=255, q_stride=6144, q_out_stride=6144), "cos_sin rows"),
    (dict(rows=0), "cos_sin rows"), (dict(ntok=-1), "negative"), (dict(pages=-1), "negative"), (dict(k_rows=None), "null"),
    (dict(pos=None), "null"), (dict(table=None), "null"), (dict(slots=None), "null"), (dict(vz=None), "null"),
    (dict(q=None), "go together"), (dict(q_out=None), "go together"), (dict(k_stride=511), "k/v token stride"),
    (dict(v_stride=0), "k/v token stride"), (dict(q_stride=3000), "q token stride"), (dict(q_out_stride=1), "q token stride"),
    (dict(q_out_stride=5000), "not another view"), (dict(q=P + 1), "misaligned"), (dict(v_rows=P + 1), "misaligned"), (dict(table=P + 2), "misaligned"),
    (dict(pos=P + 4), "misaligned"), (dict(pos=P + 2, pos64=0), "misaligned"), (dict(slots=P + 4), "misaligned"),
    (dict(k=P + 8), "misaligned"), (dict(v=P + 4), "misaligned"), (dict(k_ps=52232), "page strides"),
    (dict(v_ps=52228), "page strides"), (dict(ntok=2**40), "too many tokens"),
])
def test_rope_refuses(lib, over, text):
    refused(lib, rope, text, **over)


def test_rope_of_nothing(lib):
    assert rope(lib, ntok=0) == 0 and rope(lib, ntok=0, k_rows=None) == 0


def tree(lib, **over):
    a = dict(q=P, q_dtype=0, q_stride=4096, **CACHE, bt=P, bt_stride=32, width=32, ppb=1, lens=P, masks=P, mask_stride=13,
             batch=2, nodes=13, hkv=4, d=128, out=P, out_dtype=0, out_stride=4096, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(over)
    return lib.k8v4_attn_tree(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(hkv=1), "KV head count 1"), (dict(d=192), "head dim 192"), (dict(nodes=0), "1 to 64 nodes"),
    (dict(nodes=65, mask_stride=65), "1 to 64 nodes"), (dict(ppb=0), "pages_per_block"), (dict(pages=0), "num_pages"),
    (dict(pages=2**31), "num_pages"), (dict(batch=0), "batch"), (dict(batch=2**21), "batch"), (dict(width=0), "width"),
    (dict(width=2**24, ppb=2, bt_stride=2**24), "width"), (dict(q_dtype=2), "q dtype"), (dict(out_dtype=3), "out dtype"),
    (dict(masks=None), "null"), (dict(lens=None), "null"), (dict(ws=None), "null"), (dict(q=P + 8), "16-byte"),
    (dict(q_stride=4100), "multiple of 8"), (dict(q_stride=8), "q token stride"), (dict(out_stride=8), "out token stride"),
    (dict(out=P + 1), "out misaligned"), (dict(bt_stride=31), "row stride"), (dict(mask_stride=12), "tree_masks row stride"),
    (dict(masks=P + 4), "misaligned"), (dict(lens=P + 2), "misaligned"), (dict(k=P + 8), "k_cache"), (dict(v_ps=2), "v_cache"),
    (dict(vs=P + 4), "scale planes"), (dict(k_ps=2**31), "page strides"), (dict(vz_ps=-8), "page strides"),
    (dict(ws=P + 8), "16-byte aligned"), (dict(batch=2**20, width=2**12, bt_stride=2**12), "too large"),
])
def test_tree_refuses(lib, over, text):
    refused(lib, tree, text, **over)


@pytest.mark.parametrize("hkv,d", [(4, 128), (2, 128), (2, 256), (4, 256)])
def test_tree_workspace(lib, hkv, d):
    stride = 6 * hkv * d
    for batch, nodes in ((1, 1), (3, 8), (7, 64), (200, 21)):
        need = lib.k8v4_attn_tree_workspace_bytes(batch, nodes, hkv, d)
        assert need > 0
        over = dict(hkv=hkv, d=d, batch=batch, nodes=nodes, mask_stride=nodes, q_stride=stride, out_stride=stride)
        refused(lib, tree, "tree workspace holds %d bytes, the batch needs %d" % (need - 1, need), code=2, ws_bytes=need - 1, **over)
    for bad in ((0, 1, hkv, d), (1, 0, hkv, d), (1, 65, hkv, d), (1, 1, 3, d), (1, 1, hkv, 64), (2**21, 1, hkv, d)):
        assert lib.k8v4_attn_tree_workspace_bytes(*bad) == -1


def accept(lib, **over):
    a = dict(drafts=P, int64=0, d_stride=9, parents=P, p_stride=9, counts=P, targets=P, t_stride=9, lens=P, batch=3, nodes=9,
             width=4, path=P, path_stride=4, out=P, out_stride=4, acc=P, nxt=P, stream=None)
    a.update(over)
    return lib.k8v4_accept_tree(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(nodes=0, width=0), "1 to 64 nodes"), (dict(nodes=65), "1 to 64 nodes"), (dict(width=0), "path width"),
    (dict(width=10), "path width"), (dict(batch=-1), "batch"), (dict(drafts=None), "null"), (dict(parents=None), "null"),
    (dict(targets=None), "null"), (dict(path=None), "null"), (dict(out=None), "null"), (dict(acc=None), "null"),
    (dict(lens=None), "next_lens needs seq_lens"), (dict(d_stride=8), "draft_tokens row"), (dict(p_stride=3), "parents row"),
    (dict(t_stride=0), "target_tokens row"), (dict(path_stride=3), "path row"), (dict(out_stride=3), "out_tokens row"),
    (dict(drafts=P + 4, int64=1), "misaligned"), (dict(targets=P + 4), "misaligned"), (dict(out=P + 4), "misaligned"),
    (dict(nxt=P + 2), "misaligned"),
])
def test_accept_refuses(lib, over, text):
    refused(lib, accept, text, **over)


def keep(lib, **over):
    a = dict(**CACHE, bt=P, bt_stride=32, width=32, ppb=1, starts=P, path=P, path_stride=6, path_width=6, acc=P, batch=3,
             hkv=4, d=128, stream=None)
    a.update(over)
    return lib.k8v4_kv_keep_paged(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(hkv=3), "KV head count 3"), (dict(d=100), "head dim 100"), (dict(ppb=0), "pages_per_block"), (dict(pages=0), "num_pages"),
    (dict(batch=-1), "batch"), (dict(path_width=-1), "path width"), (dict(width=0), "width"), (dict(width=2**30, ppb=2), "width"),
    (dict(path=None), "null"), (dict(starts=None), "null"), (dict(acc=None), "null"), (dict(v=None), "null"),
    (dict(bt_stride=3), "block_table row"), (dict(path_stride=5), "path row"), (dict(path=P + 2), "misaligned"),
    (dict(k=P + 8), "misaligned"), (dict(vz=P + 2), "misaligned"), (dict(v_ps=52228), "page strides"),
])
def test_keep_refuses(lib, over, text):
    refused(lib, keep, text, **over)


def logprobs(lib, **over):
    a = dict(logits=P, dtype=2, stride=1000, tokens=P, int64=1, rows=4, vocab=1000, top=5, lp=P, ranks=P, h=P, ids=P,
             ids_stride=5, lps=P, lps_stride=5, ws=P, ws_bytes=1 << 40, stream=None)
    a.update(over)
    return lib.k8v4_token_logprobs(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(dtype=3), "logits must be"), (dict(rows=-1), "rows"), (dict(rows=2**24 + 1), "rows"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=2**24 + 1), "vocabulary"), (dict(top=-1), "likeliest"), (dict(top=65), "likeliest"), (dict(logits=None), "null"),
    (dict(lp=None), "null"), (dict(ranks=None), "null"), (dict(ids=None), "null"), (dict(lps=None), "null"),
    (dict(stride=999), "logits row stride"), (dict(ids_stride=4), "row stride"), (dict(lps_stride=4), "row stride"),
    (dict(logits=P + 2), "misaligned"), (dict(ids=P + 4), "misaligned"), (dict(tokens=P + 4), "misaligned"),
    (dict(ws=P + 8), "16-byte"),
])
def test_logprobs_refuses(lib, over, text):
    refused(lib, logprobs, text, **over)


def test_logprobs_workspace(lib):
    need = lib.k8v4_token_logprobs_workspace_bytes(2, 100000, 8)
    assert need > 0
    refused(lib, logprobs, "workspace holds %d bytes, the rows need %d" % (need - 1, need), code=2, rows=2, vocab=100000,
            stride=100000, top=8, ids_stride=8, lps_stride=8, ws_bytes=need - 1)
    refused(lib, logprobs, "workspace", code=2, rows=2, vocab=100000, stride=100000, ws=None)
    assert lib.k8v4_token_logprobs_workspace_bytes(0, 100, 5) == 0
    for bad in ((-1, 100, 5), (1, 0, 5), (1, 2**24 + 1, 5), (1, 100, 65), (1, 100, -1), (2**24 + 1, 100, 5)):
        assert lib.k8v4_token_logprobs_workspace_bytes(*bad) == -1
    assert logprobs(lib, rows=0) == 0


# ------------------------------------------------------------- the op table's checks
@pytest.fixture(scope="module")
def cpu():
    """A small cache and op arguments on the CPU: all checks but the last pass."""
    lay = PageLayout(4, 128)
    v = bind_regions(torch.zeros(4 * lay.page_bytes, dtype=torch.int8), lay)
    views = [v[n] for n in ("k", "k_scale", "v", "v_scale", "v_zero")]
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)  # noqa: E731
    i64 = lambda *s: torch.zeros(s, dtype=torch.int64)  # noqa: E731
    rows = lambda n, h: torch.zeros((n, h, 128), dtype=torch.float16)  # noqa: E731
    return {
        "rope_kv_store_paged": [rows(3, 24), rows(3, 4), rows(3, 4), i64(3), torch.zeros(9, 128), True, i64(3), *views, rows(3, 24)],
        "int8k_int4v_attn_tree": [rows(6, 24), *views, i32(2, 3), i32(2), i64(2, 3), torch.zeros(64), rows(6, 24), 3, 1],
        "accept_tree": [i32(2, 5), i32(2, 5), i64(2, 5), i32(2), i32(2, 4), i64(2, 4), i32(2), i32(2)],
        "kv_keep_paged": [*views, i32(2, 3), i32(2), i32(2, 4), i32(2), 1],
        "token_logprobs": [torch.zeros(2, 50), i64(2), torch.zeros(4), torch.zeros(2), i32(2), torch.zeros(2), i64(2, 3), torch.zeros(2, 3)],
    }


OPS = ["rope_kv_store_paged", "int8k_int4v_attn_tree", "accept_tree", "kv_keep_paged", "token_logprobs"]


@pytest.mark.parametrize("name", OPS)
def test_cpu_tensors_are_refused(lib, cpu, name):
    with pytest.raises(RuntimeError, match="K8/V4 ops need GPU tensors, got a cpu tensor"):
        getattr(ops_api.ops(), name)(*cpu[name])


F16, BF16, F32, I32, I64 = torch.float16, torch.bfloat16, torch.float32, torch.int32, torch.int64


@pytest.mark.parametrize("name,at,value,text", [
    ("rope_kv_store_paged", 0, torch.zeros(3, 23, 128, dtype=F16), "HQ = 6"), ("rope_kv_store_paged", 0, None, "go together"),
    ("rope_kv_store_paged", 0, torch.zeros(3, 24, 128, dtype=BF16), "q/k_fp16 dtypes"),
    ("rope_kv_store_paged", 1, torch.zeros(4, 4, 128, dtype=F16), "v_fp16 must match"),
    ("rope_kv_store_paged", 2, torch.zeros(3, 4, 128, dtype=BF16), "dtypes differ"),
    ("rope_kv_store_paged", 3, torch.zeros(4, dtype=I64), "positions"), ("rope_kv_store_paged", 3, torch.zeros(3), "positions"),
    ("rope_kv_store_paged", 4, torch.zeros(9, 40), "multiple of 16"), ("rope_kv_store_paged", 4, torch.zeros(9, 256), "multiple of 16"),
    ("rope_kv_store_paged", 4, torch.zeros(9, 128, dtype=torch.float64), "cos_sin"),
    ("rope_kv_store_paged", 4, torch.zeros(128, 9).t(), "rows must be contiguous"),
    ("rope_kv_store_paged", 6, torch.zeros(3, dtype=I32), "slot_mapping int64"), ("rope_kv_store_paged", 6, torch.zeros(2, dtype=I64), "slot_mapping"),
    ("rope_kv_store_paged", 12, torch.zeros(3, 24, 128, dtype=F32), "q_out must match"),
    ("int8k_int4v_attn_tree", 0, torch.zeros(7, 24, 128, dtype=F16), "out shape"),
    ("int8k_int4v_attn_tree", 0, torch.zeros(6, 24, 128), "q_fp16 must be"), ("int8k_int4v_attn_tree", 11, 4, "B\\*nodes"),
    ("int8k_int4v_attn_tree", 11, 65, "1 to 64 nodes"), ("int8k_int4v_attn_tree", 12, 0, "pages_per_block"),
    ("int8k_int4v_attn_tree", 6, torch.zeros(3, 3, dtype=I32), "block_table"), ("int8k_int4v_attn_tree", 7, torch.zeros(2, dtype=I64), "seq_lens"),
    ("int8k_int4v_attn_tree", 8, torch.zeros(2, 3, dtype=I32), "tree_masks"), ("int8k_int4v_attn_tree", 8, torch.zeros(3, 2, dtype=I64).t(), "tree_masks"),
    ("int8k_int4v_attn_tree", 10, torch.zeros(6, 24, 128, dtype=I32), "out float16"),
    ("accept_tree", 0, torch.zeros(2, 5), "draft_tokens"), ("accept_tree", 0, torch.zeros(2, 65, dtype=I32), "1 to 64 nodes"),
    ("accept_tree", 1, torch.zeros(2, 4, dtype=I32), "parents"), ("accept_tree", 2, torch.zeros(2, 5, dtype=I32), "target_tokens"),
    ("accept_tree", 3, None, "next_lens needs seq_lens"), ("accept_tree", 4, torch.zeros(2, 6, dtype=I32), "W of 1"),
    ("accept_tree", 4, torch.zeros(2, 4, dtype=I64), "path int32"), ("accept_tree", 5, torch.zeros(2, 5, dtype=I64), "out_tokens"),
    ("accept_tree", 6, torch.zeros(3, dtype=I32), "accepted"), ("accept_tree", 7, torch.zeros(2, dtype=I64), "next_lens"),
    ("kv_keep_paged", 5, torch.zeros(2, 3, dtype=I64), "block_table"), ("kv_keep_paged", 6, torch.zeros(3, dtype=I32), "seq_starts"),
    ("kv_keep_paged", 7, torch.zeros(1, 4, dtype=I32), "path int32"), ("kv_keep_paged", 7, torch.zeros(4, 2, dtype=I32).t(), "path rows"),
    ("kv_keep_paged", 8, torch.zeros(2, dtype=I64), "accepted"), ("kv_keep_paged", 9, 0, "pages_per_block"),
    ("token_logprobs", 0, torch.zeros(2, 50, dtype=I32), "logits"), ("token_logprobs", 0, torch.zeros(50, 2).t(), "rows must be contiguous"),
    ("token_logprobs", 1, None, "go together"), ("token_logprobs", 1, torch.zeros(2), "tokens"), ("token_logprobs", 3, torch.zeros(3), "logprobs"),
    ("token_logprobs", 4, torch.zeros(2, dtype=I64), "ranks"), ("token_logprobs", 5, torch.zeros(2, dtype=F16), "entropy"),
    ("token_logprobs", 6, torch.zeros(2, 3, dtype=I32), "top_ids"), ("token_logprobs", 6, torch.zeros(2, 65, dtype=I64), "0 to 64"),
    ("token_logprobs", 7, torch.zeros(2, 4), "top_logprobs"), ("token_logprobs", 7, None, "go together"),
])
def test_op_table_refuses(lib, cpu, name, at, value, text):
    args = list(cpu[name])
    args[at] = value
    with pytest.raises(RuntimeError, match=text):
        getattr(ops_api.ops(), name)(*args)


def test_another_view_of_the_query_as_output(lib, cpu):
    args = list(cpu["rope_kv_store_paged"])
    buf = torch.zeros(9, 24, 128, dtype=F16)
    args[0], args[12] = buf[:3], buf[::2][:3]
    with pytest.raises(RuntimeError, match="not another view"):
        ops_api.ops().rope_kv_store_paged(*args)


def test_more_than_a_launch_takes_is_refused(lib):
    # 2^32 threads of a launch at most.
    refused(lib, rope, "too many tokens", ntok=1 << 27)
    refused(lib, rope, "too many tokens", ntok=1 << 26)  # its queries
    refused(lib, accept, "batch", batch=1 << 24)
    refused(lib, keep, "batch", batch=1 << 24)
    refused(lib, logprobs, "too many rows", rows=1 << 24)
    refused(lib, logprobs, "too many rows", rows=(1 << 24) // 2, vocab=1 << 19, stride=1 << 19)  # two slices a row
    assert lib.k8v4_token_logprobs_workspace_bytes((1 << 24) - 1, 1000, 5) == 0

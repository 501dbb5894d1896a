"""What int8k_int4v_attn_shared, kv_load_paged and verify_drafts refuse (host checks, no GPU)."""
from __future__ import annotations

from pathlib import Path

import pytest
import torch

from k8v4_v030 import ops_api
from k8v4_v030.cache_views import bind_regions
from k8v4_v030.layout import PageLayout

P = 0x10000  # a pointer that is never dereferenced


@pytest.fixture(scope="module")
def lib():
    if not Path(ops_api.library_path()).is_file():
        pytest.skip("library not built (run __graft_entry__.build())")
    return ops_api.load_library()


def refused(lib, call, text, code=1, **over):
    assert call(lib, **over) == code
    assert text in lib.k8v4_last_error().decode()


def load(lib, **over):
    a = dict(k=P, ks=P, v=P, vs=P, vz=P, pages=64, k_ps=52224, ks_ps=52224, v_ps=52224, vs_ps=52224, vz_ps=52224,
             bt=P, bt_stride=32, width=32, ppb=1, starts=None, rows_at=P, batch=2, hkv=4, d=128, k_out=P, v_out=P,
             dtype=0, k_stride=512, v_stride=512, rows=100, stream=None)
    a.update(over)
    return lib.k8v4_kv_load_paged(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(hkv=3), "unsupported per-GPU KV head count 3"), (dict(d=64), "unsupported head dim 64"),
    (dict(dtype=3), "out dtype"), (dict(ppb=0), "pages_per_block"), (dict(pages=0), "num_pages"),
    (dict(pages=2**31), "num_pages"), (dict(batch=-1), "batch"), (dict(rows=-1), "row count"),
    (dict(k_out=None, v_out=None), "null"), (dict(bt=None), "null"), (dict(rows_at=None), "null"),
    (dict(ks=None), "null"), (dict(vz=None), "null"), (dict(width=0), "width"), (dict(width=2**31), "width"),
    (dict(ppb=2**30), "width"), (dict(bt_stride=31), "row stride"), (dict(k_stride=511), "stride"),
    (dict(v_stride=0), "stride"), (dict(k=P + 8), "aligned"), (dict(v_ps=52220), "aligned"),
    (dict(vs=P + 2), "aligned"), (dict(ks_ps=52222), "aligned"), (dict(k_out=P + 1), "misaligned"),
    (dict(v_out=P + 2, dtype=2), "misaligned"), (dict(rows_at=P + 2), "misaligned"), (dict(starts=P + 1), "misaligned"),
    (dict(rows=2**40), "too many rows"),
])
def test_load_refuses(lib, over, text):
    refused(lib, load, text, **over)


def test_load_of_nothing(lib):
    assert load(lib, rows=0) == 0 and load(lib, batch=0) == 0


def verify(lib, **over):
    a = dict(target=P, dtype=2, t_seq=400, t_row=100, draft=P, d_seq=300, d_row=100, tokens=P, int64=0, tok=3,
             counts=P, u=P, u_stride=3, s=P, lens=P, batch=4, drafts=3, vocab=100, out=P, out_stride=4, acc=P, nxt=P,
             ws=P, ws_bytes=1 << 20, stream=None)
    a.update(over)
    return lib.k8v4_verify_drafts(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(dtype=3), "probabilities must be"), (dict(batch=-1), "batch"), (dict(batch=65536), "batch"),
    (dict(drafts=-1), "drafts"), (dict(drafts=64), "drafts"), (dict(vocab=0), "vocabulary"),
    (dict(vocab=2**24 + 1), "vocabulary"), (dict(target=None), "null"), (dict(tokens=None), "null"),
    (dict(u=None), "null"), (dict(s=None), "null"), (dict(out=None), "null"), (dict(acc=None), "null"),
    (dict(ws=None), "null"), (dict(lens=None), "next_lens needs seq_lens"), (dict(t_row=99), "target row stride"),
    (dict(t_seq=0), "target sequence stride"), (dict(d_row=0), "draft row stride"), (dict(d_seq=7), "draft sequence"),
    (dict(out_stride=3), "out_tokens"), (dict(tok=2), "draft_tokens"), (dict(u_stride=0), "accept_uniform"),
    (dict(target=P + 2), "misaligned"), (dict(out=P + 4), "misaligned"), (dict(tokens=P + 4, int64=1), "misaligned"),
    (dict(ws=P + 8), "16-byte"),
])
def test_verify_refuses(lib, over, text):
    refused(lib, verify, text, **over)


def test_verify_workspace(lib):
    assert verify(lib, batch=0) == 0
    need = lib.k8v4_verify_drafts_workspace_bytes(4, 100)
    assert need > 0
    refused(lib, verify, "verify workspace holds %d bytes" % (need - 1), code=2, ws_bytes=need - 1)
    for bad in ((-1, 10), (65536, 10), (1, 0), (1, 2**24 + 1)):
        assert lib.k8v4_verify_drafts_workspace_bytes(*bad) == -1


def shared(lib, **over):
    a = dict(q=P, q_dtype=0, q_stride=24 * 128, k=P, ks=P, v=P, vs=P, vz=P, pages=64, k_ps=52224, ks_ps=52224,
             v_ps=52224, vs_ps=52224, vz_ps=52224, pre=P, pre_width=8, pre_len=512, bt=P, bt_stride=32, width=32, ppb=1,
             lens=P, batch=4, q_len=2, hkv=4, d=128, out=P, out_dtype=0, out_stride=24 * 128, ws=P, ws_bytes=1 << 30,
             stream=None)
    a.update(over)
    return lib.k8v4_attn_shared(*a.values())


@pytest.mark.parametrize("over,text", [
    (dict(hkv=3), "unsupported per-GPU KV head count 3"), (dict(d=64), "head dim"), (dict(q_len=11), "q_len*GQA"),
    (dict(q_len=0), "q_len*GQA"), (dict(ppb=0), "pages_per_block"), (dict(pages=0), "num_pages"),
    (dict(batch=0), "batch"), (dict(batch=2**21), "batch"), (dict(width=0), "width"), (dict(width=2**25), "width"),
    (dict(pre_len=-1), "negative prefix"), (dict(pre_len=2**40), "prefix too long"),
    (dict(pre_len=576), "prefix_table has 8 entries, the prefix of 576 tokens needs 9"),
    (dict(pre=None), "null"), (dict(q=None), "null"), (dict(lens=None), "null"), (dict(ws=None), "null"),
    (dict(q_dtype=2), "q dtype"), (dict(out_dtype=5), "out dtype"), (dict(q=P + 8), "16-byte"),
    (dict(q_stride=24 * 128 + 4), "multiple of 8"), (dict(q_stride=128), "q token stride"),
    (dict(out_stride=128), "out token stride"), (dict(out=P + 1), "out misaligned"), (dict(bt_stride=31), "row stride"),
    (dict(bt=P + 2), "index arrays"), (dict(pre=P + 1), "index arrays"), (dict(k=P + 8), "k_cache"),
    (dict(v_ps=52222), "v_cache"), (dict(vs=P + 4), "scale planes"), (dict(ws=P + 8), "workspace must be"),
    (dict(batch=2**16, width=2**15, bt_stride=2**15), "too large"),
    (dict(k_ps=2**31), "page strides"), (dict(vz_ps=-52224), "page strides"), (dict(ks_ps=2**32), "page strides"),
])
def test_shared_refuses(lib, over, text):
    refused(lib, shared, text, **{"ws_bytes": 1 << 40, **over})


@pytest.mark.parametrize("hkv,d", [(2, 128), (4, 128), (2, 256), (4, 256)])
def test_shared_workspace(lib, hkv, d):
    size = lib.k8v4_attn_shared_workspace_bytes
    for bad in ((0, 1, hkv, d), (1, 0, hkv, d), (1, 11, hkv, d), (1, 1, 3, d), (1, 1, hkv, 64), (2**21, 1, hkv, d)):
        assert size(*bad) == -1
    last = 0
    for batch in (1, 2, 7, 8, 9, 64, 1000):
        need = size(batch, 3, hkv, d)
        assert need > last
        last = need
    over = dict(hkv=hkv, d=d, q_stride=6 * hkv * d, out_stride=6 * hkv * d)
    refused(lib, shared, "shared-prefix workspace holds 4096 bytes", code=2, ws_bytes=4096, **over)
    refused(lib, shared, "the batch needs %d" % size(4, 2, hkv, d), code=2, ws_bytes=size(4, 2, hkv, d) - 1, **over)


def test_op_table_checks_tensors(lib):
    o = ops_api.ops()
    lay = PageLayout(2, 128)
    regions = [bind_regions(torch.zeros(3 * lay.page_bytes, dtype=torch.int8), lay)[n]
               for n in ("k", "k_scale", "v", "v_scale", "v_zero")]
    table, rows = torch.zeros((2, 1), dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    k = torch.zeros((5, 2, 128), dtype=torch.float16)

    def load(table=table, starts=None, rows=rows, ppb=1, k=k, v=k):
        o.kv_load_paged(*regions, table, starts, rows, ppb, k, v)

    for text, over in (("k_out or v_out", dict(k=None, v=None)), ("block_table", dict(table=table.long())),
                       ("row_starts", dict(rows=rows[:2])), ("seq_starts", dict(starts=rows)),
                       ("pages_per_block", dict(ppb=0)), ("dtypes differ", dict(v=k.float())),
                       ("float16, bfloat16 or float32", dict(k=k.double(), v=None)),
                       (r"k/v_out \[N,2,128\]", dict(v=k[:4])), ("strides", dict(k=k.transpose(0, 1).contiguous()
                                                                              .transpose(0, 1))),
                       ("GPU tensors", dict())):
        with pytest.raises(RuntimeError, match=text):
            load(**over)
    load(k=k[:0], v=None)  # no rows: nothing to do

    good = dict(target=torch.zeros(2, 4, 9), draft=torch.zeros(2, 3, 9), tokens=torch.zeros(2, 3, dtype=torch.int32),
                counts=torch.zeros(2, dtype=torch.int32), u=torch.zeros(2, 3), s=torch.zeros(2),
                lens=torch.zeros(2, dtype=torch.int32), ws=torch.zeros(4096), out=torch.zeros(2, 4, dtype=torch.int64),
                acc=torch.zeros(2, dtype=torch.int32), nxt=torch.zeros(2, dtype=torch.int32))
    for text, over in (("target_probs", dict(target=torch.zeros(2, 9))), ("target_probs", dict(target=good["target"].double())),
                       ("draft_probs", dict(draft=torch.zeros(2, 4, 9))), ("dtypes", dict(draft=torch.zeros(2, 3, 9).half())),
                       ("draft_tokens", dict(tokens=torch.zeros(2, 3))), ("accept_uniform", dict(u=torch.zeros(2, 4))),
                       ("sample_uniform", dict(s=torch.zeros(3))), ("out_tokens", dict(out=torch.zeros(2, 4))),
                       ("num_drafts", dict(counts=torch.zeros(2))), ("accepted", dict(acc=None)),
                       ("next_lens needs", dict(lens=None)), ("GPU tensors", dict())):
        with pytest.raises(RuntimeError, match=text):
            o.verify_drafts(*{**good, **over}.values())

    q, lens = torch.zeros(4, 12, 128, dtype=torch.float16), torch.zeros(2, dtype=torch.int32)
    pre, table = torch.zeros(2, dtype=torch.int32), torch.zeros((2, 3), dtype=torch.int32)
    base = dict(q=q, pre=pre, n=100, table=table, lens=lens, ws=torch.zeros(64), out=q.clone(), q_len=2, ppb=1)

    def shared(**over):
        a = {**base, **over}
        o.int8k_int4v_attn_shared(a["q"], *regions, a["pre"], a["n"], a["table"], a["lens"], a["ws"], a["out"],
                                  a["q_len"], a["ppb"])

    for text, over in (("pages_per_block", dict(ppb=0)), ("negative prefix", dict(n=-1)), ("exceeds BM", dict(q_len=11)),
                       (r"q_fp16 \[T,HQ,D\]", dict(q=q[0])), ("float16 or bfloat16", dict(q=q.float())),
                       ("out shape", dict(out=q[:2])), ("float16, bfloat16 or float32", dict(out=q.double())),
                       ("B\\*q_len", dict(q_len=3)), ("block_table int32", dict(table=table.long())),
                       ("block_table int32", dict(table=table[:1])), ("seq_lens", dict(lens=lens[:1])),
                       ("prefix_table", dict(pre=pre.long())), ("prefix_table", dict(pre=table)),
                       ("GPU tensors", dict())):
        with pytest.raises(RuntimeError, match=text):
            shared(**over)

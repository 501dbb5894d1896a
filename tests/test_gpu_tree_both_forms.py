"""int8k_int4v_attn_tree in both of its forms on the same trees.

The forms round differently (one a probability times its V scale, the other the
dequantized V, each to 16 bits), so over a few hundred tokens their fp32 outputs
differ in some bits; the width of a table alone changes none.  So equal bits say that two
calls took the same form.  Tolerances are test_gpu_tree's.
"""
from __future__ import annotations

import pytest
import torch

from test_gpu_tree import Trees
from test_gpu_tree_forms import CONTEXTS, widened

pytestmark = pytest.mark.gpu


# Six tables of 17 pages in all take the one form, so many pages more the other.
@pytest.mark.parametrize("hkv,d,nodes,pages", [
    (4, 128, 4, 256), (4, 128, 13, 832), (4, 128, 43, 384), (4, 128, 50, 384), (4, 128, 64, 384),
    (2, 128, 8, 512), (2, 128, 16, 1024), (2, 128, 33, 384), (2, 128, 57, 384),
    (2, 256, 5, 320), (2, 256, 16, 1024), (2, 256, 22, 384), (2, 256, 43, 384), (2, 256, 64, 384),
    (4, 256, 8, 512), (4, 256, 16, 1024),
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_both_forms(gpu_ops, hkv, d, nodes, pages, dtype):
    st = Trees(gpu_ops, hkv, d, nodes, CONTEXTS, seed=nodes, dtype=dtype)
    want = st.want()
    a = st.run(torch.float32)
    b = widened(st, pages).run(torch.float32)
    assert not torch.equal(a, b), "one form in both"
    st.check(a, want)
    st.check(b, want)


@pytest.mark.parametrize("hkv,d,nodes,pages", [(4, 128, 13, 500), (4, 128, 40, 900), (4, 256, 26, 900), (2, 128, 20, 900)])
def test_a_wider_table_in_one_form(gpu_ops, hkv, d, nodes, pages):
    st = Trees(gpu_ops, hkv, d, nodes, CONTEXTS, seed=nodes)
    a = st.run(torch.float32)
    assert torch.equal(widened(st, pages).run(torch.float32), a)

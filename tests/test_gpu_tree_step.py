"""Steps of a small attention layer with drafted trees, all of the tree operators
together: rotated store, tree attention, the head's log probabilities, the accepted
branch, its rows kept; against the same layer over plain rows in 64 bits."""
from __future__ import annotations

import math
import random

import pytest
import torch

from gpu_cases import Cache, DEV
from k8v4_v030.layout import GQA, PAGE, PageLayout
from k8v4_v030.plan import tree_depths, tree_masks

pytestmark = pytest.mark.gpu

HKV, D, VOCAB, NODES, BATCH = 4, 128, 500, 13, 3


def test_steps(gpu_ops):
    """Ten steps: what the operators leave in the cache is a linear sequence of the
    accepted tokens, bit for bit what storing them one after the other gives."""
    ops, rng = gpu_ops, random.Random(0)
    gen = torch.Generator().manual_seed(0)
    embed = torch.randn((VOCAB, (GQA + 2) * HKV * D), generator=gen).half().to(DEV)
    head = (torch.randn((GQA * HKV * D, VOCAB), generator=gen) * 0.02).to(DEV)
    angle = torch.arange(2000, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(64, dtype=torch.float64) / 64)
    cos_sin = torch.cat((angle.cos(), angle.sin()), 1).float().to(DEV)
    pages = 30
    cache, plain = Cache(pages * BATCH, PageLayout(HKV, D)), Cache(pages * BATCH, PageLayout(HKV, D))
    table = torch.randperm(pages * BATCH, generator=gen).to(torch.int32).view(BATCH, pages).to(DEV)

    def slots(b, positions):
        p = torch.tensor(positions, device=DEV)
        return table[b, p // PAGE].long() * PAGE + p % PAGE

    def rows_of(tokens):
        x = embed[torch.tensor(tokens, device=DEV)].unflatten(1, ((GQA + 2) * HKV, D))
        return x.split([GQA * HKV, HKV, HKV], 1)

    history = [[rng.randrange(VOCAB) for _ in range(n)] for n in (40, 117, 63)]  # all but the last are cached
    for b, h in enumerate(history):
        _q, k, v = rows_of(h[:-1])
        pos = torch.arange(len(h) - 1, device=DEV)
        ops.rope_kv_store_paged(None, k, v, pos, cos_sin, True, slots(b, list(range(len(h) - 1))), *cache.region_args(), None)
    ws = torch.empty(ops.attn_tree_workspace_bytes(BATCH, NODES, HKV, D), dtype=torch.uint8, device=DEV)
    lens = torch.tensor([len(h) - 1 + NODES for h in history], dtype=torch.int32, device=DEV)
    n = BATCH * NODES
    f = lambda *shape, dt=torch.float32: torch.empty(shape, dtype=dt, device=DEV)  # noqa: E731
    q_out, out = f(n, GQA * HKV, D, dt=torch.float16), f(n, GQA * HKV, D, dt=torch.float16)
    top_ids, top_lps = f(n, 1, dt=torch.int64), f(n, 1)
    path, chosen = f(BATCH, NODES, dt=torch.int32), f(BATCH, NODES, dt=torch.int64)
    accepted = f(BATCH, dt=torch.int32)
    taken = 0
    for step in range(10):
        parents = [[-1] + [rng.randrange(max(0, i - 4), i) for i in range(1, NODES)] for _ in history]
        drafts = [[h[-1]] + [rng.randrange(VOCAB) for _ in range(NODES - 1)] for h in history]
        # Drafts as a good draft model makes them: one child of the root and one of its
        # children hold what the last step's logits favoured.
        if step:
            for b in range(BATCH):
                for i in range(1, NODES):
                    if rng.random() < 0.5:
                        drafts[b][i] = guesses[b]
        base = [len(h) - 1 for h in history]
        positions = torch.tensor([c + d for c, p in zip(base, parents) for d in tree_depths(p)], device=DEV)
        masks = torch.tensor([tree_masks(p) for p in parents], device=DEV)
        places = torch.cat([slots(b, list(range(c, c + NODES))) for b, c in enumerate(base)])
        q, k, v = rows_of([t for d in drafts for t in d])
        ops.rope_kv_store_paged(q, k, v, positions, cos_sin, True, places, *cache.region_args(), q_out)
        ops.int8k_int4v_attn_tree(q_out, *cache.region_args(), table, lens, masks, ws, out, NODES, 1)
        logits = out.float().flatten(1) @ head
        lws = torch.empty(max(16, ops.token_logprobs_workspace_bytes(n, VOCAB, 1)), dtype=torch.uint8, device=DEV)
        ops.token_logprobs(logits, None, lws, None, None, None, top_ids, top_lps)
        targets = top_ids.view(BATCH, NODES)
        assert torch.equal(targets.flatten(), logits.argmax(1))
        starts = lens - NODES
        d = torch.tensor(drafts, dtype=torch.int32, device=DEV)
        if step % 2:  # make a branch certain to be accepted
            for b in range(BATCH):
                child = [i for i in range(1, NODES) if parents[b][i] == 0][-1]
                d[b, child] = targets[b, 0].to(torch.int32)
        # A draft changed behind its store is stored again, as the tree the target saw.
        drafts = d.tolist()
        _q, k, v = rows_of([t for x in drafts for t in x])
        ops.rope_kv_store_paged(None, k, v, positions, cos_sin, True, places, *cache.region_args(), None)
        ops.accept_tree(d, torch.tensor(parents, dtype=torch.int32, device=DEV), targets.contiguous(), lens, path, chosen,
                        accepted, lens)
        ops.kv_keep_paged(*cache.region_args(), table, starts, path, accepted, 1)
        guesses = []
        for b, h in enumerate(history):
            a = int(accepted[b])
            tokens = [drafts[b][i] for i in path[b, 1 : a + 1].tolist()]
            assert tokens == chosen[b, :a].tolist()
            h += chosen[b, : a + 1].tolist()
            guesses.append(h[-1])
            taken += a
            assert int(lens[b]) == len(h) - 1 + NODES
    assert taken > 5
    # The cache against one that stored the tokens one after the other.
    for b, h in enumerate(history):
        _q, k, v = rows_of(h[:-1])
        pos = torch.arange(len(h) - 1, device=DEV)
        where = slots(b, list(range(len(h) - 1)))
        ops.rope_kv_store_paged(None, k, v, pos, cos_sin, True, where, *plain.region_args(), None)
        page, row = where // PAGE, where % PAGE
        for x, y in zip(cache.region_args(), plain.region_args()):
            assert torch.equal(x[page, row], y[page, row])
    assert math.isfinite(float(out.float().abs().max()))

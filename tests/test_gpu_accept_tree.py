"""accept_tree against a walk in Python."""
from __future__ import annotations

import random

import pytest
import torch

from gpu_cases import DEV

pytestmark = pytest.mark.gpu


def walk(drafts, parents, targets, width, nodes):
    if nodes <= 0:
        return [], []
    path = [0]
    while len(path) < width:
        at = path[-1]
        nxt = [i for i in range(at + 1, nodes) if parents[i] == at and drafts[i] == targets[at] and targets[at] >= 0]
        if not nxt:
            break
        path.append(nxt[0])
    return path, [targets[i] for i in path]


class Trees:
    def __init__(self, batch, nodes, width, seed, tokens=3, int64=False, shared=False, counts=None):
        rng = random.Random(seed)
        tree = lambda: [-1] + [rng.randrange(max(0, i - 6), i) for i in range(1, nodes)]  # noqa: E731
        one = tree()
        self.parents = [one if shared else tree() for _ in range(batch)]
        self.drafts = [[rng.randrange(tokens) for _ in range(nodes)] for _ in range(batch)]
        self.targets = [[rng.randrange(-1 if tokens > 2 else 0, tokens) for _ in range(nodes)] for _ in range(batch)]
        self.counts, self.width, self.nodes = counts, width, nodes
        dt = torch.int64 if int64 else torch.int32
        self.d = torch.tensor(self.drafts, dtype=dt, device=DEV)
        p = torch.tensor(self.parents, dtype=torch.int32, device=DEV)
        self.p = p[:1].expand(batch, nodes) if shared else p
        self.t = torch.tensor(self.targets, device=DEV)
        self.lens = torch.tensor([rng.randrange(1, 9999) for _ in range(batch)], dtype=torch.int32, device=DEV)
        self.n = None if counts is None else torch.tensor(counts, dtype=torch.int32, device=DEV)
        self.path = torch.full((batch, width + 2), 99, dtype=torch.int32, device=DEV)
        self.out = torch.full((batch, width + 3), 99, dtype=torch.int64, device=DEV)
        self.acc = torch.full((batch,), 99, dtype=torch.int32, device=DEV)
        self.nxt = torch.full((batch,), 99, dtype=torch.int32, device=DEV)

    def bind(self, ops, lens="lens", nxt="nxt"):
        pick = lambda x: getattr(self, x) if isinstance(x, str) else x  # noqa: E731
        return ops.bind_accept_tree(self.d, self.p, self.t, pick(lens), self.path[:, 1 : self.width + 1],
                                    self.out[:, : self.width], self.acc, pick(nxt), self.n)

    def check(self, lens=None):
        torch.cuda.synchronize()
        lens = self.lens.tolist() if lens is None else lens
        for b, (path, out) in enumerate(zip(self.path.tolist(), self.out.tolist())):
            n = self.nodes if self.counts is None else min(max(self.counts[b], 0), self.nodes)
            want, tokens = walk(self.drafts[b], self.parents[b], self.targets[b], self.width, n)
            pad = [-1] * (self.width - len(want))
            assert path == [99] + want + pad + [99] and out == tokens + pad + [99] * 3
            assert int(self.acc[b]) == len(want) - 1
            if lens:
                assert int(self.nxt[b]) == lens[b] + len(want)


@pytest.mark.parametrize("batch,nodes,width", [(1, 1, 1), (1, 13, 13), (7, 64, 64), (300, 21, 6), (64, 64, 3), (5, 2, 2), (4, 63, 1)])
@pytest.mark.parametrize("int64,shared", [(False, False), (True, True)])
def test_walks(gpu_ops, batch, nodes, width, int64, shared):
    st = Trees(batch, nodes, width, seed=batch + nodes, int64=int64, shared=shared)
    st.bind(gpu_ops)()
    st.check()


def test_a_chain_to_its_end(gpu_ops):
    st = Trees(3, 64, 64, seed=1)
    for b in range(3):
        st.parents[b] = list(range(-1, 63))
        st.drafts[b] = [7] * 64
        st.targets[b] = [7 if i < 60 + 2 * b else 8 for i in range(64)]
    st.p.copy_(torch.tensor(st.parents, dtype=torch.int32))
    st.d.copy_(torch.tensor(st.drafts))
    st.t.copy_(torch.tensor(st.targets))
    st.bind(gpu_ops)()
    st.check()
    assert st.acc.tolist() == [60, 62, 63]


def test_node_counts_lengths_in_place_and_odd_parents(gpu_ops):
    st = Trees(6, 20, 8, seed=2, tokens=2, counts=[0, 1, 20, 7, -5, 1000])
    for b in range(6):  # parents that are none, or lie behind the node: not part of the tree
        st.parents[b][3], st.parents[b][5], st.parents[b][6] = 3, 9, -7
    st.p.copy_(torch.tensor(st.parents, dtype=torch.int32))
    before = st.lens.tolist()
    st.bind(gpu_ops, nxt="lens")()
    st.nxt = st.lens
    st.check(before)
    st.bind(gpu_ops, lens=None, nxt=None)()
    st.nxt = None
    st.check([])


def test_equal_drafts_take_the_lowest_child(gpu_ops):
    st = Trees(1, 6, 6, seed=3)
    st.parents[0], st.drafts[0], st.targets[0] = [-1, 0, 0, 0, 2, 1], [0, 5, 5, 5, 4, 4], [5, 4, 4, 4, 1, 2]
    for x, y in ((st.p, st.parents), (st.d, st.drafts), (st.t, st.targets)):
        x.copy_(torch.tensor(y))
    st.bind(gpu_ops)()
    st.check()
    assert st.path[0, 1:7].tolist() == [0, 1, 5, -1, -1, -1] and st.out[0, :6].tolist() == [5, 4, 2, -1, -1, -1]


def test_replayed_with_other_tokens(gpu_ops):
    st = Trees(9, 30, 7, seed=4)
    call = st.bind(gpu_ops)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for seed in range(3):
        new = Trees(9, 30, 7, seed=50 + seed)
        st.drafts, st.parents, st.targets = new.drafts, new.parents, new.targets
        for x, y in ((st.d, new.d), (st.p, new.p), (st.t, new.t), (st.lens, new.lens)):
            x.copy_(y)
        torch.cuda.synchronize()
        graph.replay()
        st.check()


def test_empty_batch(gpu_ops):
    st = Trees(2, 5, 3, seed=5)
    for name in ("d", "p", "t", "lens", "path", "out", "acc", "nxt"):
        setattr(st, name, getattr(st, name)[:0])
    assert st.bind(gpu_ops) is None

"""Host helpers of drafted trees."""
from __future__ import annotations

import pytest

from k8v4_v030.plan import tree_depths, tree_masks


def test_depths_and_masks():
    parents = [-1, 0, 0, 1, 3, 2]
    assert tree_depths(parents) == [0, 1, 1, 2, 3, 2]
    assert tree_masks(parents) == [0b1, 0b11, 0b101, 0b1011, 0b11011, 0b100101]


def test_a_chain_of_64_is_signed():
    words = tree_masks(list(range(-1, 63)))
    assert words[62] == 2**63 - 1 and words[63] == -1
    assert tree_masks([]) == [] and tree_depths([]) == []


def test_refusals():
    with pytest.raises(ValueError, match="parent comes before"):
        tree_masks([-1, 1])
    with pytest.raises(ValueError, match="parent comes before"):
        tree_depths([-1, -1])
    with pytest.raises(ValueError, match="at most 64"):
        tree_masks(list(range(-1, 64)))

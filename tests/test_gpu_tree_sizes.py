"""Masks of trees whose declared size is too small."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("declared", [0, 1, 2])
def test_trees_larger_than_declared_are_reported(declared) -> None:
    """A batch said to hold no nodes too: its mask rows and depths were never written."""
    from microserve_b200 import _lib
    from microserve_b200.tree import tree_masks

    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
    masks, depths = tree_masks(i32([-1, 0, 0]), i32([0, 3]), declared)
    assert masks.shape == (3, 1) and depths.shape == (3,)
    assert _lib.device_error() == 9
    # rows behind the last sequence are no nodes
    tree_masks(i32([-1, 0, 0]), i32([0, 0, 0]), 0)
    assert _lib.device_error() == 0

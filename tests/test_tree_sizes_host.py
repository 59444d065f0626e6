"""Sizes of mask rows that the kernels' indices cannot hold are refused before any launch."""

from __future__ import annotations


def test_mask_rows_beyond_the_indices_are_refused() -> None:
    from microserve_b200 import _lib

    lib = _lib.load()
    masks = lambda nodes, words: lib.ms_tree_masks(16, 16, 1, nodes, nodes, 16, words, None, None)  # noqa: E731
    assert masks(1024, 1 << 21) == _lib.MS_ERR_INVALID
    assert masks(33, 1) == _lib.MS_ERR_INVALID
    assert "words" in lib.ms_last_error().decode()

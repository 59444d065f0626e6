"""Whole rounds whose accepted paths are longer than one call moves."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .test_gpu_tree import _cache, _model, _ordinary, _prefill

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("wrong", [0, 1, 7])
def test_a_round_of_paths_beyond_one_move(wrong) -> None:
    """Trees 299 and 600 deep, `wrong` nodes that are not accepted between any two of a path: the
    streams are those of ordinary passes, in that call and in the next ones, which read what was moved."""
    from microserve_b200.tree import verify_trees

    model = _model(max_seq_len=2048)
    prompts = [[5, 9, 2], [7, 1]]
    depth = [299, 600 if wrong == 0 else 900 // (wrong + 1)]
    want = _ordinary(model, prompts, 640)
    cache = _cache(model, blocks=700)
    _prefill(model, cache, prompts)
    rng = np.random.default_rng(wrong)
    trees = []
    for i, p in enumerate(prompts):
        tokens, parents, at = [p[-1]], [-1], 0
        for t in want[i][: depth[i]]:
            # (behind the first deep path's middle the right nodes follow one another, so that nodes are still moved)
            for _ in range(wrong if len(tokens) < 500 else 0):
                tokens.append((t + 1 + int(rng.integers(0, 59))) % 61)
                parents.append(at)
            tokens.append(t)
            parents.append(at)
            at = len(tokens) - 1
        trees.append((tokens, parents))
    assert max(len(t) for t, _ in trees) <= 1024
    got = verify_trees(model, cache, [0, 1], trees)
    for g, w, d in zip(got, want, depth):
        assert g == w[: d + 1]
    for _ in range(3):
        more = verify_trees(model, cache, [0, 1], [([g[-1]], [-1]) for g in got])
        for g, m in zip(got, more):
            g += m
    for g, w in zip(got, want):
        assert g == w[: len(g)]
    cache.allocator.check_invariants()


def test_a_round_of_a_deep_tree_of_which_little_is_accepted() -> None:
    from microserve_b200.tree import verify_trees

    model = _model(max_seq_len=2048)
    prompts = [[5, 9, 2], [7, 1]]
    want = _ordinary(model, prompts, 8)
    cache = _cache(model, blocks=700)
    _prefill(model, cache, prompts)
    off = [(t + 1) % 61 for t in want[0]]
    trees = [([2, want[0][0], *[off[1]] * 400], [-1, *range(401)]), ([1, want[1][0]], [-1, 0])]
    got = verify_trees(model, cache, [0, 1], trees)
    assert got[0][:2] == want[0][:2] and got[1] == want[1][:2]
    torch.cuda.synchronize()
    assert cache.num_tokens(1) == 1 + 2

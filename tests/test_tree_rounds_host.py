"""Rounds of trees that fail on the host leave the cache as it was."""

from __future__ import annotations

from types import SimpleNamespace

import pytest


def test_a_round_that_runs_out_of_blocks_makes_no_sequence() -> None:
    from microserve_b200.cache import OutOfCacheMemory, PagedKVCache
    from microserve_b200.config import CacheConfig, ModelConfig
    from microserve_b200.tree import verify_trees

    cfg = ModelConfig(max_seq_len=256)
    cache = PagedKVCache(cfg, CacheConfig(8, 4), device="cpu")
    cache.append(0, 5)
    chain = ([1] * 30, [-1, *range(29)])
    with pytest.raises(OutOfCacheMemory):
        verify_trees(SimpleNamespace(cfg=cfg), cache, [0, 7], [chain, chain])
    assert list(cache.tables) == [0] and cache.num_tokens(0) == 5 and cache.num_free_blocks == 3
    cache.allocator.check_invariants()


def test_a_round_that_fails_after_its_blocks_were_taken_makes_no_sequence() -> None:
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, ModelConfig
    from microserve_b200.tree import verify_trees

    cfg = ModelConfig(max_seq_len=256)
    cache = PagedKVCache(cfg, CacheConfig(8, 24), device="cpu")  # (no device: the round cannot go on)
    cache.append(0, 5)
    with pytest.raises(RuntimeError):
        verify_trees(SimpleNamespace(cfg=cfg), cache, [0, 7], [([1, 2], [-1, 0])] * 2)
    assert list(cache.tables) == [0] and cache.num_tokens(0) == 5 and cache.num_free_blocks == 23
    cache.allocator.check_invariants()

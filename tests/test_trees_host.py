"""Host side of the score forms, trees and cache moves (no GPU): packed structures, the pool's
bookkeeping, what is refused before any launch."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest


def _cache(blocks: int = 24, bs: int = 8):
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, ModelConfig

    return PagedKVCache(ModelConfig(max_seq_len=256), CacheConfig(bs, blocks), device="cpu")


def test_packed_structures_equal_the_ctypes_ones() -> None:
    from microserve_b200 import _lib, attention, cache

    assert ctypes.sizeof(_lib.MsAttentionForm) == 4 * 4 + 3 * 8
    got = attention._PACK_FORM(0.5, 30.0, 7, 2, 11, 12, 13)
    assert got == bytes(_lib.MsAttentionForm(0.5, 30.0, 7, 2, 11, 12, 13))
    vals = tuple(range(1, 13))
    assert attention._PACK_BATCH(*vals) == bytes(_lib.MsBatch(*vals))
    two = (ctypes.c_void_p * 2)(5, 6)
    at = ctypes.addressof(two)
    p = lambda a: ctypes.cast(a, ctypes.POINTER(ctypes.c_void_p))  # noqa: E731
    assert attention._PACK_CACHE(1, 2, 3, 4, 5, 1, at, at + 8) == bytes(_lib.MsKVCache(1, 2, 3, 4, 5, 1, p(at), p(at + 8)))
    assert cache._PACK_CACHE(1, 2, 3, 4, 5, 1, at, at + 8) == attention._PACK_CACHE(1, 2, 3, 4, 5, 1, at, at + 8)


def test_limits_equal_the_header() -> None:
    import re

    from microserve_b200 import cache, tree

    from .conftest import ROOT

    text = (ROOT / "include" / "microserve_b200.h").read_text()
    value = lambda name: int(re.search(rf"#define {name} (\d+)", text).group(1))  # noqa: E731
    assert cache.MAX_MOVES == value("MS_KV_MOVE_MAX") and tree.MAX_NODES == value("MS_TREE_MAX")


def test_c_entry_points_refuse_before_launching() -> None:
    from microserve_b200 import _lib

    lib = _lib.load()
    bad, unsupported, large = _lib.MS_ERR_INVALID, _lib.MS_ERR_UNSUPPORTED, _lib.MS_ERR_TOO_LARGE
    keep = []

    def cache(dh=64, dtype=1, hkv=2, bs=16, blocks=10, k=1 << 20, v=1 << 21):
        two = (ctypes.c_void_p * 2)(k, v)
        at = ctypes.addressof(two)
        keep.append(two)
        p = lambda a: ctypes.cast(a, ctypes.POINTER(ctypes.c_void_p))  # noqa: E731
        return ctypes.byref(_lib.MsKVCache(1, blocks, bs, hkv, dh, dtype, p(at), p(at + 8)))

    def batch(T=3, B=1, width=2, q=3, ids=1, pos=1, starts=1, lens=1, tables=1):
        return ctypes.byref(_lib.MsBatch(T, B, width, q, 0, 0, ids, pos, 1, starts, lens, tables))

    def attend(c=None, b=None, heads=4, form=None, stride=256, out_stride=256, q=1 << 12, out=1 << 13, ws=None, n=0,
               layer=0):
        return lib.ms_paged_attention_form(q, stride, c or cache(), layer, b or batch(), heads, form, out, out_stride,
                                           ws, n, None)

    def form(**kw):
        return ctypes.byref(_lib.MsAttentionForm(**kw))

    assert attend(layer=1) == bad and attend(heads=3) == bad and attend(heads=0) == bad
    assert attend(q=None) == bad and attend(out=None) == bad
    assert attend(stride=255) == bad and attend(out_stride=255) == bad
    assert attend(ws=None, n=16) == bad and attend(ws=8, n=16) == bad
    assert attend(b=batch(T=-1)) == bad and attend(b=batch(q=0)) == bad and attend(b=batch(width=0)) == bad
    for missing in ("pos", "starts", "lens", "tables"):
        assert attend(b=batch(**{missing: None})) == bad
    assert attend(c=cache(dh=48)) == unsupported and attend(c=cache(dtype=7)) == unsupported
    assert attend(b=batch(B=70000)) == large
    assert attend(b=batch(q=1 << 24)) == large
    assert attend(form=form(softcap=-1.0)) == bad and attend(form=form(softcap=float("inf"))) == bad
    assert attend(form=form(scale=float("nan"))) == bad and attend(form=form(scale=-0.5)) == bad
    assert attend(form=form(window=-1)) == bad and attend(form=form(tree_mask=1, mask_words=0)) == bad
    assert attend(b=batch(T=0, B=0, q=0, width=0), q=None, out=None) == 0  # nothing to do
    assert lib.ms_attention_form_workspace_size(None, 4, batch(), None) == 0
    assert lib.ms_attention_form_workspace_size(cache(), 4, None, None) == 0
    assert lib.ms_attention_form_workspace_size(cache(), 3, batch(), None) == 0

    copy, move = lib.ms_kv_copy_blocks, lib.ms_kv_move_tokens
    assert copy(None, 1, 1, 1, None) == bad and copy(cache(), None, 1, 1, None) == bad
    assert copy(cache(), 1, 1, -1, None) == bad and copy(cache(k=(1 << 20) + 2), 1, 1, 1, None) == bad
    assert copy(cache(v=None), 1, 1, 1, None) == bad and copy(cache(), None, None, 0, None) == 0
    assert move(cache(), None, 1, 1, 1, None) == bad and move(cache(), 1, 1, -1, 1, None) == bad
    assert move(cache(), 1, 1, 1, 257, None) == large and move(cache(), None, None, 0, 4, None) == 0
    assert move(cache(dh=512, dtype=0), 1, 1, 1, 256, None) == large

    masks = lib.ms_tree_masks
    assert masks(None, 1, 1, 1, 1, 1, 1, None, None) == bad and masks(1, 1, -1, 1, 1, 1, 1, None, None) == bad
    assert masks(1, 1, 1, 40, 40, 1, 1, None, None) == bad and masks(1, 1, 1, 2000, 1025, 1, 64, None, None) == large
    assert masks(None, None, 0, 0, 0, None, 0, None, None) == 0

    def accept(logits=1 << 12, stride=8, vocab=8, target=None, b=None, parents=1, most=2, bs=16, blocks=9, out=1, num=1,
               nodes=1, src=1, dst=1):
        return lib.ms_tree_accept(logits, stride, vocab, target, b or batch(), parents, most, bs, blocks, out, num,
                                  nodes, src, dst, None)

    assert accept(logits=None) == bad and accept(target=1) == bad
    assert accept(stride=7) == bad and accept(vocab=0) == bad and accept(most=-1) == bad
    assert accept(src=None) == bad and accept(bs=0) == bad and accept(blocks=0) == bad
    assert accept(parents=None) == bad and accept(out=None) == bad and accept(nodes=None) == bad
    assert accept(b=batch(ids=None)) == bad and accept(b=batch(q=1025)) == large
    assert accept(b=batch(T=0, B=0)) == 0


def test_fork_many_gives_every_child_its_own_last_block() -> None:
    from microserve_b200.cache import OutOfCacheMemory

    c = _cache()
    c.append(0, 19)
    c.reserve_many([0], [40])  # capacity is not shared
    c.fork_many(0, [1, 2])
    assert c.tables[1].blocks[:2] == c.tables[2].blocks[:2] == c.tables[0].blocks[:2]
    assert len({c.tables[s].blocks[2] for s in (0, 1, 2)}) == 3
    assert [len(c.tables[s].blocks) for s in (0, 1, 2)] == [5, 3, 3]
    c.append_many([0, 1, 2], [7, 5, 6])
    c.allocator.check_invariants()
    free = c.num_free_blocks
    with pytest.raises(OutOfCacheMemory):
        c.fork_many(0, list(range(10, 40)))
    assert c.num_free_blocks == free and 10 not in c.tables
    with pytest.raises(KeyError):
        c.fork_many(99, [50])
    c.fork_many(0, [])
    for s in (0, 1, 2):
        c.free(s)
    assert c.num_free_blocks == 24


def test_unshare_many_leaves_one_holder_and_is_all_or_nothing() -> None:
    from microserve_b200.cache import OutOfCacheMemory

    c = _cache(blocks=6)
    c.append(0, 12)
    for s in (1, 2, 3):
        c.fork(0, s)
    held = [c.tables[s].blocks for s in range(4)]
    c.append(9, 8 * 2)  # two blocks are left: three sequences need one each
    with pytest.raises(OutOfCacheMemory):
        c.unshare_many([0, 1, 2, 3])
    assert [c.tables[s].blocks for s in range(4)] == held
    c.allocator.check_invariants()
    c.free(9)
    c.unshare_many([0, 1, 2, 2, 3])  # a sequence named twice counts once
    lasts = [c.tables[s].blocks[-1] for s in range(4)]
    assert len(set(lasts)) == 4 and held[0][-1] in lasts
    c.unshare_many([0, 1, 2, 3])
    assert [c.tables[s].blocks[-1] for s in range(4)] == lasts
    c.allocator.check_invariants()


def test_compact_renames_blocks_and_keeps_references() -> None:
    c = _cache(blocks=30)
    rng = np.random.default_rng(0)
    for s in range(6):
        c.append(s, int(rng.integers(1, 25)))
    c.fork(1, 10)
    c.free(0)
    c.free(4)
    tokens = {s: c.num_tokens(s) for s in (1, 2, 3, 5, 10)}
    counts = {s: len(c.tables[s].blocks) for s in tokens}
    used = c.allocator.num_used
    moved = c.compact()
    assert moved > 0 and c.moves == 1
    assert c.allocator.num_used == used
    assert {s: c.num_tokens(s) for s in tokens} == tokens
    assert {s: len(c.tables[s].blocks) for s in tokens} == counts
    assert c.tables[1].blocks == c.tables[10].blocks
    every = [b for s in (1, 2, 3, 5) for b in c.tables[s].blocks]
    assert sorted(every) == list(range(used))
    assert all(c.allocator.refcount(b) == (2 if b in c.tables[1].blocks else 1) for b in every)
    c.allocator.check_invariants()
    assert c.compact() == 0 and c.moves == 1
    c.append(50, 1)
    assert c.tables[50].blocks == [used]
    c.reset()
    c.allocator.check_invariants()
    assert _cache().compact() == 0


def test_trees_are_checked() -> None:
    from microserve_b200.tree import MAX_NODES, _check_tree

    _check_tree([1], [-1], 5)
    _check_tree([1, 2, 2, 0], [-1, 0, 0, 2], 5)
    for tokens, parents in (([], []), ([1, 2], [-1]), ([1, 2], [-1, 1]), ([1, 2], [-1, -1]), ([1, 2], [0, 0]),
                            ([1, 5], [-1, 0]), ([-1], [-1]), ([1] * (MAX_NODES + 1), [-1, *range(MAX_NODES)])):
        with pytest.raises(ValueError):
            _check_tree(tokens, parents, 5)


def test_a_cache_without_a_device_moves_no_tensors() -> None:
    from microserve_b200.cache import copy_blocks, move_tokens
    import torch

    pool = torch.zeros((2, 1, 4, 1, 8, 8))
    i = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        copy_blocks(pool, i, i)
    with pytest.raises(RuntimeError):
        move_tokens(pool, i.view(1, 1), i.view(1, 1))


def test_unsharing_counts_as_a_change_of_blocks() -> None:
    """A planned round holds its tables on the device: it is dropped when a block of them is replaced."""
    c = _cache()
    c.append(0, 5)
    c.fork(0, 1)
    c.unshare_many([1])
    assert c.moves == 1
    c.unshare_many([0, 1])  # nothing is shared any more
    assert c.moves == 1

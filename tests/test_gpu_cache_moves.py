"""Copies of pages and moves of tokens inside the pools: bit for bit against indexing."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"
SHAPES = [  # dtype, layers, blocks, heads, block size, d_head
    (torch.bfloat16, 2, 40, 4, 16, 64), (torch.bfloat16, 3, 50, 8, 16, 128), (torch.float32, 4, 30, 4, 16, 32),
    (torch.bfloat16, 1, 33, 1, 1, 2), (torch.float32, 5, 37, 3, 5, 6), (torch.bfloat16, 130, 9, 2, 8, 8),
    (torch.float32, 1, 20, 2, 64, 128), (torch.bfloat16, 2, 64, 1, 7, 10),
]


def _pool(shape, seed: int) -> torch.Tensor:
    dtype, layers, blocks, heads, bs, dh = shape
    bits = torch.int16 if dtype is torch.bfloat16 else torch.int32
    g = torch.Generator(device=DEV).manual_seed(seed)
    # any bits at all, NaN among them
    return torch.randint(-2 ** 15, 2 ** 15, (2, layers, blocks, heads, bs, dh), generator=g, device=DEV,
                         dtype=torch.int64).to(bits).view(dtype)


def _bits(t: torch.Tensor) -> torch.Tensor:
    return t.view(torch.int16 if t.dtype is torch.bfloat16 else torch.int32)


def _i32(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("n", [0, 1, 3, 99])
def test_copy_blocks(shape, n) -> None:
    from microserve_b200 import _lib
    from microserve_b200.cache import copy_blocks

    rng = np.random.default_rng(n)
    pool = _pool(shape, n)
    blocks = shape[2]
    order = rng.permutation(blocks)
    dst = order[: min(n, blocks // 2)]
    src = rng.choice(order[len(dst) :], len(dst))  # sources repeat
    want = _bits(pool).clone()
    want[:, :, dst] = want[:, :, src]
    copy_blocks(pool, _i32(src), _i32(dst))
    assert torch.equal(_bits(pool), want)
    assert _lib.device_error() == 0


@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("groups,per", [(1, 1), (7, 3), (5, 9), (2, 40), (1, 256), (3, 0)])
def test_move_tokens(shape, groups, per) -> None:
    """Chains, swaps and skipped pairs inside each group."""
    from microserve_b200 import _lib
    from microserve_b200.cache import move_tokens

    blocks, bs = shape[2], shape[4]
    slots = blocks * bs
    share = slots // groups
    if share < 2:
        pytest.skip("no slots for so many groups")
    rng = np.random.default_rng(groups * 1000 + per)
    src, dst = np.full((groups, per), -1), np.full((groups, per), -1)
    own = rng.permutation(slots)
    for g in range(groups):
        mine = own[g * share : (g + 1) * share]
        n = min(per, share)
        src[g, :n] = rng.choice(mine, n)  # any, also destinations
        dst[g, :n] = rng.permutation(mine)[:n]
        hide = rng.random(per) < 0.2
        src[g, hide] = -1 - rng.integers(0, 5)
        dst[g, rng.random(per) < 0.1] = -1
    pool = _pool(shape, per)
    before = _bits(pool).clone()
    want = before.clone()
    for s, d in zip(src.ravel(), dst.ravel()):
        if s >= 0 and d >= 0:
            want[:, :, d // bs, :, d % bs] = before[:, :, s // bs, :, s % bs]
    move_tokens(pool, _i32(src), _i32(dst))
    assert torch.equal(_bits(pool), want)
    assert _lib.device_error() == 0


def test_bad_places_are_skipped_and_reported() -> None:
    from microserve_b200 import _lib
    from microserve_b200.cache import copy_blocks, move_tokens

    shape = SHAPES[0]
    for src, dst in (([0, 40], [2, 3]), ([0, -1], [2, 3]), ([0, 1], [2, 1 << 30])):
        pool = _pool(shape, 1)
        want = _bits(pool).clone()
        want[:, :, 2] = want[:, :, 0]
        copy_blocks(pool, _i32(src), _i32(dst))
        assert torch.equal(_bits(pool), want)
        assert _lib.device_error() == 2
    for src, dst in (([[0, 640]], [[2, 3]]), ([[0, 1]], [[2, 1 << 30]])):
        pool = _pool(shape, 2)
        want = _bits(pool).clone()
        want[:, :, 0, :, 2] = want[:, :, 0, :, 0]
        move_tokens(pool, _i32(src), _i32(dst))
        assert torch.equal(_bits(pool), want)
        assert _lib.device_error() == 1


def test_refusals() -> None:
    from microserve_b200.cache import copy_blocks, move_tokens

    pool = _pool(SHAPES[0], 0)
    a, b = _i32([0, 1]), _i32([2, 3])
    for args in ((pool[0], a, b), (pool.half(), a, b), (pool[:, :, ::2], a, b), (pool, a.long(), b), (pool, a, b[:1]),
                 (pool, a.cpu(), b)):
        with pytest.raises(ValueError):
            copy_blocks(*args)
    a, b = a.view(1, 2), b.view(1, 2)
    for args in ((pool, a[0], b[0]), (pool, a, b.view(2, 1)), (pool, a.float(), b),
                 (pool, torch.zeros((1, 257), dtype=torch.int32, device=DEV),
                  torch.zeros((1, 257), dtype=torch.int32, device=DEV))):
        with pytest.raises(ValueError):
            move_tokens(*args)


def _cache(blocks: int = 24, dtype: str = "bfloat16"):
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, ModelConfig

    cfg = ModelConfig(vocab_size=16, n_layers=3, d_model=128, n_heads=4, n_kv_heads=2, max_seq_len=256, dtype=dtype)
    cache = PagedKVCache(cfg, CacheConfig(8, blocks, dtype), DEV)
    cache.pool.copy_(torch.randn(cache.pool.shape, device=DEV))
    return cache


def _content(cache, s: int) -> torch.Tensor:
    n, bs = cache.num_tokens(s), cache.block_size
    pages = torch.tensor(cache.tables[s].blocks[: -(-n // bs)], dtype=torch.long, device=DEV)
    t = cache.pool[:, :, pages].permute(0, 1, 3, 2, 4, 5)
    return t.reshape(*t.shape[:3], -1, t.shape[-1])[..., :n, :].clone()


@pytest.mark.parametrize("n", [1, 8, 13, 16])
def test_fork_many_and_unshare_many(n) -> None:
    from microserve_b200.cache import OutOfCacheMemory

    cache = _cache()
    cache.append(0, n)
    was = _content(cache, 0)
    cache.fork_many(0, [1, 2, 3])
    for s in range(4):
        assert cache.num_tokens(s) == n and torch.equal(_content(cache, s), was)
    tails = {cache.tables[s].blocks[-1] for s in range(4)}
    assert len(tails) == (4 if n % 8 else 1)
    cache.allocator.check_invariants()
    # plain forks share everything until they are given their own
    for s in (4, 5):
        cache.fork(0, s)
    cache.unshare_many([4, 0, 5])
    # block 0's holders: one of the three may keep it (unless a full block is shared with 1, 2, 3)
    lasts = [cache.tables[s].blocks[-1] for s in (0, 4, 5)]
    assert len(set(lasts)) == 3
    for s in (0, 4, 5):
        assert torch.equal(_content(cache, s), was)
    cache.allocator.check_invariants()
    with pytest.raises(ValueError):
        cache.fork_many(0, [9, 9])
    with pytest.raises(ValueError):
        cache.fork_many(0, [9, 1])
    if n % 8:
        held = cache.num_free_blocks
        with pytest.raises(OutOfCacheMemory):
            cache.fork_many(0, list(range(20, 60)))
        assert cache.num_free_blocks == held and 20 not in cache.tables
    for s in range(6):
        cache.free(s)
    assert cache.num_free_blocks == 24


def test_compact_keeps_every_sequence() -> None:
    cache = _cache(blocks=40)
    rng = np.random.default_rng(0)
    for s in range(8):
        cache.append(s, int(rng.integers(1, 30)))
    cache.fork(2, 20)
    cache.fork_many(3, [21, 22])
    for s in (0, 3, 5):
        cache.free(s)
    live = [1, 2, 4, 6, 7, 20, 21, 22]
    was = {s: _content(cache, s) for s in live}
    used = cache.allocator.num_used
    assert cache.compact() > 0
    assert cache.moves == 1
    for s in live:
        assert torch.equal(_content(cache, s), was[s])
        assert max(cache.tables[s].blocks) < used
    cache.allocator.check_invariants()
    assert cache.compact() == 0
    cache.append(50, 3)
    assert cache.tables[50].blocks == [used]  # the lowest free block
    for s in (*live, 50):
        cache.free(s)
    cache.allocator.check_invariants()
    assert cache.num_free_blocks == 40


def test_pools_beyond_four_gigabytes() -> None:
    """Blocks and slots whose offsets pass 32 bits, in bytes and in elements."""
    from microserve_b200.cache import copy_blocks, move_tokens

    blocks = (2 ** 32 + 2 ** 26) // (16 * 64)
    pool = torch.empty((2, 1, blocks, 1, 16, 64), dtype=torch.bfloat16, device=DEV)
    at = torch.tensor([3, blocks - 2], device=DEV)
    pool[:, :, at] = torch.randn((2, 1, 2, 1, 16, 64), device=DEV).to(torch.bfloat16)
    was = pool[:, :, at].clone()
    copy_blocks(pool, _i32([3, blocks - 2]), _i32([blocks - 1, 4]))
    assert torch.equal(pool[:, :, blocks - 1], was[:, :, 0]) and torch.equal(pool[:, :, 4], was[:, :, 1])
    last = (blocks - 2) * 16
    move_tokens(pool, _i32([[last + 5, 3 * 16 + 1]]), _i32([[3 * 16 + 1, last + 9]]))
    assert torch.equal(pool[:, :, 3, :, 1], was[:, :, 1, :, 5])
    assert torch.equal(pool[:, :, blocks - 2, :, 9], was[:, :, 0, :, 1])


@pytest.mark.parametrize("which", ["target", "draft", "both"])
def test_compaction_between_chained_rounds(golden, which) -> None:
    """The caches of a speculative decoder compacted between rounds, with the next round's draft side
    planned on the device already: the streams stay what they are without."""
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, SamplingConfig
    from microserve_b200.scheduler import Request
    from microserve_b200.speculative import SpeculativeDecoder

    from .test_gpu_model import device_model

    target, draft = device_model(golden, "target"), device_model(golden, "draft")
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 32, int(n)).tolist() for n in rng.integers(2, 20, 6)]
    sc = SamplingConfig(temperature=0.9, top_k=20, max_new_tokens=200)

    def serve(compact: bool):
        dec = SpeculativeDecoder(target, draft, CacheConfig(8, 128), gamma=3)
        cache = PagedKVCache(target.cfg, CacheConfig(8, 128), DEV)
        reqs = [Request(i, list(p), sc) for i, p in enumerate(prompts)]
        gens = {i: torch.Generator().manual_seed(900 + i) for i in range(6)}
        live, moved = [0, 1, 2, 3, 4, 5], 0
        for call in range(9):
            if call == 3:  # holes in the middle of both pools
                for i in (1, 4):
                    cache.free(i)
                    dec.free(i)
                live = [0, 2, 3, 5]
            if compact and call in (4, 5, 7):
                moved += cache.compact() if which != "draft" else 0
                moved += dec.draft_cache.compact() if which != "target" else 0
                cache.allocator.check_invariants()
            for i, toks in zip(live, dec.step([reqs[i] for i in live], cache, gens), strict=True):
                reqs[i].output_ids.extend(toks)
        return [r.output_ids for r in reqs], moved, dec

    want, _, plain = serve(False)
    got, moved, dec = serve(True)
    assert got == want and moved > 0
    assert dec.lookahead_hits > 0 and (which == "target" or plain.lookahead_hits > dec.lookahead_hits)

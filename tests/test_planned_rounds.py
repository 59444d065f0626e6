"""A planned round holds its draft tables on the device: it has to be dropped when a block of one of
them is replaced, by whichever call."""

from __future__ import annotations

import pytest


def test_unsharing_one_block_counts_as_a_change_of_blocks() -> None:
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, ModelConfig

    c = PagedKVCache(ModelConfig(max_seq_len=256), CacheConfig(8, 24), device="cpu")
    c.append(0, 5)
    c.fork(0, 1)
    c.unshare_last_block(1)
    assert c.moves == 1 and c.tables[0].blocks != c.tables[1].blocks
    c.unshare_last_block(0)  # nothing is shared any more
    assert c.moves == 1
    c.append(0, 0)
    c.allocator.check_invariants()


@pytest.mark.gpu
def test_unsharing_between_chained_rounds(golden) -> None:
    """A fork of a draft sequence keeps what it shared, although the next round was planned before the
    sequence took a block of its own."""
    import numpy as np
    import torch

    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, SamplingConfig
    from microserve_b200.scheduler import Request
    from microserve_b200.speculative import SpeculativeDecoder

    from .test_gpu_model import device_model

    target, draft = device_model(golden, "target"), device_model(golden, "draft")
    rng = np.random.default_rng(5)
    prompts = [rng.integers(0, 32, int(n)).tolist() for n in rng.integers(2, 20, 4)]
    sc = SamplingConfig(temperature=0.9, top_k=20, max_new_tokens=200)

    def serve(change: bool):
        dec = SpeculativeDecoder(target, draft, CacheConfig(64, 32), gamma=3)
        cache = PagedKVCache(target.cfg, CacheConfig(8, 128), "cuda")
        reqs = [Request(i, list(p), sc) for i, p in enumerate(prompts)]
        gens = {i: torch.Generator().manual_seed(900 + i) for i in range(4)}
        held = None
        for call in range(7):
            if change and call == 4:
                dec.draft_cache.fork(2, 77)
                page = dec.draft_cache.tables[77].blocks[-1]
                dec.draft_cache.unshare_last_block(2)
                assert dec.draft_cache.tables[2].blocks[-1] != page
                torch.cuda.synchronize()
                held = (page, dec.draft_cache.pool[:, :, page].clone())
            for i, toks in enumerate(dec.step(reqs, cache, gens)):
                reqs[i].output_ids.extend(toks)
        return [r.output_ids for r in reqs], held, dec

    want, _, plain = serve(False)
    got, (page, was), dec = serve(True)
    assert got == want
    assert torch.equal(dec.draft_cache.pool[:, :, page], was)
    assert 0 < dec.lookahead_hits < plain.lookahead_hits

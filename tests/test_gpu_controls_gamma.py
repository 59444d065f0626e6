"""Penalties beside rounds of more proposals than they count: ordinary passes, not a round that fails."""

from __future__ import annotations

import pytest
import torch

from .test_gpu_controls_engine import _engine, _prompts, assert_greedy

pytestmark = pytest.mark.gpu


def test_rounds_too_long_for_penalties(golden) -> None:
    from microserve_b200 import _lib
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, SamplingConfig
    from microserve_b200.scheduler import Request

    eng = _engine(golden, 65, blocks=256)
    prompts = _prompts(golden, 3)
    plain = SamplingConfig(temperature=0.0, max_new_tokens=12)
    biased = SamplingConfig(temperature=0.0, max_new_tokens=12, logit_bias={3: 4.0})
    penalised = SamplingConfig(temperature=0.0, max_new_tokens=6, frequency_penalty=0.9)
    settings = [plain, biased, penalised]
    reqs = [eng.add_request(p, s) for p, s in zip(prompts, settings)]
    got = {o.request_id: o.output_ids for o in eng.run()}
    for r, p, s in zip(reqs, prompts, settings):
        assert_greedy(eng.model, p, s, got[r.request_id])
    assert eng.stats.num_spec_rounds > 0  # the others, once the penalised one is done

    # a round controls biases whatever its length, and penalties up to 64 proposals
    assert eng.spec.can_control(plain) and eng.spec.can_control(biased)
    assert not eng.spec.can_control(penalised)

    # the decoder refuses before it takes anything
    dec = eng.spec
    cache = PagedKVCache(eng.model.cfg, CacheConfig(8, 64, eng.model.cfg.dtype), "cuda")
    free = dec.draft_cache.num_free_blocks
    request = Request(99, prompts[0], penalised)
    with pytest.raises(ValueError, match="64 proposals"):
        dec.step([request], cache, {99: torch.Generator().manual_seed(0)})
    assert dec.draft_cache.num_free_blocks == free and cache.num_free_blocks == 64
    assert not dec.controls._slot
    assert _lib.device_error() == 0

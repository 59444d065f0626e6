"""What the logit controls refuse on the host, before a request or a pass changes anything (no GPU)."""

from __future__ import annotations

import numpy as np
import pytest
import torch

INF = float("inf")


def request(rid: int = 0, **sampling):
    from microserve_b200.config import SamplingConfig
    from microserve_b200.scheduler import Request

    return Request(rid, [1, 2], SamplingConfig(**sampling))


def controls(vocab: int = 10):
    from microserve_b200.logits import RequestControls

    return RequestControls(vocab, torch.device("cpu"))


def only(*tokens: int):
    return lambda said: np.isin(np.arange(10), tokens)


@pytest.mark.parametrize("value", [-INF, -1e39])  # (below the range of float32)
def test_biases_that_ban_what_the_mask_allows_are_refused(value: float) -> None:
    """A row of -inf alone has nothing to draw: the mask and the bans are looked at together."""
    rc = controls()
    banned = {5: value, 7: value}
    with pytest.raises(ValueError, match="no token"):
        rc.masks_of([request(), request(1, allowed_tokens=only(5, 7), logit_bias=banned)])
    for ok in (request(allowed_tokens=only(5, 6, 7), logit_bias=banned),
               request(allowed_tokens=only(5, 7), logit_bias={5: value, 7: -100.0}),
               request(allowed_tokens=only(5, 7), logit_bias={6: value})):
        got = rc.masks_of([ok])
        assert np.array_equal(got[0], ok.sampling.allowed_tokens([]))  # the mask itself is as it was given


def test_biases_that_ban_the_whole_vocabulary_are_refused() -> None:
    rc = controls()
    every = {v: -INF for v in range(10)}
    with pytest.raises(ValueError, match="every token"):
        rc.check(request(logit_bias=every).sampling)
    with pytest.raises(ValueError, match="every token"):  # a decoder's caller has not called check
        rc.prepare([request(1, logit_bias={1: 2.0}), request(logit_bias=every)])
    assert not rc._slot
    every[3] = -1e30
    rc.check(request(logit_bias=every).sampling)


@pytest.mark.parametrize("kw", [
    dict(repetition_penalty=1e-46),  # 0 in float32: x / 0
    dict(repetition_penalty=2.0 ** -150),
    dict(repetition_penalty=1e39),
    dict(presence_penalty=1e39), dict(presence_penalty=-1e39),
    dict(frequency_penalty=1e39),  # inf * 0 occurrences
    dict(frequency_penalty=-1e39),
    dict(frequency_penalty=1e37, max_new_tokens=100),  # beyond the range once a token repeats enough
])
def test_penalties_beyond_float32_are_refused(kw: dict) -> None:
    from microserve_b200.config import SamplingConfig
    from microserve_b200.sampling import validate

    with pytest.raises(ValueError, match="penalty"):
        validate(SamplingConfig(**kw))


def test_penalties_within_float32_are_accepted() -> None:
    from microserve_b200.config import SamplingConfig
    from microserve_b200.sampling import validate

    for kw in (dict(repetition_penalty=1e-45), dict(repetition_penalty=3e38), dict(presence_penalty=-3e38),
               dict(frequency_penalty=1e36, max_new_tokens=100), dict(frequency_penalty=3e38, max_new_tokens=1),
               dict(frequency_penalty=0.5, max_new_tokens=0)):
        cfg = SamplingConfig(**kw)
        validate(cfg)
        for v in (cfg.repetition_penalty, cfg.presence_penalty, cfg.frequency_penalty):
            assert np.isfinite(np.float32(v))
        assert np.float32(cfg.repetition_penalty) > 0

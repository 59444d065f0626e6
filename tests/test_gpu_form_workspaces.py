"""Passes of one model with a form share no workspace: not with one another, nor with passes without."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .test_gpu_tree import _cache, _model

pytestmark = pytest.mark.gpu


def _batch(model, n: int, seed: int, blocks: int = 200):
    from microserve_b200.batching import build_paged_batch

    rng = np.random.default_rng(seed)
    cache = _cache(model, blocks=blocks)
    return build_paged_batch(cache, [0, 1, 2], [rng.integers(0, 61, n).tolist() for _ in range(3)], [0] * 3), cache


def test_a_graph_without_a_form_keeps_its_workspace() -> None:
    """A larger pass with a form after the capture replaces nothing that the graph uses."""
    from microserve_b200.attention import AttentionForm

    model = _model()
    batch, cache = _batch(model, 9, 0)
    want = model.forward_paged(batch, cache).clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        got = model.forward_paged(batch, cache)
    held = model._ws
    big, big_cache = _batch(model, 200, 1)
    model.forward_paged(big, big_cache, form=AttentionForm(softcap=2.0))
    assert model._ws is held
    got.zero_()
    g.replay()
    torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)


def test_passes_with_forms_on_two_streams_at_once() -> None:
    from microserve_b200.attention import AttentionForm

    model = _model()
    forms = [AttentionForm(softcap=2.0), AttentionForm(window=5), None]
    held = [_batch(model, n, n) for n in (150, 200, 180)]
    want = [model.forward_paged(b, c, form=f).clone() for (b, c), f in zip(held, forms)]
    streams = [torch.cuda.Stream() for _ in held]
    torch.cuda.synchronize()
    got = []
    for _ in range(20):
        for s, (b, c), f in zip(streams, held, forms):
            with torch.cuda.stream(s):
                got.append(model.forward_paged(b, c, form=f))
    torch.cuda.synchronize()
    for i, t in enumerate(got):
        torch.testing.assert_close(t, want[i % 3], rtol=1e-4, atol=1e-5)

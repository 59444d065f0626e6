"""An infinite value whose weight float32 cannot hold: the result is infinite all the same."""

from __future__ import annotations

import pytest
import torch

from .form_check import check, make, reference, run
from .test_gpu_form_infinities import INF, KERNELS, NAN

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_value_far_away(kernel, long, value) -> None:
    """The first key of a context whose scores fall with the distance, alone or in a KV range of its own."""
    dtype, hq, hkv, dh, n, _ = kernel
    cached = [3000, 2500] if long else [400, 330]
    x = make(53, dtype, hq, hkv, dh, 16, cached, [n, n], alibi=True)
    for b in range(2):
        x.v[x.tables[b, 0], :, b, 3 + b] = value
    ref, tol = reference(x)
    # (64 bits hold the weights of the nearer heads only: in the formula every value that is seen counts)
    for b in range(2):
        ref[b * n : (b + 1) * n, :, 3 + b] = value
    got = run(x)
    g = got.double().cpu()
    assert torch.equal(g.isnan(), ref.isnan())
    assert torch.equal(g.isposinf(), ref.isposinf()) and torch.equal(g.isneginf(), ref.isneginf())
    check(got, x, (ref, tol))

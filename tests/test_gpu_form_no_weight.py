"""Rows whose scores are all -inf give 0, as rows that see nothing do, whatever the values are."""

from __future__ import annotations

import pytest

import torch

from .form_check import check, make, reference, run
from .test_gpu_form_infinities import INF, KERNELS, NAN

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [1.0, INF, NAN])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_scores_of_minus_infinity(kernel, long, tree, value) -> None:
    """Every third token's; the others' scores are finite, and see the value."""
    dtype, hq, hkv, dh, n, seqs = kernel
    cached = [2900, 1500] if long else [150] * seqs
    x = make(58, dtype, hq, hkv, dh, 16, cached, [n] * len(cached), tree=tree)
    x.k[..., 3] = torch.where(x.k[..., 3].isfinite(), torch.ones_like(x.k[..., 3]), x.k[..., 3])
    x.q[::3, :, 3] = -INF
    for b in range(len(cached)):
        x.v[x.tables[b, 1], :, 2, 5] = value
        if n > 1:
            j = x.context[b] - 1
            x.v[x.tables[b, j // 16], :, j % 16, 6] = value
    ref, tol = reference(x)
    ref[::3], tol[::3] = 0.0, 0.0
    got = run(x)
    assert not bool(got[::3].any())
    assert torch.equal(got.double().cpu().isnan(), ref.isnan())
    check(got, x, (ref, tol))

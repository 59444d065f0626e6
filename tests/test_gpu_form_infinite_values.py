"""Values that are not finite where every row of a step sees them."""

from __future__ import annotations

import pytest
import torch

from .form_check import check, make, reference, run
from .test_gpu_form_infinities import INF, KERNELS, NAN

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("form", [{}, dict(alibi=True, softcap=20.0), dict(tree=True)], ids=str)
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_value_that_every_row_sees(kernel, form, value) -> None:
    """One dimension of one value of each sequence's cached context is infinite or NaN: that dimension of
    the result is, and no other."""
    dtype, hq, hkv, dh, n, seqs = kernel
    x = make(43, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs, **form)
    for b in range(seqs):
        j = (37 * b) % 128
        x.v[x.tables[b, j // 16], :, j % 16, b % dh] = value
    ref, tol = reference(x)
    got = run(x)
    g = got.double().cpu()
    assert torch.equal(g.isnan(), ref.isnan())
    assert torch.equal(g.isposinf(), ref.isposinf()) and torch.equal(g.isneginf(), ref.isneginf())
    check(got, x, (ref, tol))

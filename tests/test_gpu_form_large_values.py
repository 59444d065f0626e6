"""Values near the type's largest: a mean of finite values is finite, in every kernel."""

from __future__ import annotations

import pytest
import torch

from .form_check import check, make, run
from .test_gpu_form_infinities import KERNELS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("long", [False, True])
@pytest.mark.parametrize("spread", [0.0, 0.5, 2.0])
@pytest.mark.parametrize("kernel", KERNELS)
def test_sums_of_the_largest_values(kernel, spread, long) -> None:
    """All values are the type's largest but for their signs, by dimension: the result of each is nearly
    that, and sums of them before the division would not be finite."""
    dtype, hq, hkv, dh, n, seqs = kernel
    cached, n_seqs = ([2900, 1500], 2) if long else ([150] * seqs, seqs)
    x = make(44, dtype, hq, hkv, dh, 16, cached, [n] * n_seqs, spread=spread)
    held = x.v.isfinite()
    # (results may be off by a few roundings of 2^-8 in bf16, of 2^-20 in float32, which must not overflow either)
    big = torch.finfo(dtype).max * (0.98 if dtype is torch.bfloat16 else 1 - 2.0 ** -10)
    sign = torch.where(torch.arange(dh) % 3 == 0, -1.0, 1.0)
    x.v = torch.where(held, (big * sign).to(dtype), x.v)
    check(run(x), x)


@pytest.mark.parametrize("kernel", KERNELS)
def test_scores_that_grow(kernel) -> None:
    """Every key scores a little more than the one before: sums grow while the maximum does."""
    dtype, hq, hkv, dh, n, seqs = kernel
    x = make(45, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs)
    x.q[:] = 1.0
    for b in range(seqs):
        for j in range(x.context[b]):
            x.k[x.tables[b, j // 16], :, j % 16] = 0.04 * (j % 64) * dh ** -0.5
    held = x.v.isfinite()
    x.v = torch.where(held, torch.tensor(torch.finfo(dtype).max * 0.98).to(dtype), x.v)
    check(run(x), x)

"""Caps of any size: one far above the scores leaves them as they are."""

from __future__ import annotations

import pytest
import torch

from .form_check import check, make, run
from .test_gpu_form_infinities import KERNELS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("cap", [1e4, 1e6, 1e9, 1e20, 3e38])
@pytest.mark.parametrize("kernel", KERNELS)
def test_caps_far_above_the_scores(kernel, cap, tree) -> None:
    dtype, hq, hkv, dh, n, seqs = kernel
    x = make(48, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs, softcap=cap, tree=tree)
    check(run(x), x)


@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_rows_near_the_cap_beside_rows_far_below(kernel, alibi) -> None:
    """Some rows reach the cap, the others do not lose bits to it."""
    dtype, hq, hkv, dh, n, seqs = kernel
    x = make(49, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs, softcap=1e5, alibi=alibi)
    x.q[::3, ::2] *= 65536.0
    check(run(x), x)


@pytest.mark.parametrize("cap", [0.5, 50.0, 1e5])
@pytest.mark.parametrize("kernel", KERNELS)
def test_keys_near_the_cap_beside_keys_far_below(kernel, cap) -> None:
    x = make(50, *kernel[:4], 16, [150] * kernel[5], [kernel[4]] * kernel[5], softcap=cap)
    for b in range(kernel[5]):
        j = 9 * b % 140
        x.k[x.tables[b, j // 16], :, j % 16] *= cap / 4
    check(run(x), x)

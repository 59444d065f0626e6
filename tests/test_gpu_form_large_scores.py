"""Scores far beyond what float32 resolves: the largest has to keep a weight, and no weight may overflow."""

from __future__ import annotations

import pytest
import torch

from .form_check import make, run
from .test_gpu_form_infinities import KERNELS

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("scale", [1e4, 1e8, 1e12, 1e20])
@pytest.mark.parametrize("alibi", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_row_that_sees_one_key_takes_its_value(kernel, alibi, scale) -> None:
    dtype, hq, hkv, dh, n, seqs = kernel
    x = make(46, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs, window=1, scale=scale, alibi=alibi)
    got = run(x).cpu()
    for b in range(seqs):
        for i in range(n):
            j, row = 150 + i, b * n + i
            v = x.v[x.tables[b, j // 16], :, j % 16].repeat_interleave(hq // hkv, 0)
            # (p v / p in float32, within 2^-22 of v, and rounded to v in bf16)
            off = 0.0 if dtype is torch.bfloat16 else 2.0 ** -22
            assert bool(((got[row] - v).abs() <= off * v.abs()).all()), (b, i)


@pytest.mark.parametrize("scale", [1.0, 1e6, 1e10, 1e15])
@pytest.mark.parametrize("cap", [0.0, 1e12])
@pytest.mark.parametrize("kernel", KERNELS)
def test_equal_scores_of_any_size_share_the_weight(kernel, cap, scale) -> None:
    """All keys of a sequence alike: the result is the mean of the values that are seen, off by at most a
    sum's roundings and, in bf16, those of the weights and of the result."""
    dtype, hq, hkv, dh, n, seqs = kernel
    x = make(47, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs, scale=scale, softcap=cap)
    key = torch.randn(dh, generator=torch.Generator().manual_seed(1)).to(dtype)
    x.k = torch.where(x.k.isfinite(), key, x.k)
    got = run(x).double().cpu()
    for b in range(seqs):
        pages = torch.from_numpy(x.tables[b, : -(-x.context[b] // 16)].astype("int64"))
        v = x.v[pages].permute(1, 0, 2, 3).reshape(hkv, -1, dh).double()
        for i in range(n):
            seen = v[:, : 150 + i + 1]
            want = seen.mean(1).repeat_interleave(hq // hkv, 0)
            size = seen.abs().mean(1).repeat_interleave(hq // hkv, 0)
            tol = 2.0 ** -23 * (150 + n + 8) * size
            if dtype is torch.bfloat16:
                tol = tol + 2.0 ** -8 * (2 * want.abs() + size)
            assert bool(((got[b * n + i] - want).abs() <= tol).all()), (b, i)

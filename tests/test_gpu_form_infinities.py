"""Keys and values that are not finite and that a row sees: the formula's infinities and NaN, whichever
kernel takes the call and wherever in a step the key stands."""

from __future__ import annotations

import pytest
import torch

from .form_check import check, make, reference, run

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
INF, NAN = float("inf"), float("nan")

# dtype, hq, hkv, dh, tokens a sequence, sequences: CUDA cores; mma.sync with 16 and 32 rows; tcgen05 in
# tiles of 64 rows of many sequences, of 128 and of 256
KERNELS = [(F32, 2, 1, 32, 3, 16), (BF16, 4, 1, 128, 3, 16), (BF16, 8, 1, 64, 4, 16), (BF16, 64, 8, 64, 5, 40),
           (BF16, 64, 8, 128, 3, 40), (BF16, 8, 2, 64, 20, 16), (BF16, 8, 1, 128, 12, 16), (BF16, 8, 1, 64, 20, 16),
           (BF16, 8, 1, 128, 20, 16)]


def _inputs(kernel, seed: int, **form):
    dtype, hq, hkv, dh, n, seqs = kernel
    return make(seed, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs, **form)


def _held(got: torch.Tensor, x) -> None:
    ref, tol = reference(x)
    assert torch.equal(got.double().cpu().isnan(), ref.isnan())
    check(got, x, (ref, tol))


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("form", [{}, dict(alibi=True), dict(softcap=20.0), dict(tree=True)], ids=str)
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_key_that_is_not_finite(kernel, form, value) -> None:
    """One dimension of one key in each sequence, at another place modulo 16 in each: the score is NaN, or
    infinite with the sign of the query's dimension.  In the cached context, which every row sees."""
    x = _inputs(kernel, 40, **form)
    for b in range(len(x.context)):
        j = 32 * (b % 4) + b % 16
        x.k[x.tables[b, j // 16], :, j % 16, 3] = value
    _held(run(x), x)


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_key_of_the_pass_that_is_not_finite(kernel, value) -> None:
    """Among the pass's own tokens: rows before it do not see it."""
    x = _inputs(kernel, 41)
    n = kernel[4]
    for b in range(len(x.context)):
        j = 150 + b % n
        x.k[x.tables[b, j // 16], :, j % 16, 3] = value
    _held(run(x), x)


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_long_context_with_a_key_that_is_not_finite(kernel, first) -> None:
    """Two sequences, whose KV axis is cut into ranges: one range alone holds the key."""
    dtype, hq, hkv, dh, n, _ = kernel
    x = make(42, dtype, hq, hkv, dh, 16, [3000, 2500], [n, n])
    j = 3 if first else 2307
    x.k[x.tables[0, j // 16], :, j % 16, 3] = INF
    _held(run(x), x)

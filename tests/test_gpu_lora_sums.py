"""The adapters' long sums: no drift from the tensor cores' truncation, whatever kernel takes the call."""

from __future__ import annotations

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda"


def run(of: np.ndarray, rank: int, K: int, N: int) -> tuple[torch.Tensor, torch.Tensor]:
    """(the kernel's result, the adapters' part in 64 bits) over a base of zeros, scales 1."""
    from microserve_b200.lora import LoraPlan, LoraProjection, lora_add

    n = int(of.max()) + 1
    g = torch.Generator(device=DEV).manual_seed(K + n)
    x = torch.randn((len(of), K), generator=g, device=DEV).bfloat16()
    a = (torch.randn((n * rank, K), generator=g, device=DEV) * K ** -0.5).bfloat16()
    b = (torch.randn((n * rank, N), generator=g, device=DEV) * 0.2).bfloat16()
    i32 = dict(dtype=torch.int32, device=DEV)
    proj = LoraProjection(a=a, b=b, offsets=torch.arange(n, **i32) * rank, ranks=torch.full((n,), rank, **i32),
                          scales=torch.ones(n, device=DEV), max_rank=rank, slices=[N])
    got = lora_add(x, torch.zeros((len(of), N), device=DEV), proj, LoraPlan.build(of, DEV))
    want = torch.empty((len(of), N), dtype=torch.float64, device=DEV)
    for i in range(n):
        t = torch.from_numpy(np.flatnonzero(of == i)).to(DEV)
        rows = slice(i * rank, (i + 1) * rank)
        want[t] = (x[t].double() @ a[rows].double().t()) @ b[rows].double()
    return got.double(), want


@pytest.mark.parametrize("tokens,adapters,rank,mmas", [
    (32, 4, 16, 2),  # both products in one launch; the second on the CUDA cores
    (200, 40, 16, 8 + 3),  # 5 tokens a tile
    (200, 40, 64, 8 + 12),
    (240, 20, 16, 8 + 3),  # 12 a tile
    (240, 20, 64, 4 + 12),
    (990, 33, 16, 4 + 3),  # 30 a tile, through shared memory
    (990, 33, 128, 4 + 24),
    (9600, 1, 16, 32 + 3),  # a prompt's, on tcgen05
    (9600, 1, 128, 32 + 24),
])
def test_long_sums_do_not_drift(tokens: int, adapters: int, rank: int, mmas: int) -> None:
    """An MMA's running sum loses what is below its 24 bits, always towards zero: on average
    half a unit, at most 2^-24 of the sum; the running sum is on average half of the final one
    towards its sign, so a chain of n of them comes out up to n 2^-25 too small.  Chains are
    ``mmas`` long: the partial sums of the first product, and in the second one three for every
    16 rank rows.  Everything else rounds to nearest and averages out over the thousands of values
    (2^-24 / sqrt(500) is below 2^-28).  Unbroken sums over K lose more than the bound."""
    of = np.arange(tokens) % adapters
    got, want = run(of, rank, 28672, 256)
    drift = float(((want - got) * want.sign()).mean() / want.abs().mean())
    assert abs(drift) <= mmas * 2.0 ** -25 + 2.0 ** -28
    # and no value is off by more than the roundings that meet in it
    assert float((got - want).norm() / want.norm()) <= 1e-6

"""An infinite input of a token with an adapter: the formula's +-inf, whatever kernel takes the call."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .test_gpu_lora import DEV, Case

pytestmark = pytest.mark.gpu

CASES = {
    "one_launch": dict(of=[0, 1, 0], ranks=[16, 5], K=256, slices=[128]),
    "few": dict(of=np.arange(60) % 12, ranks=[16, 5, 24] * 4, K=256, slices=[128]),
    "some": dict(of=np.arange(60) % 5, ranks=[40, 5, 24, 16, 1], K=264, slices=[128, 32, 32]),
    "tiles": dict(of=np.arange(200) % 6, ranks=[40, 5, 24, 16, 1, 72], K=264, slices=[128, 32, 32]),
    "prompt": dict(of=np.arange(200) // 100, ranks=[24, 5], K=256, slices=[256, 128]),
    "long_prompt": dict(of=np.arange(4300) // 4000, ranks=[24, 5], K=256, slices=[256, 128]),
    # slices that end inside the columns of one step
    "some_slice_edges": dict(of=np.arange(60) % 5, ranks=[40, 5, 24, 16, 1], K=264, slices=[72, 8, 27, 21]),
    "prompt_slice_edges": dict(of=np.arange(200) // 100, ranks=[24, 5], K=256, slices=[203, 150, 47]),
    "prompt_narrow_slices": dict(of=np.arange(200) // 100, ranks=[24, 5], K=256, slices=[30, 40, 58]),
    "rows_off_16_bytes": dict(of=np.arange(60) % 3, ranks=[40, 5, 24], K=67, slices=[50]),
    "f32": dict(of=np.arange(60) % 3, ranks=[40, 5, 24], K=67, slices=[50], dtype="float32"),
    "f32_long_k": dict(of=np.arange(60) % 3, ranks=[40, 5, 24], K=300, slices=[50], dtype="float32"),
}


@pytest.mark.parametrize("name", list(CASES))
def test_an_infinite_input_gives_the_formulas_infinities(name: str) -> None:
    from microserve_b200 import _lib
    from microserve_b200.lora import lora_add

    kw = {"dtype": "bfloat16", **CASES[name]}
    c = Case(np.asarray(kw.pop("of")).tolist(), **kw)
    bad = [0, c.T // 2, c.T - 1]
    k0 = c.K - 2
    # B's signs are those of what it meets, times one of the column's: all products are +inf, or all -inf
    of_col = np.repeat(np.arange(c.ns), c.slices)
    sign = torch.from_numpy(np.where(np.arange(c.N) % 3, 1.0, -1.0)).to(DEV)
    a, b = c.a.clone(), c.b
    a[:, k0] = torch.where(a[:, k0] == 0, 1.0, a[:, k0])
    c.a.copy_(a)
    for o, r in zip(c.offs, c.ranks):
        for j in range(c.ns):
            at = torch.from_numpy(np.flatnonzero(of_col == j)).to(DEV)
            s = a[c.ns * o + j * r : c.ns * o + (j + 1) * r, k0].double().sign()
            mag = b[o : o + r, at].abs().double().clamp(min=0.01)
            b[o : o + r, at] = (mag * s[:, None] * sign[at]).to(b.dtype)
    clean = lora_add(c.x, c.base, c.proj, c.plan)
    c.x[bad, k0] = float("inf")
    for out in (torch.float32, torch.bfloat16):
        got = lora_add(c.x, c.base, c.proj, c.plan, out_dtype=out)
        assert torch.equal(got[bad].double(), (sign * float("inf")).expand(len(bad), -1))
        keep = torch.ones(c.T, dtype=torch.bool, device=DEV)
        keep[bad] = False
        assert torch.isfinite(got[keep]).all()
        if out is torch.float32:
            assert torch.equal(got[keep], clean[keep])
    assert _lib.device_error() == 0

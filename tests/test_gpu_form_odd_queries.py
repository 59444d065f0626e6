"""Queries that are not finite hurt their own rows only, and few values among many keys cost no more than a
look at the values."""

from __future__ import annotations

import pytest
import torch

from .form_check import DEV, check, make, reference, run
from .test_gpu_form_infinities import INF, KERNELS, NAN

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("value", [INF, -INF, NAN])
@pytest.mark.parametrize("form", [{}, dict(tree=True, softcap=20.0)], ids=str)
@pytest.mark.parametrize("kernel", KERNELS)
def test_a_query_that_is_not_finite(kernel, form, value) -> None:
    dtype, hq, hkv, dh, n, seqs = kernel
    x = make(51, dtype, hq, hkv, dh, 16, [150] * seqs, [n] * seqs, **form)
    x.q[::3, 1, 5] = value
    ref, tol = reference(x)
    got = run(x)
    assert torch.equal(got.double().cpu().isnan(), ref.isnan())
    check(got, x, (ref, tol))


@pytest.mark.parametrize("value", [INF, NAN])
@pytest.mark.parametrize("dh", [64, 128])
def test_long_prompts_of_which_all_tokens_see_one_odd_value(dh, value) -> None:
    """In its dimension every result is what the value is, in the others as without it; in less than twenty times
    the time (a row at a time, key by key, it would take a thousand times as long)."""
    from microserve_b200.attention import paged_attention

    g = torch.Generator(device=DEV).manual_seed(0)
    x = make(52, torch.bfloat16, 1, 1, 64, 16, [0], [2048])
    q = torch.randn((2048, 32, dh), generator=g, device=DEV).bfloat16()
    k, v = (torch.randn((x.k.shape[0], 8, 16, dh), generator=g, device=DEV).bfloat16() for _ in range(2))
    batch, form = x.batch(), x.form()

    def timed():
        paged_attention(q, k, v, batch, form)
        a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        a.record()
        for _ in range(5):
            out = paged_attention(q, k, v, batch, form)
        b.record()
        torch.cuda.synchronize()
        return out, a.elapsed_time(b)

    want, before = timed()
    v[x.tables[0, 0], :, 1, 7] = value
    got, after = timed()
    rest = [d for d in range(dh) if d != 7]
    assert torch.equal(got[:, :, rest], want[:, :, rest])
    assert torch.equal(got[0], want[0])  # the first token does not see the second
    odd = got[1:, :, 7]
    assert bool((odd.isnan() if value != value else odd == value).all())
    assert after < 20 * before

"""Rows that are computed again (infinite values, sums that overflow) in the layouts that the kernels take
value by value: strided and unaligned queries and results, unaligned pools, small heads, padded batches."""

from __future__ import annotations

import pytest
import torch

from .form_check import DEV, check, make, reference, run

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
INF = float("inf")


def _values(x, what: str):
    """Infinite values in two places, or the type's largest everywhere."""
    if what == "large":
        big = torch.finfo(x.v.dtype).max * (0.98 if x.v.dtype is BF16 else 1 - 2.0 ** -10)
        x.v = torch.where(x.v.isfinite(), torch.full_like(x.v, big), x.v)
    else:
        bs = x.v.shape[2]
        for b, j in ((0, 3), (1, x.context[1] - 2)):
            x.v[x.tables[b, j // bs], :, j % bs, 5] = INF
    return reference(x)


@pytest.mark.parametrize("what", ["large", "infinite"])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("dtype,hq,hkv,dh,n", [(F32, 8, 2, 64, 5), (BF16, 8, 2, 64, 5), (BF16, 8, 2, 128, 30),
                                               (BF16, 8, 1, 64, 40)])
@pytest.mark.parametrize("extra,shift", [(256, 0), (7, 0), (9, 1), (8, 8)])
def test_strides(dtype, hq, hkv, dh, n, extra, shift, tree, what) -> None:
    x = make(54, dtype, hq, hkv, dh, 16, [333, 90], [n, n], tree=tree)
    want = _values(x, what)
    T, width = 2 * n, hq * dh
    wide = torch.zeros((T, width + extra + shift), device=DEV, dtype=dtype)
    q = wide[:, shift : shift + width].view(T, hq, dh)
    q.copy_(x.q.to(DEV))
    holder = torch.full((T, width + extra + shift), 7.0, device=DEV, dtype=dtype)
    out = holder[:, shift : shift + width].view(T, hq, dh)
    check(run(x, q=q, out=out), x, want)
    assert bool((holder[:, :shift] == 7).all()) and bool((holder[:, shift + width :] == 7).all())


@pytest.mark.parametrize("what", ["large", "infinite"])
@pytest.mark.parametrize("dtype,hq,hkv,dh,bs", [(F32, 4, 2, 8, 4), (F32, 8, 1, 16, 8), (F32, 6, 2, 128, 5),
                                                (BF16, 4, 2, 8, 16), (BF16, 4, 2, 16, 16), (BF16, 4, 2, 32, 16),
                                                (BF16, 4, 2, 64, 12), (BF16, 3, 3, 128, 2)])
@pytest.mark.parametrize("cached", [[40, 7], [3000, 900]])
def test_caches_of_the_cuda_core_kernel(dtype, hq, hkv, dh, bs, cached, what) -> None:
    x = make(55, dtype, hq, hkv, dh, bs, cached, [5, 9], tree=True)
    want = _values(x, what)
    check(run(x), x, want)


@pytest.mark.parametrize("what", ["large", "infinite"])
@pytest.mark.parametrize("dtype,shift", [(F32, 1), (BF16, 1), (BF16, 4)])
def test_pools_that_start_anywhere(dtype, shift, what) -> None:
    from microserve_b200.attention import paged_attention

    x = make(56, dtype, 4, 2, 64, 16, [70, 20], [30, 9], tree=True)
    want = _values(x, what)
    pools = []
    for t in (x.k, x.v):
        flat = torch.empty(t.numel() + shift, dtype=dtype, device=DEV)
        pools.append(flat[shift:].view(t.shape).copy_(t))
    check(paged_attention(x.q.to(DEV), *pools, x.batch(), x.form()), x, want)


@pytest.mark.parametrize("what", ["large", "infinite"])
@pytest.mark.parametrize("hq,dh,n", [(4, 64, 1), (16, 128, 20), (16, 64, 40)])
def test_captured_and_replayed(hq, dh, n, what) -> None:
    """A graph of a call whose values are ordinary, replayed after they have become odd, and ordinary again."""
    from microserve_b200.attention import paged_attention

    x = make(57, BF16, hq, 2, dh, 16, [900, 300], [n, n], window=200, prefix=[20, 0])
    q, k, v, batch, form = x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), x.batch(), x.form()
    plain, before = reference(x), x.v.clone()
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(q, k, v, batch, form, out)
    g.replay()
    check(out, x, plain)
    want = _values(x, what)
    v.copy_(x.v)
    g.replay()
    check(out, x, want)
    v.copy_(before)
    g.replay()
    check(out, x, plain)

"""Low-rank adapters beside a shared projection (ms_lora_add) against the 64-bit restatement."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.controls import lora_row, swiglu

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Case:
    def __init__(self, of: list[int], ranks: list[int], K: int, slices: list[int], dtype: str, *,
                 interleaved: bool = False, seed: int = 0, gaps: bool = False) -> None:
        from microserve_b200.lora import LoraPlan, LoraProjection

        g = torch.Generator(device=DEV).manual_seed(seed + K + len(of))
        self.dt = getattr(torch, dtype)
        self.of, self.ranks, self.slices, self.interleaved = of, ranks, slices, interleaved
        T, N, ns = len(of), sum(slices), len(slices)
        offs = np.cumsum([0] + [r + (3 if gaps else 0) for r in ranks])
        R = int(offs[-1])
        self.offs, self.ns, self.N, self.T, self.K = offs[:-1], ns, N, T, K
        self.x = torch.randn((T, K), generator=g, device=DEV).to(self.dt)
        self.a = (torch.randn((ns * R, K), generator=g, device=DEV) * K ** -0.5).to(self.dt)
        self.b = (torch.randn((R, N), generator=g, device=DEV) * 0.2).to(self.dt)
        if gaps:  # the rows between adapters belong to nobody and may hold anything
            own = np.zeros(R, bool)
            for o, r in zip(self.offs, ranks):
                own[o : o + r] = True
            idle = torch.from_numpy(~own).to(DEV)
            self.b[idle] = float("nan")
            self.a.view(-1, K)[self._idle_rows()] = float("nan")
        self.base = torch.randn((T, N), generator=g, device=DEV)
        self.scales = torch.rand(len(ranks), generator=g, device=DEV) + 0.5
        i32 = lambda v: torch.tensor(np.asarray(v), dtype=torch.int32, device=DEV)  # noqa: E731
        self.proj = LoraProjection(a=self.a, b=self.b, offsets=i32(self.offs), ranks=i32(ranks),
                                   scales=self.scales, max_rank=max(ranks, default=0), slices=slices,
                                   interleaved=interleaved)
        self.plan = LoraPlan.build(of, DEV)

    def _idle_rows(self) -> torch.Tensor:
        own = np.zeros(self.a.shape[0], bool)
        for o, r in zip(self.offs, self.ranks):
            own[self.ns * o : self.ns * (o + r)] = True
        return torch.from_numpy(np.flatnonzero(~own)).to(DEV)

    def want(self) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
        col = np.arange(self.N)
        sl = (col // 8) % 2 if self.interleaved else np.repeat(np.arange(self.ns), self.slices)
        x, base = self.x.double().cpu().numpy(), self.base.double().cpu().numpy()
        a, b = self.a.double().cpu().numpy(), self.b.double().cpu().numpy()
        sc = self.scales.cpu().numpy()
        ys, parts, terms = base.copy(), np.zeros_like(base), np.zeros_like(base)
        for t, i in enumerate(self.of):
            if i < 0 or self.ranks[i] == 0:
                continue
            o, r = int(self.offs[i]), self.ranks[i]
            aa = a[self.ns * o : self.ns * (o + r)].reshape(self.ns, r, self.K)
            ys[t], parts[t], terms[t] = lora_row(x[t], base[t], aa, b[o : o + r], sc[i], sl)
        return ys, parts, terms

    def tolerance(self, y: np.ndarray, terms: np.ndarray, out: torch.dtype) -> np.ndarray:
        """The products are exact in float32; a sum of n terms, added in any order and
        truncated, is off by at most n 2^-23 of the terms' magnitudes (K in the first
        product, twice the padded rank in the second); s as hi + lo is off by 2^-17; one
        rounding of the result to `out`, and float32's of it before."""
        rank = 2 * (max(self.ranks, default=0) + 16)
        return terms * ((self.K + rank + 4) * 2.0 ** -23 + 2.0 ** -17) + \
            np.abs(y) * (EPS[out] + 2.0 ** -23) + 1e-30

    def check(self, got: torch.Tensor) -> None:
        y, part, terms = self.want()
        g = got.double().cpu().numpy()
        assert np.isfinite(g).all()
        err = np.abs(g - y)
        assert (err <= self.tolerance(y, terms, got.dtype)).all()
        # and over all values: the adapters' part to 2^-15 of its norm, which a wrong
        # adapter, slice, scale or rank row exceeds by far
        bound = 2.0 ** -15 * np.linalg.norm(part) + (EPS[got.dtype] + 2.0 ** -23) * np.linalg.norm(y)
        assert np.linalg.norm(err) <= bound


def mixed(n: int, adapters: int, seed: int = 0) -> list[int]:
    return np.random.default_rng(seed).integers(-1, adapters, n).tolist()


CASES = {
    "one_token": dict(of=[0], ranks=[16], K=2048, slices=[2048], dtype="bfloat16"),
    "one_token_of_none": dict(of=[-1], ranks=[16], K=64, slices=[128], dtype="bfloat16"),
    "no_adapters": dict(of=[-1, -1, -1], ranks=[], K=64, slices=[128], dtype="bfloat16"),
    "few": dict(of=[0, 1, -1, 1, 2, 0, 3], ranks=[16, 5, 0, 1], K=200, slices=[4096], dtype="bfloat16"),
    "few_in_a_long_tile": dict(of=[0] * 20 + [1, 2, -1], ranks=[16, 8, 3], K=4104, slices=[1000], dtype="bfloat16"),
    "few_and_small": dict(of=[0, -1], ranks=[7], K=8, slices=[8], dtype="bfloat16"),
    "few_and_wider": dict(of=[0, 1, 0], ranks=[16, 5], K=64, slices=[4104], dtype="bfloat16"),
    "few_of_rank_17": dict(of=[0, 1, 0], ranks=[17, 5], K=64, slices=[64], dtype="bfloat16"),
    "few_at_the_most": dict(of=list(range(16)) + list(range(16)), ranks=[16] * 16, K=520, slices=[72], dtype="bfloat16"),
    "one_more_than_few": dict(of=list(range(33)), ranks=[16] * 33, K=64, slices=[72], dtype="bfloat16"),
    "qkv_mixed": dict(of=mixed(77, 9), ranks=[8, 16, 32, 64, 1, 5, 24, 0, 128], K=2048,
                      slices=[2048, 256, 256], dtype="bfloat16"),
    "qkv_narrow_slices": dict(of=mixed(40, 3), ranks=[16, 8, 40], K=200, slices=[72, 8, 24], dtype="bfloat16"),
    "four_slices": dict(of=mixed(21, 2), ranks=[12, 30], K=136, slices=[64, 16, 40, 8], dtype="bfloat16"),
    "many_per_adapter": dict(of=mixed(700, 2), ranks=[64, 17], K=520, slices=[392], dtype="bfloat16"),
    "every_token_its_own": dict(of=list(range(150))[::-1], ranks=[16] * 150, K=1024, slices=[512], dtype="bfloat16"),
    "tile_edges": dict(of=[0] * 64 + [1] * 65 + [2] * 33 + [-1] * 31 + [3] * 32 + [4], ranks=[16] * 5, K=256,
                       slices=[128], dtype="bfloat16"),
    "largest_rank": dict(of=mixed(50, 2), ranks=[256, 200], K=264, slices=[136, 128, 64], dtype="bfloat16"),
    "long_k": dict(of=mixed(9, 3), ranks=[16, 16, 64], K=14336, slices=[256], dtype="bfloat16"),
    "gaps": dict(of=mixed(60, 3), ranks=[16, 5, 33], K=128, slices=[96, 32], dtype="bfloat16", gaps=True),
    "odd_k": dict(of=mixed(30, 2), ranks=[3, 20], K=67, slices=[50], dtype="bfloat16"),
    "odd_n": dict(of=mixed(30, 2), ranks=[3, 20], K=64, slices=[33, 18], dtype="bfloat16"),
    # long runs of one adapter: pairs of tiles, odd runs, a short last tile
    "prompts": dict(of=[0] * 300 + [-1] * 70 + [1] * 129 + [2] * 64 + [3] * 127, ranks=[16, 64, 8, 33], K=256,
                    slices=[384], dtype="bfloat16"),
    "prompts_interrupted": dict(of=([0] * 50 + [1] * 60) * 6, ranks=[128, 72], K=200, slices=[200], dtype="bfloat16"),
    "prompts_qkv": dict(of=[0] * 200 + [1] * 150, ranks=[40, 16], K=512, slices=[512, 64, 64], dtype="bfloat16"),
    "prompts_slice_edges": dict(of=[0] * 130 + [1] * 70 + [-1] * 40, ranks=[24, 64], K=128, slices=[203, 150, 47],
                                dtype="bfloat16"),
    "prompts_narrow_slices": dict(of=[0] * 130, ranks=[24], K=128, slices=[30, 40, 58], dtype="bfloat16"),
    "prompts_none": dict(of=[-1] * 200 + [0] * 64, ranks=[16], K=64, slices=[136], dtype="bfloat16"),
    "prompts_rank_256": dict(of=[0] * 140, ranks=[256], K=72, slices=[264], dtype="bfloat16"),
    "long_prompts": dict(of=[0] * 2070 + [-1] * 70 + [1] * 2150, ranks=[24, 64], K=200, slices=[136], dtype="bfloat16"),
    "long_prompts_shared_k": dict(of=[0] * 4300, ranks=[16], K=1096, slices=[72, 24], dtype="bfloat16"),
    "long_prompts_rank_256": dict(of=[0] * 4225, ranks=[256], K=72, slices=[64, 32, 40], dtype="bfloat16"),
    "f32": dict(of=mixed(61, 3), ranks=[4, 5, 12], K=128, slices=[128, 128, 128], dtype="float32"),
    "f32_long_k": dict(of=mixed(30, 3) + [-1], ranks=[4, 5, 12], K=259, slices=[70, 130], dtype="float32"),
    "f32_many_rows": dict(of=mixed(13, 2), ranks=[129, 3], K=40, slices=[300, 21], dtype="float32"),
    "f32_one_token": dict(of=[0], ranks=[3], K=256, slices=[257], dtype="float32"),
    "f32_full_tiles": dict(of=[0] * 150 + [-1] * 9, ranks=[6], K=96, slices=[96], dtype="float32"),
    "f32_most": dict(of=mixed(17, 2), ranks=[64, 64], K=256, slices=[33, 20, 1, 9], dtype="float32"),
    "f32_odd": dict(of=mixed(13, 2), ranks=[7, 1], K=33, slices=[29], dtype="float32"),
}


@pytest.mark.parametrize("name", list(CASES))
def test_adapters_match_the_restatement(name: str) -> None:
    from microserve_b200 import _lib
    from microserve_b200.lora import lora_add

    c = Case(**CASES[name])
    out = lora_add(c.x, c.base, c.proj, c.plan)
    c.check(out)
    c.check(lora_add(c.x, c.base, c.proj, c.plan, out_dtype=torch.bfloat16))
    for _ in range(2):  # no atomics on floats: the same bits every time
        assert torch.equal(lora_add(c.x, c.base, c.proj, c.plan), out)
    there = c.base.clone()
    assert lora_add(c.x, there, c.proj, c.plan, out=there) is there
    assert torch.equal(there, out)
    none = torch.tensor([i < 0 for i in c.of], device=DEV)
    assert torch.equal(out[none], c.base[none])
    assert _lib.device_error() == 0


@pytest.mark.parametrize("dtype,of,ranks,K,N", [
    ("bfloat16", mixed(80, 5), [8, 16, 32, 64, 3], 2048, 1408),
    ("bfloat16", [1] * 130, [16, 128], 264, 176),
    ("bfloat16", [0] * 300 + [1] * 200 + [-1] * 90 + [2] * 65, [128, 64, 20], 512, 1152),
    ("bfloat16", [-1] * 129 + [0] * 64, [8], 64, 144),
    ("bfloat16", [0, -1, 0], [16], 72, 16),
    ("float32", mixed(61, 3), [4, 5, 12], 128, 704),
    ("bfloat16", mixed(20, 2), [4, 9], 65, 48),
])
def test_swiglu_epilogue(dtype: str, of: list[int], ranks: list[int], K: int, N: int) -> None:
    from microserve_b200.lora import lora_add

    c = Case(of, ranks, K, [N // 2, N // 2], dtype, interleaved=True)
    c.check(lora_add(c.x, c.base, c.proj, c.plan))  # the sum itself, interleaved
    y, _, terms = c.want()
    tol = c.tolerance(y, terms, torch.float32)
    want = np.stack([swiglu(r) for r in y])
    v = y.reshape(len(of), -1, 2, 8)
    tv = tol.reshape(len(of), -1, 2, 8)
    gate, up = v[:, :, 0].reshape(want.shape), v[:, :, 1].reshape(want.shape)
    tg, tu = tv[:, :, 0].reshape(want.shape), tv[:, :, 1].reshape(want.shape)
    act = np.abs(gate / (1 + np.exp(-gate)))
    for od in (c.dt, torch.bfloat16):
        got = lora_add(c.x, c.base, c.proj, c.plan, swiglu=True, out_dtype=od)
        assert got.shape == (len(of), N // 2) and got.dtype == od
        err = np.abs(got.double().cpu().numpy() - want)
        # |silu'| < 1.1; exp and the quotient approximated to 2^-20 (|gate| < 16 here)
        bound = 1.1 * tg * np.abs(up) + act * tu + 1.1 * tg * tu + \
            np.abs(want) * (EPS[od] + 2.0 ** -20) + 1e-30
        assert (err <= bound).all()


@pytest.mark.parametrize("of,ranks,K,dtype", [
    ([0, 1, 0], [16, 8], 64, "bfloat16"),
    (mixed(40, 6), [256, 16, 40, 64, 3, 128], 64, "bfloat16"),
    ([0] * 24 + [1] * 30, [256, 40], 64, "bfloat16"),
    ([0] * 300, [128], 64, "bfloat16"),
    (mixed(30, 3), [256, 7, 20], 64, "float32"),
])
def test_the_base_is_rounded_once(of: list[int], ranks: list[int], K: int, dtype: str) -> None:
    """A base far above the adapters' part, a float32 result: beside the part's own error
    (Case.tolerance), one rounding of the sum."""
    from microserve_b200.lora import lora_add

    c = Case(of, ranks, K, [136], dtype)
    c.base *= 4096.0
    y, _, terms = c.want()
    got = lora_add(c.x, c.base, c.proj, c.plan).double().cpu().numpy()
    part = c.tolerance(np.zeros_like(y), terms, torch.float32)
    assert (np.abs(got - y) <= part * (1 + 2.0 ** -20) + np.abs(y) * 2.0 ** -24 * (1 + 2.0 ** -20)).all()


def test_strides_and_rows_behind_the_batch() -> None:
    from microserve_b200.lora import lora_add

    c = Case(mixed(50, 3), [16, 8, 20], 128, [128, 64], "bfloat16")
    T, K, N = c.T, c.K, c.N
    xs = torch.randn((T + 2, K + 24), device=DEV).bfloat16()
    xs[:T, :K] = c.x
    bs = torch.full((T + 2, N + 6), 5.0, device=DEV)
    bs[:T, :N] = c.base
    for od, pad in ((torch.float32, 10), (torch.bfloat16, 2), (torch.bfloat16, 1), (torch.float32, 3)):
        ob = torch.full((T + 2, N + pad), 9.0, device=DEV, dtype=od)
        lora_add(xs[:T, :K], bs[:T, :N], c.proj, c.plan, out=ob[:T, :N])
        c.check(ob[:T, :N])
        assert (ob[T:] == 9.0).all() and (ob[:, N:] == 9.0).all()
    lora_add(xs[:T, :K], bs[:T, :N], c.proj, c.plan, out=bs[:T, :N])
    c.check(bs[:T, :N])
    assert (bs[T:] == 5.0).all() and (bs[:, N:] == 5.0).all()
    xo = torch.randn((T, K + 3), device=DEV).bfloat16()  # rows off the 16-byte grid
    xo[:, 1 : K + 1] = c.x
    c.check(lora_add(xo[:, 1 : K + 1], c.base, c.proj, c.plan))


@pytest.mark.parametrize("ranks", [[16, 24], [16, 8]])
def test_nan_of_one_token_stays_with_it(ranks: list[int]) -> None:
    from microserve_b200.lora import lora_add

    c = Case([0, 1, 0, -1, 1, 0], ranks, 256, [128], "bfloat16")
    clean = lora_add(c.x, c.base, c.proj, c.plan)
    c.x[2] = float("nan")
    c.x[3] = float("inf")  # no adapter: not read
    got = lora_add(c.x, c.base, c.proj, c.plan)
    assert torch.isnan(got[2]).all()
    keep = torch.tensor([0, 1, 3, 4, 5], device=DEV)
    assert torch.equal(got[keep], clean[keep])


def test_bad_plans_and_adapters_are_skipped() -> None:
    """Wrong ids on the device set the error word; the tokens concerned are left alone."""
    from microserve_b200 import _lib
    from microserve_b200.lora import lora_add

    def run(c: Case) -> torch.Tensor:
        out = torch.full((c.T, c.N), 4.0, device=DEV)
        lora_add(c.x, c.base, c.proj, c.plan, out=out)
        assert _lib.device_error() != 0
        return out

    kw = dict(of=[0] * 3 + [1] * 4, ranks=[16, 8], K=64, slices=[64], dtype="bfloat16")
    for dtype in ("bfloat16", "float32"):
        kw["dtype"] = dtype
        good = lora_add(*(lambda c: (c.x, c.base, c.proj, c.plan))(Case(**kw)))
        for col, val in ((0, -1), (0, 5), (1, 65), (1, -2), (2, 2)):
            c = Case(**kw)
            c.plan.tiles[0, col] = val
            out = run(c)
            assert (out[:3] == 4.0).all() and torch.equal(out[3:], good[3:])
        for name, val in (("ranks", 17), ("ranks", -1), ("offsets", 10), ("offsets", -1)):
            c = Case(**kw)
            getattr(c.proj, name)[0] = val
            out = run(c)
            assert (out[:3] == 4.0).all() and torch.equal(out[3:], good[3:])
        for val in (-1, 7):
            c = Case(**kw)
            c.plan.order[1] = val
            out = run(c)
            assert (out[1] == 4.0).all()
            keep = torch.tensor([0, 2, 3, 4, 5, 6], device=DEV)
            assert torch.equal(out[keep], good[keep])


@pytest.mark.parametrize("bad", [(-64, 64, 0, 0), (-1, 64, 0, 0), (0, 65, 0, 0), (0, 64, 3, 0)])
def test_a_bad_tile_before_a_prompt_costs_only_itself(bad: tuple[int, ...]) -> None:
    from microserve_b200 import _lib
    from microserve_b200.lora import LoraPlan, lora_add

    c = Case([0] * 256, [24], 128, [256], "bfloat16")
    good = lora_add(c.x, c.base, c.proj, c.plan)
    tiles = torch.cat([torch.tensor([bad], dtype=torch.int32, device=DEV), c.plan.tiles])
    got = lora_add(c.x, c.base, c.proj, LoraPlan(c.plan.order, tiles))
    assert _lib.device_error() != 0
    assert torch.equal(got, good)


@pytest.mark.parametrize("tokens,ranks,K,dtype", [
    (90, [16, 8, 32, 16], 1024, "bfloat16"),
    (9, [16, 8, 3, 16], 1024, "bfloat16"),  # one launch
    (40, [16, 8, 3, 16], 200, "float32"),
    (40, [16, 8, 3, 16], 1024, "float32"),
    (4500, [16, 8], 520, "bfloat16"),
])
def test_two_streams_and_replayed_graphs(tokens: int, ranks: list[int], K: int, dtype: str) -> None:
    """Each call has its own scratch: calls on two streams, and two captured graphs, do not mix."""
    from microserve_b200.lora import lora_add

    cs = [Case(mixed(tokens, len(ranks), s), ranks, K, [512], dtype, seed=s) for s in range(2)]
    want = [lora_add(c.x, c.base, c.proj, c.plan) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    for _ in range(20):
        outs = []
        for c, s in zip(cs, streams):
            with torch.cuda.stream(s):
                outs.append(lora_add(c.x, c.base, c.proj, c.plan))
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))
    graphs, outs = [], [torch.empty_like(w) for w in want]
    for c, o in zip(cs, outs):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            lora_add(c.x, c.base, c.proj, c.plan, out=o)
        graphs.append(graph)
    for k in (0, 1, 1, 0):
        outs[k].zero_()
        cs[k].x.copy_(-cs[k].x)
        graphs[k].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[k], lora_add(cs[k].x, cs[k].base, cs[k].proj, cs[k].plan))


def test_refusals() -> None:
    from dataclasses import replace

    from microserve_b200.lora import LoraPlan, lora_add

    c = Case([0, 1, -1], [16, 8], 64, [64, 64], "bfloat16", interleaved=True)

    def refused(x=c.x, base=c.base, proj=c.proj, plan=c.plan, **kw) -> None:
        with pytest.raises(ValueError):
            lora_add(x, base, proj, plan, **kw)

    refused(x=c.x.half())
    refused(x=c.x.float())  # adapters in another type
    refused(x=c.x[:2])
    refused(x=c.x.t().contiguous().t())
    refused(base=c.base.bfloat16())
    refused(base=c.base[:, :64])
    refused(proj=replace(c.proj, slices=[64, 63]))
    refused(proj=replace(c.proj, slices=[96, 32]))
    refused(proj=replace(c.proj, slices=[]))
    refused(proj=replace(c.proj, max_rank=257))
    refused(proj=replace(c.proj, a=c.a[:-1]))
    refused(proj=replace(c.proj, b=c.b[:, :64]))
    refused(proj=replace(c.proj, ranks=c.proj.ranks.long()))
    refused(proj=replace(c.proj, scales=c.proj.scales.cpu()))
    refused(plan=LoraPlan(c.plan.order[:2], c.plan.tiles))
    refused(plan=LoraPlan(c.plan.order, c.plan.tiles[:, :3]))
    refused(proj=replace(c.proj, interleaved=False), swiglu=True)
    refused(out=torch.empty((3, 64), device=DEV))
    refused(out=torch.empty((3, 128), device=DEV, dtype=torch.float16))
    refused(out=torch.empty((3, 128), device=DEV).t().contiguous().t())
    from microserve_b200._lib import MicroserveError

    with pytest.raises(MicroserveError, match="overlap"):
        buf = torch.zeros(3 * 128 + 2, device=DEV)
        lora_add(c.x, buf[:384].view(3, 128), c.proj, c.plan, out=buf[2:].view(3, 128))
    with pytest.raises(MicroserveError):  # the SwiGLU cannot go back into the base
        lora_add(c.x, c.base, c.proj, c.plan, swiglu=True, out=c.base[:, :64])

"""Host side of the logit controls and the adapters (no GPU): plans, packed structures, what is
refused before any launch."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch


def test_plan_covers_every_token_once_in_tiles_of_one_adapter() -> None:
    from microserve_b200.lora import TILE, LoraPlan

    rng = np.random.default_rng(0)
    for n, k in ((0, 1), (1, 1), (64, 1), (65, 1), (500, 3), (1000, 200)):
        of = rng.integers(-1, k, n)
        order, tiles = LoraPlan.host_arrays(of)
        assert order.dtype == tiles.dtype == np.int32 and tiles.shape[1] == 4
        assert sorted(order.tolist()) == list(range(n))
        seen = np.zeros(n, int)
        for start, count, adapter, _ in tiles:
            assert 1 <= count <= TILE
            seen[start : start + count] += 1
            assert (of[order[start : start + count]] == adapter).all()
        assert (seen == 1).all()
        # no more tiles than the tokens of each adapter need
        _, sizes = np.unique(of, return_counts=True)
        assert len(tiles) == (-(-sizes // TILE)).sum()
    order, tiles = LoraPlan.host_arrays(np.array([-7, 2, -1]))  # any negative id: none
    assert set(tiles[:, 2].tolist()) == {-1, 2}


def test_masks_are_packed_by_token() -> None:
    from microserve_b200.logits import pack_masks

    for v in (1, 31, 32, 33, 100):
        a = np.random.default_rng(v).random((3, v)) < 0.5
        w = pack_masks(a).view(np.uint32)
        assert w.shape == (3, -(-v // 32))
        for t in range(v):
            assert np.array_equal((w[:, t // 32] >> np.uint32(t % 32)) & 1, a[:, t])


def test_packed_structures_equal_the_ctypes_ones() -> None:
    from microserve_b200 import _lib, logits, lora

    vals = tuple(range(1, 17))
    assert logits._PACK_CONTROLS(*vals) == bytes(_lib.MsLogitControls(*vals))
    assert lora._PACK_ADAPTERS(1, 2, 3, 0, 4, 5, 6) == bytes(_lib.MsLoraAdapters(1, 2, 3, 0, 4, 5, 6))
    assert lora._PACK_PLAN(1, 2, 3, 4) == bytes(_lib.MsLoraPlan(1, 2, 3, 4))


def test_c_entry_points_refuse_before_launching() -> None:
    """Bad sizes and missing arrays return a status without a GPU."""
    from microserve_b200 import _lib

    lib = _lib.load()
    bad = _lib.MS_ERR_INVALID

    def controls(**kw) -> ctypes.c_void_p:
        s = _lib.MsLogitControls(**kw)
        controls.keep = s
        return ctypes.byref(s)

    def apply(c, n=1, r=1, v=8, stride=8, out=1 << 20, ld=8, src=1 << 12) -> int:
        return lib.ms_apply_logit_controls(src, stride, out, ld, n, r, v, c, None)

    assert apply(None) == bad
    assert apply(controls(), n=-1) == bad and apply(controls(), r=0) == bad
    assert apply(controls(), v=0) == bad and apply(controls(), stride=7) == bad
    assert apply(controls(), ld=7) == bad and apply(controls(), out=0) == bad
    assert apply(controls(), out=(1 << 12) + 16) == bad  # overlaps
    assert apply(controls(), out=1 << 12, ld=16) == bad  # in place with two strides
    assert apply(controls(slots=1)) == bad
    assert apply(controls(proposals=1, n_proposals=65)) == bad
    assert apply(controls(proposals=1, n_proposals=2, first_proposal=1), n=1, r=3) == bad
    assert apply(controls(first_proposal=-1)) == bad
    assert apply(controls(bias_start=1, n_bias=2)) == bad
    assert apply(controls(mask_rows=1)) == bad
    assert apply(controls(), n=0) == _lib.MS_OK
    assert lib.ms_token_counts_append(None, None, 4, 8, None, 2, None, None, 0, None, 0, 3, None,
                                      None) == bad
    assert lib.ms_token_counts_append(1, 1, 0, 8, 1, 2, 1, None, 0, None, 0, 3, None, None) == bad
    assert lib.ms_token_counts_reset(None, None, 4, 8, None, 2, None) == bad
    assert lib.ms_token_counts_reset(None, None, 4, 8, None, 0, None) == _lib.MS_OK

    def lora(K=64, N=64, ns=1, cols=(64,), inter=0, swiglu=0, ad=None, pl=None, dt=1, od=0, x=1 << 12,
             x_ld=64, base=1 << 16, base_ld=64, out=1 << 20, out_ld=64, ws=0, n_ws=0, a=1 << 12,
             b=1 << 12) -> int:
        ad = ad or _lib.MsLoraAdapters(1, 16, 16, 0, 1, 1, 1)
        pl = pl or _lib.MsLoraPlan(4, 1, 1, 16)
        c = (ctypes.c_int32 * len(cols))(*cols)
        return lib.ms_lora_add(x, x_ld, base, base_ld, out, out_ld, a, b, K, N, ns,
                               ctypes.addressof(c), inter, swiglu, ctypes.byref(ad),
                               ctypes.byref(pl), dt, od, ws, n_ws, None)

    assert lora(K=0) == bad and lora(N=0) == bad and lora(ns=5, cols=(1,) * 5) == bad
    assert lora(dt=7) == bad and lora(od=7) == bad and lora(ns=2, cols=(32, 31)) == bad
    assert lora(ns=2, cols=(64, 0)) == bad and lora(inter=1) == bad and lora(swiglu=1) == bad
    assert lora(ns=2, cols=(20, 20), N=40, inter=1) == bad
    assert lora(x=0) == bad and lora(x_ld=63) == bad and lora(base_ld=63) == bad
    assert lora(out_ld=63) == bad and lora(out=(1 << 16) + 32) == bad  # overlaps the base
    assert lora(out=1 << 16, od=1) == bad  # bf16 over the float32 base
    assert lora(x=(1 << 20) + 512) == bad and lora(x=(1 << 20) - 256) == bad  # x overlaps out
    assert lora(ws=1 << 24, n_ws=8, K=263, x_ld=263) == _lib.MS_ERR_WORKSPACE  # too small
    assert lora(a=0) == bad
    assert lora(ad=_lib.MsLoraAdapters(1, 16, 257, 0, 1, 1, 1)) == bad
    assert lora(ad=_lib.MsLoraAdapters(1, 16, 16, 0, 0, 1, 1)) == bad
    assert lora(pl=_lib.MsLoraPlan(4, 65536, 1, 16)) == bad
    assert lora(pl=_lib.MsLoraPlan(4, 1, 1, 4)) == bad  # tiles off 16 bytes
    assert lora(pl=_lib.MsLoraPlan(0, 0, 0, 0)) == _lib.MS_OK


def test_host_tensors_are_refused() -> None:
    from microserve_b200.logits import LogitControls, apply_logit_controls
    from microserve_b200.lora import LoraPlan, LoraProjection, lora_add

    with pytest.raises(RuntimeError, match="CUDA"):
        apply_logit_controls(torch.zeros((1, 8)), LogitControls())
    z = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="CUDA"):
        lora_add(torch.zeros((1, 8)), torch.zeros((1, 8)),
                 LoraProjection(torch.zeros((1, 8)), torch.zeros((1, 8)), z, z, z.float(), 1, [8]),
                 LoraPlan(z, z.view(1, 1)))


def test_sampling_settings_are_checked() -> None:
    from microserve_b200.config import SamplingConfig
    from microserve_b200.logits import RequestControls
    from microserve_b200.sampling import validate

    validate(SamplingConfig(repetition_penalty=0.5, presence_penalty=-2.0, frequency_penalty=3.0))
    for kw in (dict(repetition_penalty=0.0), dict(repetition_penalty=float("nan")),
               dict(repetition_penalty=float("inf")), dict(presence_penalty=float("inf")),
               dict(frequency_penalty=float("nan"))):
        with pytest.raises(ValueError):
            validate(SamplingConfig(**kw))
    rc = RequestControls(10, torch.device("cpu"))
    rc.check(SamplingConfig())
    rc.check(SamplingConfig(logit_bias={0: 1.0, 9: -float("inf")}))
    for bias in ({10: 1.0}, {-1: 1.0}, {1: float("nan")}, {1: float("inf")}, {1.5: 0.0}):
        with pytest.raises(ValueError):
            rc.check(SamplingConfig(logit_bias=bias))
    assert not SamplingConfig().controlled and SamplingConfig(logit_bias={1: 0.5}).controlled
    assert not SamplingConfig(logit_bias={}).controlled


def test_adapter_pools_on_the_host() -> None:
    """Loading, growing, unloading and reusing the rank axis; weights land in their rows."""
    from types import SimpleNamespace

    from microserve_b200.config import ModelConfig
    from microserve_b200.lora import LoraAdapters

    cfg = ModelConfig(vocab_size=65, n_layers=2, d_model=64, n_heads=4, n_kv_heads=2, d_ff=96)
    model = SimpleNamespace(cfg=cfg, device=torch.device("cpu"), dtype=torch.float32, adapters=None)
    ads = LoraAdapters(model, rank_capacity=4)
    assert model.adapters is ads
    shape = {"attn.q_proj": (64, 64), "attn.v_proj": (64, 32), "ffn.up_proj": (64, 96),
             "ffn.down_proj": (96, 64)}

    def state(rank: int, parts, seed: int) -> dict[str, torch.Tensor]:
        g = torch.Generator().manual_seed(seed)
        out = {}
        for i in range(2):
            for p in parts:
                k, n = shape[p]
                out[f"blocks.{i}.{p}.lora_A.weight"] = torch.randn(rank, k, generator=g)
                out[f"blocks.{i}.{p}.lora_B.weight"] = torch.randn(n, rank, generator=g)
        return out

    x, y = state(3, ["attn.q_proj", "ffn.up_proj"], 1), state(6, ["attn.v_proj", "ffn.down_proj"], 2)
    ads.load("x", x, alpha=6.0)
    ads.load("y", y)
    assert ads._offset == [0, 3] and ads._rank == [3, 6] and ads._scale == [2.0, 1.0]
    c = ads.c_struct()
    assert c.adapters.total_rank == ads._capacity >= 9 and c.adapters.max_rank == 6
    assert bool(c.a_qkv) and bool(c.a_gate_up) and bool(c.a_down) and not bool(c.a_o)
    for layer in range(2):
        p = ads.projection("qkv", layer)
        q = x[f"blocks.{layer}.attn.q_proj.lora_A.weight"]
        assert torch.equal(p.a[:3], q) and (p.a[3:9] == 0).all()  # q's rows, then k's and v's
        v = y[f"blocks.{layer}.attn.v_proj.lora_A.weight"]
        assert torch.equal(p.a[9 + 12 : 9 + 18], v)
        assert torch.equal(p.b[3:9, 96:], y[f"blocks.{layer}.attn.v_proj.lora_B.weight"].t())
        assert (p.b[3:9, :96] == 0).all() and (p.b[:3, 64:] == 0).all()
        gu = ads.projection("gate_up", layer)
        assert gu.interleaved
        up = gu.b[:3].view(3, -1, 2, 8)[:, :, 1].reshape(3, -1)
        assert torch.equal(up, x[f"blocks.{layer}.ffn.up_proj.lora_B.weight"].t())
        assert (gu.b[:3].view(3, -1, 2, 8)[:, :, 0] == 0).all()
    ads.acquire("x")
    with pytest.raises(ValueError, match="held"):
        ads.unload("x")
    ads.release("x")
    ads.unload("x")
    assert ads.names == ["y"] and ads.id_of(None) == -1
    with pytest.raises(ValueError):
        ads.id_of("x")
    ads.load("z", state(2, ["attn.q_proj"], 3))  # takes x's place and id
    assert ads.id_of("z") == 0 and ads._offset[0] == 0
    assert (ads.projection("gate_up", 0).b[:2] == 0).all()  # nothing of x is left in z's rows
    assert ads.ids_of_tokens(["z", None, "y"], [2, 1, 3]).tolist() == [0, 0, -1, 1, 1, 1]


def test_a_load_that_fails_leaves_the_adapters_usable(monkeypatch: pytest.MonkeyPatch) -> None:
    """Growing the rank axis replaces the pools; their addresses are not kept past it."""
    from types import SimpleNamespace

    from microserve_b200.config import ModelConfig
    from microserve_b200.lora import LoraAdapters

    cfg = ModelConfig(vocab_size=65, n_layers=1, d_model=64, n_heads=4, d_ff=96)
    model = SimpleNamespace(cfg=cfg, device=torch.device("cpu"), dtype=torch.float32, adapters=None)
    ads = LoraAdapters(model, rank_capacity=2)
    key = "blocks.0.attn.o_proj.lora_"
    state = lambda r: {key + "A.weight": torch.ones(r, 64), key + "B.weight": torch.ones(64, r)}  # noqa: E731
    ads.load("x", state(2))
    assert ads.c_struct().a_o[0] == ads._a["o"][0].data_ptr()
    grown = ads._reserve

    def reserve(rank: int) -> int:
        grown(rank)
        raise RuntimeError("out of memory")

    monkeypatch.setattr(ads, "_reserve", reserve)
    with pytest.raises(RuntimeError):
        ads.load("y", state(5))
    assert ads.names == ["x"]
    assert ads.c_struct().a_o[0] == ads._a["o"][0].data_ptr()
    assert (ads.projection("o", 0).a[:2] == 1).all()
    ads.acquire("x")
    with pytest.raises(ValueError, match="held"):
        LoraAdapters(model)
    assert model.adapters is ads

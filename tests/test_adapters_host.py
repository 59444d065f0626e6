"""The adapters' pools on the host (no GPU)."""

from __future__ import annotations

from types import SimpleNamespace

import pytest
import torch

KEY = "blocks.0.attn.o_proj.lora_"


def adapters(capacity: int = 2):
    from microserve_b200.config import ModelConfig
    from microserve_b200.lora import LoraAdapters

    cfg = ModelConfig(vocab_size=65, n_layers=1, d_model=64, n_heads=4, d_ff=96)
    model = SimpleNamespace(cfg=cfg, device=torch.device("cpu"), dtype=torch.float32, adapters=None)
    return LoraAdapters(model, rank_capacity=capacity)


def state(rank: int, value: float) -> dict[str, torch.Tensor]:
    return {KEY + "A.weight": torch.full((rank, 64), value), KEY + "B.weight": torch.full((64, rank), -value)}


@pytest.mark.parametrize("fails_at", [1, 2, 3, 4])
def test_a_growth_that_runs_out_of_memory_changes_nothing(fails_at: int, monkeypatch: pytest.MonkeyPatch
                                                          ) -> None:
    ads = adapters()
    ads.load("x", state(2, 1.0))
    pools, calls = ads._pools, []

    def failing(name: str, capacity: int):
        calls.append(name)
        if len(calls) == fails_at:
            raise RuntimeError("out of memory")
        return pools(name, capacity)

    before = {n: (ads._a[n][0], ads._b[n][0]) for n in ads._a}
    monkeypatch.setattr(ads, "_pools", failing)
    with pytest.raises(RuntimeError, match="memory"):
        ads.load("y", state(5, 2.0))
    monkeypatch.undo()
    assert ads.names == ["x"] and ads._capacity == 2
    assert all(ads._a[n][0] is a and ads._b[n][0] is b for n, (a, b) in before.items())
    assert ads.c_struct().a_o[0] == ads._a["o"][0].data_ptr()
    # and the loads after it work
    for name, rank, value in (("y", 5, 2.0), ("z", 4, 3.0), ("w", 1, 4.0)):
        ads.load(name, state(rank, value))
    p = ads.projection("o", 0)
    for name, rank, value in (("x", 2, 1.0), ("y", 5, 2.0), ("z", 4, 3.0), ("w", 1, 4.0)):
        o = ads._offset[ads.id_of(name)]
        assert (p.a[o : o + rank] == value).all() and (p.b[o : o + rank] == -value).all()
    assert all(ads._b[n][0].shape[0] == ads._capacity for n in ads._b)
    assert ads.c_struct().adapters.total_rank == ads._capacity


def test_a_forward_with_adapters_needs_their_plan() -> None:
    """Adapters without a plan, or with a bad one, are refused before anything is launched (the
    workspace is missing as well, so that nothing could be)."""
    import ctypes

    from microserve_b200 import _lib

    one = (ctypes.c_void_p * 1)(1 << 12)
    ptrs = ctypes.cast(one, ctypes.POINTER(ctypes.c_void_p))
    model = _lib.MsModel(65, 64, 1, 4, 4, 16, 96, 128, _lib.DTYPE_F32, 1e-5, 1 << 12, 1 << 12, 1 << 12,
                         1 << 12, *[ptrs] * 6)
    cache = _lib.MsKVCache(1, 8, 8, 4, 16, _lib.DTYPE_F32, ptrs, ptrs)
    batch = _lib.MsBatch(4, 1, 8, 4, 4, 0, *[1 << 12] * 6)
    lora = _lib.MsLoraModel(_lib.MsLoraAdapters(1, 16, 16, 0, 1 << 12, 1 << 12, 1 << 12))
    null = ctypes.POINTER(_lib.MsLoraPlan)()

    def refused(plan, match: str, adapters=lora) -> None:
        with pytest.raises(_lib.MicroserveError, match=match):
            _lib.call("ms_forward_lora", ctypes.byref(model), ctypes.byref(cache), ctypes.byref(batch),
                      ctypes.byref(adapters), plan, None, 0, 1 << 12, 0, None, 0, None)

    refused(null, "without a plan")
    refused(ctypes.byref(_lib.MsLoraPlan(4, -1, 1 << 12, 1 << 12)), "plan sizes")
    refused(ctypes.byref(_lib.MsLoraPlan(4, 1, 1 << 12, 1 << 12)), "adapter sizes",
            _lib.MsLoraModel(_lib.MsLoraAdapters(1, 16, -1, 0, 1 << 12, 1 << 12, 1 << 12)))
    refused(ctypes.byref(_lib.MsLoraPlan(4, 1, 1 << 12, 1 << 12)), "workspace")  # nothing else is wrong
    refused(ctypes.byref(_lib.MsLoraPlan(4, 0, None, None)), "workspace")  # ms_forward

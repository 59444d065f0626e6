"""Low-rank adapters of many requests at once beside the shared projections.

A request may name an adapter; every projection of the decoder then adds
``scale * B (A x)`` for its tokens, next to the shared product, in one pair of
launches for the whole batch (``ms_lora_add``), whatever adapters its tokens
use.  The reference has no adapters.

Layout.  Adapter ``i`` has rank ``ranks[i]`` and occupies ``offsets[i] ..
offsets[i] + ranks[i]`` of the adapters' common rank axis of length R:
``a`` is ``(n_slices * R, K)``, adapter ``i``'s rows from ``n_slices *
offsets[i]``, slice by slice; ``b`` is ``(R, N)``, transposed, so a column range is
read in whole lines.  ``n_slices`` is the number of projections fused into one
(q, k, v: 3; gate, up: 2).
"""

from __future__ import annotations

import ctypes
from collections.abc import Sequence
from dataclasses import dataclass

import numpy as np
import torch

from . import _lib

TILE = 64  # tokens of a plan's tile (MS_LORA_TILE)
MAX_RANK = 256  # MS_LORA_MAX_RANK
_check = _lib.check_tensor
_CODES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


@dataclass
class LoraProjection:
    """One projection's adapters: ``a`` (n_slices * R, K) and ``b`` (R, N) in the
    model's dtype; ``offsets``, ``ranks`` int32 and ``scales`` float32, one per
    adapter; ``max_rank`` bounds the ranks; ``slices`` are the column counts of the
    fused projections, or with ``interleaved`` two slices alternate every 8
    columns (the gate/up layout)."""

    a: torch.Tensor
    b: torch.Tensor
    offsets: torch.Tensor
    ranks: torch.Tensor
    scales: torch.Tensor
    max_rank: int
    slices: Sequence[int]
    interleaved: bool = False


@dataclass
class LoraPlan:
    """Which tokens of a batch use which adapter: ``order`` (T,) int32 lists the
    tokens grouped by adapter, ``tiles`` (n, 4) int32 are (first position in
    ``order``, count of at most 64, adapter or -1, 0)."""

    order: torch.Tensor
    tiles: torch.Tensor

    @staticmethod
    def host_arrays(adapter_of_token: np.ndarray) -> tuple[np.ndarray, np.ndarray]:
        """``order`` and ``tiles`` as int32 host arrays."""
        of = np.asarray(adapter_of_token, dtype=np.int64)
        order = np.argsort(of, kind="stable")
        ids, first = np.unique(of[order], return_index=True)
        lens = np.diff(np.append(first, of.size))
        n = -(-lens // TILE)
        within = np.arange(int(n.sum())) - np.repeat(np.cumsum(n) - n, n)
        start = np.repeat(first, n) + TILE * within
        count = np.minimum(TILE, np.repeat(first + lens, n) - start)
        tiles = np.stack([start, count, np.maximum(np.repeat(ids, n), -1), np.zeros_like(start)], 1)
        return order.astype(np.int32), tiles.astype(np.int32)

    @classmethod
    def build(cls, adapter_of_token: Sequence[int] | np.ndarray,
              device: str | torch.device = "cuda") -> LoraPlan:
        """The plan of a batch from each token's adapter (negative: none)."""
        order, tiles = cls.host_arrays(np.asarray(adapter_of_token))
        dev = torch.device(device)
        return cls(torch.from_numpy(order).to(dev), torch.from_numpy(tiles).to(dev))


def lora_add(
    x: torch.Tensor,
    base: torch.Tensor,
    proj: LoraProjection,
    plan: LoraPlan,
    *,
    swiglu: bool = False,
    out: torch.Tensor | None = None,
    out_dtype: torch.dtype = torch.float32,
) -> torch.Tensor:
    """``base + scale * B (A x)`` for every token, with its own adapter.

    ``x`` (T, K) in the model's dtype, ``base`` (T, N) float32, both with
    contiguous rows.  ``swiglu`` returns ``silu(gate) * up`` (T, N/2) of an
    interleaved projection instead.  ``out`` (float32 or bfloat16) defaults to a
    new tensor of ``out_dtype``; it may be ``base`` itself (no SwiGLU): tokens
    without an adapter are then not touched."""
    dev = _lib.cuda_index(x)
    T, K = x.shape
    if base.dim() != 2 or base.shape[0] != T or base.dtype is not torch.float32 \
            or base.get_device() != dev:
        raise ValueError(f"base must be a float32 ({T}, N) tensor on cuda:{dev}")
    N = base.shape[1]
    x_ld, x_inner = x.stride()
    base_ld, base_inner = base.stride()
    if (T > 1 and (x_ld < K or base_ld < N)) or x_inner != 1 or base_inner != 1:
        raise ValueError("x and base need contiguous, non-overlapping rows")
    dtype = x.dtype
    if dtype not in _CODES:
        raise ValueError(f"x must be float32 or bfloat16, got {dtype}")
    slices = proj.slices
    ns = len(slices)
    if not 1 <= ns <= 4 or sum(slices) != N or min(slices) < 1:
        raise ValueError(f"slices {list(slices)} do not make up {N} columns")
    if proj.interleaved and (ns != 2 or N % 16 or slices[0] != slices[1]):
        raise ValueError("interleaved columns are two equal slices alternating every 8 columns")
    if swiglu and not proj.interleaved:
        raise ValueError("SwiGLU needs interleaved gate/up columns")
    if not 0 <= proj.max_rank <= MAX_RANK:
        raise ValueError(f"max_rank {proj.max_rank} is not in 0..{MAX_RANK}")
    R = proj.b.shape[0]
    pa = _check(proj.a, "a", dtype, dev, (ns * R, K))
    pb = _check(proj.b, "b", dtype, dev, (R, N))
    n = proj.ranks.numel()
    i32 = torch.int32
    ad = _lib.MsLoraAdapters(n, R, proj.max_rank, 0, _check(proj.offsets, "offsets", i32, dev, (n,)),
                             _check(proj.ranks, "ranks", i32, dev, (n,)),
                             _check(proj.scales, "scales", torch.float32, dev, (n,)))
    n_tiles = plan.tiles.shape[0]
    pl = _lib.MsLoraPlan(T, n_tiles, _check(plan.order, "order", i32, dev, (T,)),
                         _check(plan.tiles, "tiles", i32, dev, (n_tiles, 4)))
    width = N // 2 if swiglu else N
    if out is None:
        out = torch.empty((T, width), dtype=out_dtype, device=x.device)
    elif out.shape != (T, width) or out.get_device() != dev or out.stride(1) != 1 \
            or (T > 1 and out.stride(0) < width):
        raise ValueError(f"out must be a ({T}, {width}) tensor on cuda:{dev} with contiguous rows")
    if out.dtype not in _CODES:
        raise ValueError(f"out must be float32 or bfloat16, got {out.dtype}")
    if T == 0:
        return out
    # ms_lora_workspace_size: s as up to three bf16 terms of the padded rank
    need = T * ns * ((proj.max_rank + 15) // 16 * 16) * 6
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=x.device)
    cols = (ctypes.c_int32 * ns)(*slices)
    _lib.launch_on(dev, "ms_lora_add", x.data_ptr(), max(x_ld, K), base.data_ptr(),
                   max(base_ld, N), out.data_ptr(), max(out.stride(0), width), pa, pb, K, N, ns,
                   ctypes.addressof(cols), int(proj.interleaved), int(swiglu), ctypes.byref(ad),
                   ctypes.byref(pl), _CODES[dtype], _CODES[out.dtype], ws.data_ptr(), ws.numel())
    return out

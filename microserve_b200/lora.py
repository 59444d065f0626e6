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
import struct
from collections.abc import Iterable, Mapping, Sequence
from dataclasses import dataclass
from typing import TYPE_CHECKING

import numpy as np
import torch

from . import _lib

if TYPE_CHECKING:
    from .model import Transformer

TILE = 64  # tokens of a plan's tile (MS_LORA_TILE)
MAX_RANK = 256  # MS_LORA_MAX_RANK
_check = _lib.check_tensor
# the C structures as bytes (a third of the time ctypes structures take to fill)
_PACK_ADAPTERS = struct.Struct("=iiiiQQQ").pack
_PACK_PLAN = struct.Struct("=iiQQ").pack
_PACK_COLUMNS = [struct.Struct(f"={k}i").pack for k in range(5)]
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

    def c_struct(self, n_tokens: int, device: torch.device) -> _lib.MsLoraPlan:
        index = torch.cuda.current_device() if device.index is None else device.index
        n = self.tiles.shape[0]
        return _lib.MsLoraPlan(
            n_tokens, n, _check(self.order, "order", torch.int32, index, (n_tokens,)),
            _check(self.tiles, "tiles", torch.int32, index, (n, 4)))


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
    without an adapter are then not touched.  Rows of tokens that no tile of
    ``plan`` lists (``LoraPlan.build`` lists all) are not written."""
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
    n_tiles = plan.tiles.shape[0]
    ad = _PACK_ADAPTERS(n, R, proj.max_rank, 0, _check(proj.offsets, "offsets", i32, dev, (n,)),
                        _check(proj.ranks, "ranks", i32, dev, (n,)),
                        _check(proj.scales, "scales", torch.float32, dev, (n,)))
    pl = _PACK_PLAN(T, n_tiles, _check(plan.order, "order", i32, dev, (T,)),
                    _check(plan.tiles, "tiles", i32, dev, (n_tiles, 4)))
    width = N // 2 if swiglu else N
    if out is None:
        # (empty_like costs half of what empty does)
        out = torch.empty_like(base) if out_dtype is torch.float32 and width == N \
            and base.is_contiguous() else torch.empty((T, width), dtype=out_dtype, device=x.device)
    elif out.shape != (T, width) or out.get_device() != dev or out.stride(1) != 1 \
            or (T > 1 and out.stride(0) < width):
        raise ValueError(f"out must be a ({T}, {width}) tensor on cuda:{dev} with contiguous rows")
    if out.dtype not in _CODES:
        raise ValueError(f"out must be float32 or bfloat16, got {out.dtype}")
    if T == 0:
        return out
    args = (x.data_ptr(), max(x_ld, K), base.data_ptr(), max(base_ld, N), out.data_ptr(),
            max(out.stride(0), width), pa, pb, K, N, ns, _PACK_COLUMNS[ns](*slices),
            int(proj.interleaved), int(swiglu), ad, pl, _CODES[dtype], _CODES[out.dtype])
    # little work usually takes one launch without scratch (one_launch, any_fused)
    if (T <= 32 and T <= 8 * n_tiles and N <= 4096 and proj.max_rank <= 16 and ns == 1) \
            if dtype is torch.bfloat16 else (K <= 256 and ns * proj.max_rank <= 256):
        rc = _lib.launch_status(dev, "ms_lora_add", *args, None, 0)
        if rc != _lib.MS_ERR_WORKSPACE:
            if rc:
                _lib.check("ms_lora_add", rc)
            return out
    # ms_lora_workspace_size: s as up to three bf16 terms of the padded rank
    need = T * ns * ((proj.max_rank + 15) // 16 * 16) * 6
    ws = torch.empty(max(need, 16), dtype=torch.uint8, device=x.device)
    _lib.launch_on(dev, "ms_lora_add", *args, ws.data_ptr(), ws.numel())
    return out


# fused projection -> (its parts' state-dict names, interleaved)
_PROJECTIONS: dict[str, tuple[tuple[str, ...], bool]] = {
    "qkv": (("attn.q_proj", "attn.k_proj", "attn.v_proj"), False),
    "o": (("attn.o_proj",), False),
    "gate_up": (("ffn.gate_proj", "ffn.up_proj"), True),
    "down": (("ffn.down_proj",), False),
}


class LoraAdapters:
    """The adapters loaded beside a :class:`Transformer`, by name.

    ``load`` takes a state dict with, for any of the model's projections,
    ``blocks.{i}.attn.q_proj.lora_A.weight`` (rank, in) and ``...lora_B.weight``
    (out, rank), all of one rank; projections it does not name get nothing.
    Adapters share one rank axis per projection, grown by doubling; ``unload``
    frees an adapter's part of it and is refused while requests hold the
    adapter (``acquire`` / ``release``, kept by the engine).  Loading writes the
    weights on the current stream: call it from the stream that runs the model.
    """

    def __init__(self, model: Transformer, rank_capacity: int = 64) -> None:
        if rank_capacity < 1:
            raise ValueError("rank_capacity must be at least 1")
        if model.adapters is not None and any(model.adapters._users.values()):
            raise ValueError("the model's adapters are held by requests")
        self.cfg, self.device, self.dtype = model.cfg, model.device, model.dtype
        c = model.cfg
        d, ff = c.d_model, c.ffn_hidden
        q, kv = c.n_heads * c.d_head, c.kv_heads * c.d_head
        # (inputs, column counts of the fused parts)
        self._shape = {"qkv": (d, (q, kv, kv)), "o": (q, (d,)), "gate_up": (d, (ff, ff)),
                       "down": (ff, (d,))}
        self._capacity = rank_capacity
        self._a: dict[str, list[torch.Tensor]] = {}
        self._b: dict[str, list[torch.Tensor]] = {}
        for name in self._shape:
            self._a[name], self._b[name] = self._pools(name, rank_capacity)
        self._ids: dict[str, int] = {}
        self._offset: list[int] = []  # per id; rank 0: a free id
        self._rank: list[int] = []
        self._scale: list[float] = []
        self._users: dict[str, int] = {}
        self._uses: list[set[str]] = []  # the projections each id changes
        self._c: _lib.MsLoraModel | None = None
        model.adapters = self

    def _pools(self, name: str, capacity: int) -> tuple[list[torch.Tensor], list[torch.Tensor]]:
        k, cols = self._shape[name]
        z = lambda rows, width: torch.zeros((rows, width), dtype=self.dtype,  # noqa: E731
                                            device=self.device)
        n = range(self.cfg.n_layers)
        return ([z(len(cols) * capacity, k) for _ in n], [z(capacity, sum(cols)) for _ in n])

    # -- loading ----------------------------------------------------------------
    @property
    def names(self) -> list[str]:
        return list(self._ids)

    def __contains__(self, name: object) -> bool:
        return name in self._ids

    def _reserve(self, rank: int) -> int:
        """The first gap of ``rank`` rows in the rank axis, growing it if there is none."""
        used = sorted((o, r) for o, r in zip(self._offset, self._rank) if r)
        at = 0
        for o, r in used:
            if o - at >= rank:
                return at
            at = o + r
        if at + rank > self._capacity:
            capacity = max(2 * self._capacity, at + rank)
            # all of them before any is replaced: memory may run out in between
            grown = {name: self._pools(name, capacity) for name in self._shape}
            for name, (a, b) in grown.items():
                ns = len(self._shape[name][1])
                for pool, new, per in ((self._a[name], a, ns), (self._b[name], b, 1)):
                    for old, fresh in zip(pool, new):
                        fresh[: per * self._capacity].copy_(old)
            self._c = None  # it holds the old pools' addresses
            for name, (a, b) in grown.items():
                self._a[name], self._b[name] = a, b
            self._capacity = capacity
        return at

    def load(self, name: str, state: Mapping[str, torch.Tensor], alpha: float | None = None) -> int:
        """Add adapter ``name``; its part is scaled by ``alpha / rank`` (1 without ``alpha``).
        Returns its id.  Nothing changes when the state dict is refused."""
        if name in self._ids:
            raise ValueError(f"adapter {name!r} is already loaded")
        parts: dict[tuple[int, str], tuple[torch.Tensor, torch.Tensor]] = {}
        left, rank = set(state), None
        for i in range(self.cfg.n_layers):
            for proj, (names, _) in _PROJECTIONS.items():
                k, cols = self._shape[proj]
                for part, n in zip(names, cols):
                    key = f"blocks.{i}.{part}.lora_"
                    ka, kb = key + "A.weight", key + "B.weight"
                    if ka not in state and kb not in state:
                        continue
                    if ka not in state or kb not in state:
                        raise ValueError(f"adapter {name!r}: {key}A and {key}B go together")
                    a, b = (torch.as_tensor(state[x]) for x in (ka, kb))
                    r = a.shape[0] if a.dim() == 2 else 0
                    if rank is None:
                        rank = r
                    if a.shape != (r, k) or b.shape != (n, r) or r != rank:
                        raise ValueError(f"adapter {name!r}: {key}A {tuple(a.shape)}, {key}B "
                                         f"{tuple(b.shape)} do not fit ({rank}, {k}), ({n}, {rank})")
                    parts[i, part] = (a, b)
                    left -= {ka, kb}
        if left:
            raise ValueError(f"adapter {name!r}: unknown weights {sorted(left)[:3]}")
        if rank is None or not 1 <= rank <= MAX_RANK:
            raise ValueError(f"adapter {name!r}: rank {rank} is not in 1..{MAX_RANK}")
        scale = 1.0 if alpha is None else float(alpha) / rank
        if not np.isfinite(scale):
            raise ValueError(f"adapter {name!r}: alpha {alpha}")
        at = self._reserve(rank)
        for i in range(self.cfg.n_layers):
            for proj, (names, interleaved) in _PROJECTIONS.items():
                k, cols = self._shape[proj]
                ns = len(cols)
                pa = self._a[proj][i][ns * at : ns * (at + rank)]
                pb = self._b[proj][i][at : at + rank]
                for j, part in enumerate(names):
                    col0 = sum(cols[:j])
                    dst = pb.view(rank, -1, ns, 8)[:, :, j] if interleaved else \
                        pb[:, col0 : col0 + cols[j]]
                    got = parts.get((i, part))
                    if got is None:
                        pa[j * rank : (j + 1) * rank].zero_()
                        dst.zero_()
                    else:
                        pa[j * rank : (j + 1) * rank].copy_(got[0])
                        dst.copy_(got[1].t().reshape(dst.shape))
        free = [i for i, r in enumerate(self._rank) if r == 0]
        if free:
            i = free[0]
        else:
            i = len(self._rank)
            self._offset.append(0)
            self._rank.append(0)
            self._scale.append(0.0)
            self._uses.append(set())
        self._uses[i] = {p for p, (names, _) in _PROJECTIONS.items()
                         if any((layer, n) in parts for layer in range(self.cfg.n_layers)
                                for n in names)}
        self._offset[i], self._rank[i], self._scale[i] = at, rank, scale
        self._ids[name] = i
        self._users[name] = 0
        self._c = None
        return i

    def unload(self, name: str) -> None:
        """Forget an adapter that no request holds."""
        if name not in self._ids:
            raise ValueError(f"no adapter {name!r}")
        if self._users[name]:
            raise ValueError(f"adapter {name!r} is held by {self._users[name]} requests")
        del self._users[name]
        self._rank[self._ids.pop(name)] = 0
        self._c = None

    def acquire(self, name: str) -> None:
        if name not in self._ids:
            raise ValueError(f"no adapter {name!r} is loaded")
        self._users[name] += 1

    def release(self, name: str) -> None:
        self._users[name] -= 1

    # -- use ----------------------------------------------------------------------
    def id_of(self, name: str | None) -> int:
        """The id of an adapter (-1 for None)."""
        if name is None:
            return -1
        if name not in self._ids:
            raise ValueError(f"no adapter {name!r} is loaded")
        return self._ids[name]

    def ids_of_tokens(self, names: Iterable[str | None], lens: Sequence[int] | np.ndarray
                      ) -> np.ndarray:
        """Each token's adapter id, for sequences of ``lens`` tokens."""
        ids = np.fromiter((self.id_of(n) for n in names), np.int64)
        return np.repeat(ids, lens)

    def plan(self, names: Iterable[str | None], lens: Sequence[int] | np.ndarray) -> LoraPlan:
        """The plan of a batch whose sequence ``i`` has ``lens[i]`` tokens and adapter ``names[i]``."""
        return LoraPlan.build(self.ids_of_tokens(names, lens), self.device)

    def projection(self, name: str, layer: int) -> LoraProjection:
        """One layer's ``"qkv"``, ``"o"``, ``"gate_up"`` or ``"down"`` for :func:`lora_add`."""
        self.c_struct()
        return LoraProjection(
            a=self._a[name][layer], b=self._b[name][layer], offsets=self._d_offsets,
            ranks=self._d_ranks, scales=self._d_scales, max_rank=max(self._rank, default=0),
            slices=self._shape[name][1], interleaved=_PROJECTIONS[name][1])

    def c_struct(self) -> _lib.MsLoraModel:
        if self._c is None:
            t = lambda v, d: torch.tensor(v, dtype=d).to(self.device)  # noqa: E731
            self._d_offsets, self._d_ranks = t(self._offset, torch.int32), t(self._rank, torch.int32)
            self._d_scales = t(self._scale, torch.float32)
            head = _lib.MsLoraAdapters(len(self._rank), self._capacity, max(self._rank, default=0), 0,
                                       self._d_offsets.data_ptr(), self._d_ranks.data_ptr(),
                                       self._d_scales.data_ptr())
            # a projection that no loaded adapter changes costs nothing
            used = set().union(*(u for u, r in zip(self._uses, self._rank) if r))
            self._arrays = [_lib.pointer_array(pool[name]) if name in used else None
                            for name in self._shape for pool in (self._a, self._b)]
            ptr = ctypes.POINTER(ctypes.c_void_p)
            cast = lambda x: ptr() if x is None else ctypes.cast(x, ptr)  # noqa: E731
            self._c = _lib.MsLoraModel(head, *map(cast, self._arrays))
        return self._c

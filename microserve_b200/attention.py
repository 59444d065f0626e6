"""Paged attention whose scores or visible keys are other than plain causal (``ms_paged_attention_form``).

A form may cap the scores by a tanh, let them fall with the distance (a slope per
head), limit them to a sliding window, let every token see a prefix of its
sequence, and lay a tree of drafted tokens behind each cached context.  The
reference has plain causal attention only (src/microserve/model.py:200-221), which
``Transformer.forward_paged`` keeps computing when it is given no form.
"""

from __future__ import annotations

import struct
from ctypes import addressof, c_void_p
from dataclasses import dataclass
from typing import TYPE_CHECKING

import torch

from . import _lib

if TYPE_CHECKING:
    from .model import PagedBatch

_check = _lib.check_tensor
# the C structures as bytes (a third of the time ctypes structures take to fill)
_PACK_CACHE = struct.Struct("=iiiiiiQQ").pack
_PACK_BATCH = struct.Struct("=iiiiiiQQQQQQ").pack
_PACK_FORM = struct.Struct("=ffiiQQQ").pack
_CODES = {torch.float32: _lib.DTYPE_F32, torch.bfloat16: _lib.DTYPE_BF16}


@dataclass
class AttentionForm:
    """Scores ``c - slopes[h] * |p_q - p_k|`` with ``c = softcap * tanh(s / softcap)`` and
    ``s = scale * q . k``, over the keys that a query sees.

    ``scale`` 0 stands for ``1 / sqrt(d_head)``, ``softcap`` 0 for no cap, ``window`` 0 for no
    window.  A query at position ``p_q`` sees key ``j`` of its sequence when ``j <
    prefix_lens[b]``, or when it is seen and ``p_q - p_k < window``: without ``tree_mask`` the keys
    ``p_k = j <= p_q``; with it every key before the pass's own tokens, and of those token
    ``i`` where bit ``i % 32`` of word ``i / 32`` of the query's row is set (``p_k`` is then
    that token's position: siblings share one).  ``slopes`` (n_heads,) float32, ``prefix_lens``
    (B,) int32, ``tree_mask`` (T, words) int32, from :func:`microserve_b200.tree.tree_masks`
    or any other bits.

    A query that sees nothing gives 0.  bfloat16 caches with heads of 64 or 128 round each weight to
    bfloat16 for the product with the values, and divide by the sum of the rounded ones; all other sums
    are float32."""

    softcap: float = 0.0
    slopes: torch.Tensor | None = None
    window: int = 0
    prefix_lens: torch.Tensor | None = None
    tree_mask: torch.Tensor | None = None
    scale: float = 0.0

    def fields(self, index: int, n_heads: int, batch: PagedBatch) -> tuple[float | int, ...]:
        """The C structure's values for a batch on CUDA device ``index``, checked."""
        # (not (a <= x < b): NaN is refused too)
        if not 0.0 <= self.softcap < 3.4e38 or not 0.0 <= self.scale < 3.4e38:
            raise ValueError("softcap and scale must be finite and not negative (0: none, the default)")
        if 0.0 < self.softcap < 1e-45 or 0.0 < self.scale < 1e-45:  # (would be 0 in float32)
            raise ValueError("softcap and scale must be 0 or within float32's range")
        if not 0 <= self.window < 1 << 31:
            raise ValueError("window must be 0 (none) or a number of tokens")
        slopes = prefix = mask = words = 0
        if self.slopes is not None:
            slopes = _check(self.slopes, "slopes", torch.float32, index, (n_heads,))
        if self.prefix_lens is not None:
            prefix = _check(self.prefix_lens, "prefix_lens", torch.int32, index, (batch.batch_size,))
        if self.tree_mask is not None:
            if self.tree_mask.dim() != 2 or 32 * self.tree_mask.shape[1] < batch.max_q:
                raise ValueError(f"tree_mask must have a bit for each of {batch.max_q} tokens")
            words = self.tree_mask.shape[1]
            mask = _check(self.tree_mask, "tree_mask", torch.int32, index, (batch.n_tokens, words))
            if batch.n_tokens == 0:
                mask = words = 0
        return self.scale, self.softcap, self.window, words, slopes, prefix, mask

    def c_struct(self, index: int, n_heads: int, batch: PagedBatch) -> _lib.MsAttentionForm:
        return _lib.MsAttentionForm(*self.fields(index, n_heads, batch))


def pack_batch(batch: PagedBatch, index: int, tokens: bool = False) -> bytes:
    """``ms_batch`` of a batch, its arrays checked; ``tokens``: with its token ids (attention
    reads none, nor the slots)."""
    T, B = batch.n_tokens, batch.q_lens.numel()
    i32 = torch.int32
    tables = batch.block_tables
    shape = tables.shape
    if len(shape) != 2:
        raise ValueError("block_tables must be (B, max_blocks)")
    return _PACK_BATCH(
        T, B, shape[1], batch.max_q, batch.max_context, 0,
        _check(batch.input_ids, "input_ids", i32, index, (T,)) if tokens else 0,
        _check(batch.positions, "positions", i32, index, (T,)), 0,
        _check(batch.q_start, "q_start", i32, index, (B + 1,)),
        _check(batch.context_lens, "context_lens", i32, index, (B,)),
        _check(tables, "block_tables", i32, index, (B, shape[1])))


def _heads(t: torch.Tensor, name: str, index: int, dtype: torch.dtype, n_tokens: int, heads: int,
           dh: int) -> int:
    """The row stride of a (T, heads, d_head) tensor whose rows are contiguous."""
    if t.shape != (n_tokens, heads, dh) or t.dtype is not dtype or t.get_device() != index:
        raise ValueError(f"{name} must be {dtype} ({n_tokens}, {heads}, {dh}) on cuda:{index}; got "
                         f"{t.dtype} {tuple(t.shape)} on {t.device}")
    s0, s1, s2 = t.stride()
    if (dh > 1 and s2 != 1) or (heads > 1 and s1 != dh) or (n_tokens > 1 and s0 < heads * dh):
        raise ValueError(f"{name} must have contiguous heads, one behind the other")
    return s0 if n_tokens > 1 else heads * dh


def paged_attention(
    q: torch.Tensor,
    k_pool: torch.Tensor,
    v_pool: torch.Tensor,
    batch: PagedBatch,
    form: AttentionForm | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of ``q`` (T, n_heads, d_head) over one layer's pools (``PagedKVCache.k_cache[l]``,
    ``v_cache[l]``), which hold the batch's own keys and values already.

    ``form`` None: plain causal.  Rows of ``q`` may be strided (the first columns of a fused
    projection); ``out`` too, and it must not overlap ``q`` or the pools.  A query that sees no
    key gives 0.  float32 or bfloat16, d_head 8, 16, 32, 64 or 128."""
    index = _lib.cuda_index(q)
    q_shape, shape = q.shape, k_pool.shape
    if len(q_shape) != 3 or len(shape) != 4:
        raise ValueError("q must be (T, n_heads, d_head) and a pool (blocks, n_kv_heads, block_size, d_head)")
    T, heads, dh = q_shape
    dt = q.dtype
    code = _CODES.get(dt)
    if code is None:
        raise ValueError(f"q must be float32 or bfloat16, got {dt}")
    if batch.n_tokens != T:
        raise ValueError(f"q has {T} tokens, the batch {batch.n_tokens}")
    blocks, hkv, block, pool_dh = shape
    pointers = (c_void_p * 2)(_check(k_pool, "k_pool", dt, index, shape),
                              _check(v_pool, "v_pool", dt, index, shape))
    if pool_dh != dh or hkv == 0 or heads % hkv:
        raise ValueError(f"q has {heads} heads of {dh}, the pools {hkv} of {pool_dh}")
    q_stride = _heads(q, "q", index, dt, T, heads, dh)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)
        out_stride = heads * dh
    else:
        out_stride = _heads(out, "out", index, dt, T, heads, dh)
        _refuse_overlap(q, q_stride, out, out_stride, heads * dh)
    if T == 0:
        return out
    where = addressof(pointers)
    cache = _PACK_CACHE(1, blocks, block, hkv, dh, code, where, where + 8)
    cb = pack_batch(batch, index)
    cf = None if form is None else _PACK_FORM(*form.fields(index, heads, batch))
    need = (_lib._lib or _lib.load()).ms_attention_form_workspace_size(cache, heads, cb, cf)
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _lib.launch_on(index, "ms_paged_attention_form", q.data_ptr(), q_stride, cache, 0, cb, heads, cf,
                   out.data_ptr(), out_stride, None if ws is None else ws.data_ptr(), need)
    return out


def _refuse_overlap(q: torch.Tensor, q_stride: int, out: torch.Tensor, out_stride: int, width: int) -> None:
    size, T = q.element_size(), q.shape[0]
    a, b = q.data_ptr(), out.data_ptr()
    apart = a + ((T - 1) * q_stride + width) * size <= b or b + ((T - 1) * out_stride + width) * size <= a
    if T and not apart:
        gap = (b - a) % (q_stride * size)  # other columns of the same rows
        if q_stride != out_stride or gap < width * size or gap > (q_stride - width) * size:
            raise ValueError("out must not overlap q")

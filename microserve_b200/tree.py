"""Trees of drafted tokens: verified in one paged pass, instead of one chain per request.

A tree's nodes are tokens of one sequence's pass: node 0 is the last token that the
target has not seen, every other node names an earlier one as its parent and
stands one position behind it.  A node attends to the cached context, its ancestors
and itself (``AttentionForm.tree_mask``).  The target's token after a node is
emitted; when a child of the node is that token, the walk goes on there.  The
accepted path's keys and values are then moved behind node 0 (``move_tokens``)
and the sequence cut to it.  The reference verifies chains only (reference
src/microserve/speculative.py:158-211).

With ``SamplingConfig`` draws, the token after a node at depth ``d`` uses the
request's uniform of draw step ``step + d``, as a run of ordinary passes does: the
stream is the one that those would draw, whatever the trees are.
"""

from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass
from typing import TYPE_CHECKING

import numpy as np
import torch

from . import _lib
from .attention import AttentionForm, pack_batch
from .batching import batch_from_host, host_batch_arrays, pack_int32
from .cache import MAX_MOVES, PagedKVCache, move_tokens
from .config import SamplingConfig
from .sampling import make_params, params_to_device, validate

if TYPE_CHECKING:
    from .model import PagedBatch, Transformer

MAX_NODES = 1024  # MS_TREE_MAX
_check = _lib.check_tensor


def tree_masks(parents: torch.Tensor, q_start: torch.Tensor, max_nodes: int,
               words: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
    """Mask rows (T, words) int32 for ``AttentionForm.tree_mask`` and depths (T,) int32 of the nodes
    of trees with up to ``max_nodes`` nodes each: ``parents`` (T,) int32 gives each node's
    parent by its number in its own tree, -1 for a root; sequence ``b``'s nodes are
    ``[q_start[b], q_start[b + 1])``.  ``words`` defaults to what ``max_nodes`` needs."""
    index = _lib.cuda_index(parents)
    T, B = parents.numel(), q_start.numel() - 1
    if not 0 <= max_nodes <= MAX_NODES:
        raise ValueError(f"trees of {max_nodes} nodes (at most {MAX_NODES})")
    words = words or max(1, -(-max_nodes // 32))
    if words < 0 or 32 * words < max_nodes:
        raise ValueError(f"{words} words are too few for {max_nodes} nodes")
    p = _check(parents, "parents", torch.int32, index, (T,))
    s = _check(q_start, "q_start", torch.int32, index, (max(B, 0) + 1,))
    masks = torch.empty((T, words), dtype=torch.int32, device=parents.device)
    depths = torch.empty(T, dtype=torch.int32, device=parents.device)
    if T:
        _lib.launch_on(index, "ms_tree_masks", p, s, B, T, max_nodes, masks.data_ptr(), words,
                       depths.data_ptr())
    return masks, depths


@dataclass
class TreeAccept:
    """What a walk accepted; rows are -1 behind it.  ``tokens`` (B, max_accept + 1) the emitted
    tokens, ``num_accepted`` (B,), ``nodes`` (B, max_accept) the accepted nodes after node 0,
    ``src_slots`` and ``dst_slots`` (B, max_accept) the moves that put them behind it."""

    tokens: torch.Tensor
    num_accepted: torch.Tensor
    nodes: torch.Tensor
    src_slots: torch.Tensor
    dst_slots: torch.Tensor


def accept_trees(target: torch.Tensor, batch: PagedBatch, parents: torch.Tensor, max_accept: int,
                 block_size: int, num_blocks: int = 0) -> TreeAccept:
    """Walk down each tree of ``batch`` (its ``input_ids`` are the nodes) along the target's tokens.

    ``target``: the float32 logits (T, vocab) of all nodes, whose largest is the token
    (the lowest of equals; only the path's rows are read), or the drawn tokens (T,) int32.
    At most ``max_accept`` nodes behind node 0 are accepted.  ``num_blocks`` 0: the tables' block
    ids are not checked against a pool."""
    index = _lib.cuda_index(target)
    T, B = batch.n_tokens, batch.q_lens.numel()
    if max_accept < 0 or block_size < 1 or num_blocks < 0:
        raise ValueError("max_accept and num_blocks must not be negative, block_size positive")
    if batch.max_q > MAX_NODES:
        raise ValueError(f"trees of {batch.max_q} nodes (at most {MAX_NODES})")
    logits = tokens = stride = vocab = 0
    if target.dim() == 2:
        vocab, stride = target.shape[1], target.stride(0)
        if target.shape[0] != T or target.dtype is not torch.float32 or vocab == 0 \
                or (vocab > 1 and target.stride(1) != 1) or (T > 1 and stride < vocab):
            raise ValueError(f"logits must be a float32 ({T}, vocab) tensor with contiguous rows")
        logits = target.data_ptr()
    else:
        tokens = _check(target, "target tokens", torch.int32, index, (T,))
    cb = pack_batch(batch, index, True)
    p = _check(parents, "parents", torch.int32, index, (T,))
    # one allocation: tokens, nodes, sources, destinations, counts
    A = max_accept
    flat = parents.new_empty(B * (4 * A + 2))
    view, o, rows = flat.as_strided, flat.storage_offset(), (A, 1)
    out = TreeAccept(view((B, A + 1), (A + 1, 1), o), view((B,), (1,), o + B * (4 * A + 1)),
                     view((B, A), rows, o + B * (A + 1)), view((B, A), rows, o + B * (2 * A + 1)),
                     view((B, A), rows, o + B * (3 * A + 1)))
    if B:
        at = flat.data_ptr()
        _lib.launch_on(index, "ms_tree_accept", logits or None, stride, vocab, tokens or None, cb,
                       p or None, A, block_size, num_blocks or 0x7FFFFFFF // block_size, at,
                       at + 4 * B * (4 * A + 1), at + 4 * B * (A + 1), at + 4 * B * (2 * A + 1),
                       at + 4 * B * (3 * A + 1))
    return out


def _check_tree(tokens: Sequence[int], parents: Sequence[int], vocab: int) -> None:
    if len(tokens) != len(parents) or not tokens:
        raise ValueError("a tree needs a token and a parent for each node, and node 0")
    if len(tokens) > MAX_NODES:
        raise ValueError(f"a tree of {len(tokens)} nodes (at most {MAX_NODES})")
    if parents[0] != -1 or any(not 0 <= p < i for i, p in enumerate(parents) if i):
        raise ValueError("node 0 is the root (parent -1); every other node's parent is an earlier node")
    if any(not 0 <= t < vocab for t in tokens):
        raise ValueError("a node's token is outside the vocabulary")


def verify_trees(
    model: Transformer,
    cache: PagedKVCache,
    seq_ids: Sequence[int],
    trees: Sequence[tuple[Sequence[int], Sequence[int]]],
    sampling: Sequence[SamplingConfig] | None = None,
    seeds: Sequence[int] | None = None,
    steps: Sequence[int] | None = None,
) -> list[list[int]]:
    """One verify pass over a tree ``(tokens, parents)`` for each sequence; returns the emitted tokens
    of each (at least one), the last of which is the next tree's node 0.

    The cache holds everything before node 0; afterwards it holds node 0 and the accepted
    nodes too.  ``sampling`` None: greedy; else draws with each request's ``seeds`` and draw
    ``steps`` (the emitted tokens take one step each).  A sequence whose last block is shared
    with a fork needs its own first (``cache.unshare_many``).  On an error the cache is as it
    was, except that blocks may have been allocated and freed."""
    if not (len(seq_ids) == len(trees)):
        raise ValueError("seq_ids and trees must align")
    if not seq_ids:
        return []
    cfg = model.cfg
    B = len(seq_ids)
    if sampling is not None:
        if not (len(sampling) == B and seeds is not None and steps is not None
                and len(seeds) == B and len(steps) == B):
            raise ValueError("sampling needs a configuration, a seed and a step for each sequence")
        for s in sampling:
            validate(s)
            if s.controlled:
                raise ValueError("penalties, biases and allowed tokens cannot be combined with trees")
    for tokens, parents in trees:
        _check_tree(tokens, parents, cfg.vocab_size)
    if len(set(seq_ids)) != B:
        raise ValueError("a sequence appears twice in one batch")
    depths = []
    for _, parents in trees:
        d = [0]
        for p in parents[1:]:
            d.append(d[p] + 1)
        depths.append(d)
    before = [cache.num_tokens(s) for s in seq_ids]
    if any(n + max(d) >= cfg.max_seq_len for n, d in zip(before, depths)):
        raise ValueError(f"a tree reaches beyond max_seq_len={cfg.max_seq_len}")
    for s, n in zip(seq_ids, before):
        held = cache.tables[s].blocks[n // cache.block_size :] if s in cache.tables else []
        if any(cache.allocator.refcount(block) > 1 for block in held):
            raise ValueError(f"sequence {s} shares its last block with another: unshare it first")
    new = [s for s in seq_ids if s not in cache.tables]
    try:
        parts, width, max_q, n_tokens = host_batch_arrays(cache, seq_ids, [t for t, _ in trees], before)
    except BaseException:
        for s in new:
            cache.free(s)
        raise
    emitted, kept = [], list(before)
    try:
        parts[1] = np.array([n + k for n, d in zip(before, depths) for k in d], np.int32)
        flat = np.array([p for _, ps in trees for p in ps], np.int32)
        parts.append(flat)
        blob, spans = pack_int32(parts)
        dev = torch.from_numpy(blob).to(cache.device)
        batch = batch_from_host(dev, spans[:7], B, width, max_q, n_tokens, int(parts[4].max()))
        parents_dev = dev[spans[7][0] : spans[7][0] + spans[7][1]]
        masks, _ = tree_masks(parents_dev, batch.q_start, max_q)
        logits = model.forward_paged(batch, cache, form=AttentionForm(tree_mask=masks))
        target = logits
        if sampling is not None and not all(s.greedy for s in sampling):
            rows = [(s, seed, step + k) for s, seed, step, d in zip(sampling, seeds, steps, depths) for k in d]
            params = params_to_device(
                make_params([r[0] for r in rows], [r[1] for r in rows], [r[2] for r in rows]), cache.device)
            target = torch.empty(n_tokens, dtype=torch.int32, device=cache.device)
            _lib.launch_on(_lib.cuda_index(logits), "ms_sample", logits.data_ptr(), cfg.vocab_size, n_tokens,
                           cfg.vocab_size, params.data_ptr(), None, _lib.LANE_SAMPLE, target.data_ptr(),
                           None, None, None, None)
        most = max(max(d) for d in depths)
        got = accept_trees(target, batch, parents_dev, most, cache.block_size, cache.cfg.num_blocks)
        # (a path's nodes never stand before their new places, so what a later call still has to read
        # is not written by an earlier one)
        for at in range(0, most, MAX_MOVES):
            src, dst = (t[:, at : at + MAX_MOVES].contiguous() for t in (got.src_slots, got.dst_slots))
            move_tokens(cache.pool, src, dst)
        accepted = got.num_accepted.tolist()
        emitted = [row[: n + 1] for row, n in zip(got.tokens.tolist(), accepted)]
        kept = [n + 1 + k for n, k in zip(before, accepted)]
        new = []
    finally:
        cache.truncate_many(seq_ids, kept)
        for s in new:  # (only an error leaves any)
            cache.free(s)
    return emitted

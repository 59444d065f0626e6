"""What a request sets for its own logits before a draw: penalties for repeated
tokens, per-token biases and grammar masks.

``apply_logit_controls`` computes, for row ``i`` of request ``b`` (a row that
sees the request's first ``first_proposal + i`` proposals of a speculative
round as already said) and token ``v`` with raw logit ``x``::

    c = times v was generated;  s = v is in the prompt or was generated
    y = (x / repetition if x > 0 else x * repetition) if s else x
    y = y - frequency * c - (presence if c > 0 else 0)
    y = y + bias[v]
    y = y if the row's mask allows v else -inf

in float32, one kernel (``ms_apply_logit_controls``) for the whole batch.  What each
request has said lives on the device (:class:`TokenCounts`) and is updated from
the drawn tokens there, so a speculative round never waits for the host.
The reference samples from unmodified logits; none of this has a counterpart
there.  :class:`RequestControls` is the host side the engine and the
speculative decoder use.
"""

from __future__ import annotations

import struct
from collections.abc import Iterable, Sequence
from dataclasses import dataclass
from typing import TYPE_CHECKING

import numpy as np
import torch

from . import _lib
from .batching import HostStaging, pack_int32

if TYPE_CHECKING:
    from .config import SamplingConfig
    from .scheduler import Request

MAX_PROPOSALS = 64
_check = _lib.check_tensor
# ms_logit_controls as bytes (a third of the time a ctypes structure takes to fill)
_PACK_CONTROLS = struct.Struct("=QQQQiiQiiQQQQQii").pack


def mask_words(vocab_size: int) -> int:
    """32-bit words of one mask or seen row."""
    return (vocab_size + 31) // 32


def pack_masks(allowed: np.ndarray) -> np.ndarray:
    """``(n, vocab)`` truth values (True: allowed) as ``(n, words)`` int32 words,
    token ``v`` at bit ``v % 32`` of word ``v // 32``."""
    allowed = np.asarray(allowed, dtype=bool)
    n, vocab = allowed.shape
    full = np.zeros((n, mask_words(vocab) * 32), dtype=np.uint8)
    full[:, :vocab] = allowed
    return np.packbits(full, axis=1, bitorder="little").view("<u4").view(np.int32)


@dataclass
class TokenCounts:
    """What the requests have said, one slot each: ``counts`` (slots, vocab)
    int32, how often each token was generated; ``seen`` (slots, words) int32
    bit words, set for tokens in the prompt or generated."""

    counts: torch.Tensor
    seen: torch.Tensor

    @classmethod
    def empty(cls, n_slots: int, vocab_size: int, device: str | torch.device = "cuda") -> TokenCounts:
        dev = _lib.require_cuda(device)
        if n_slots < 1 or vocab_size < 1:
            raise ValueError("n_slots and vocab_size must be at least 1")
        return cls(torch.zeros((n_slots, vocab_size), dtype=torch.int32, device=dev),
                   torch.zeros((n_slots, mask_words(vocab_size)), dtype=torch.int32, device=dev))

    @property
    def n_slots(self) -> int:
        return self.counts.shape[0]

    @property
    def vocab_size(self) -> int:
        return self.counts.shape[1]

    def pointers(self, index: int) -> tuple[int | None, int | None]:
        """Data pointers of counts and seen, checked to lie on CUDA device ``index``."""
        n, v = self.counts.shape
        return (_check(self.counts, "counts", torch.int32, index, (n, v)),
                _check(self.seen, "seen", torch.int32, index, (n, mask_words(v))))

    def reset(self, slots: torch.Tensor) -> None:
        """Forget everything in ``slots`` (int32, device; negative: skipped)."""
        dev = _lib.cuda_index(self.counts)
        c, s = self.pointers(dev)
        p = _check(slots, "slots", torch.int32, dev, (slots.numel(),))
        _lib.launch_on(dev, "ms_token_counts_reset", c, s, self.n_slots, self.vocab_size, p,
                       slots.numel())

    def append(self, slots: torch.Tensor, tokens: torch.Tensor, lens: torch.Tensor | None = None,
               len_add: int = 0, row_start: torch.Tensor | None = None, max_len: int | None = None,
               n_prompt: torch.Tensor | None = None) -> None:
        """Count sequence ``i``'s tokens into slot ``slots[i]``.

        Without ``row_start``, ``tokens`` is (n, width) int32 and row ``i``'s
        first ``lens[i] + len_add`` tokens count (all of them without
        ``lens``).  With it (int64), ``tokens`` is flat, sequence ``i`` starts at
        ``row_start[i]`` and ``max_len`` bounds every length; each sequence must
        lie inside ``tokens``.  The first ``n_prompt[i]`` tokens are prompt:
        they only become seen."""
        dev = _lib.cuda_index(self.counts)
        c, s = self.pointers(dev)
        n = slots.numel()
        ps = _check(slots, "slots", torch.int32, dev, (n,))
        pl = None if lens is None else _check(lens, "lens", torch.int32, dev, (n,))
        pp = None if n_prompt is None else _check(n_prompt, "n_prompt", torch.int32, dev, (n,))
        pr = None
        if row_start is None:
            stride = width = tokens.shape[-1]
            pt = _check(tokens, "tokens", torch.int32, dev, (n, width))
        else:
            pr = _check(row_start, "row_start", torch.int64, dev, (n,))
            pt = _check(tokens, "tokens", torch.int32, dev, (tokens.numel(),))
            if max_len is None or lens is None:
                raise ValueError("flat tokens need lens and max_len")
            stride, width = 0, max_len
        if lens is None:
            len_add = width
        if n == 0 or width == 0:
            return
        _lib.launch_on(dev, "ms_token_counts_append", c, s, self.n_slots, self.vocab_size, ps, n,
                       pt, pr, stride, pl, len_add, width, pp)


@dataclass
class LogitControls:
    """The controls of a batch's requests, as device tensors (None: not used).

    ``slots`` (B,) int32, the requests' rows in a :class:`TokenCounts` (negative: no
    penalties) and ``penalties`` (B, 3) float32: repetition, presence,
    frequency.  ``bias_start`` (B + 1,), ``bias_ids`` int32 and ``bias_values``
    float32: request ``b``'s biases are entries ``bias_start[b]`` up to
    ``bias_start[b + 1]``, ids ascending.  ``masks`` (n, words) int32 bit words (see
    :func:`pack_masks`) and ``mask_rows`` (rows,) int32: each row's mask
    (negative: none)."""

    slots: torch.Tensor | None = None
    penalties: torch.Tensor | None = None
    bias_start: torch.Tensor | None = None
    bias_ids: torch.Tensor | None = None
    bias_values: torch.Tensor | None = None
    masks: torch.Tensor | None = None
    mask_rows: torch.Tensor | None = None


def apply_logit_controls(
    logits: torch.Tensor,
    controls: LogitControls,
    counts: TokenCounts | None = None,
    *,
    rows_per_request: int = 1,
    proposals: torch.Tensor | None = None,
    first_proposal: int = 0,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """The controlled logits of ``(B * rows_per_request, vocab)`` float32 rows.

    ``proposals`` (gamma, B) int32 are a speculative round's draft tokens: row
    ``i`` of a request treats its first ``first_proposal + i`` as generated.
    ``out`` may be ``logits`` itself (only the changed logits are then touched)
    or a tensor that does not overlap it; by default a new one is returned.
    Masked tokens become ``-inf``; a row whose mask and biases leave nothing is all
    ``-inf`` (there is nothing to draw from it: do not).  Rows may be strided; a row's logits must be contiguous."""
    dev = _lib.cuda_index(logits)
    if logits.dim() != 2 or logits.dtype is not torch.float32 or logits.stride(1) != 1:
        raise ValueError("logits must be a float32 (rows, vocab) tensor with contiguous rows")
    rows, vocab = logits.shape
    if rows_per_request < 1 or rows % rows_per_request:
        raise ValueError(f"{rows} rows are not a multiple of rows_per_request={rows_per_request}")
    B = rows // rows_per_request
    if out is None:
        # (empty_like costs half of what empty does)
        out = torch.empty_like(logits) if logits.is_contiguous() else \
            torch.empty((rows, vocab), dtype=torch.float32, device=logits.device)
    elif out is not logits and (out.shape != logits.shape or out.dtype is not torch.float32
                                or out.get_device() != dev or out.stride(1) != 1):
        raise ValueError("out must be a float32 tensor of the logits' shape with contiguous rows")
    if rows == 0 or vocab == 0:
        return out
    c = controls
    i32, f32 = torch.int32, torch.float32
    slots = penalties = p_counts = p_seen = props = starts = ids = values = mask_rows = masks = 0
    n_slots = n_props = n_bias = n_masks = 0
    if c.slots is not None:
        if counts is None or c.penalties is None:
            raise ValueError("penalties need slots, penalties and token counts")
        if counts.counts.shape[1] != vocab:
            raise ValueError(f"token counts are for a vocabulary of {counts.vocab_size}, not {vocab}")
        slots = _check(c.slots, "slots", i32, dev, (B,))
        penalties = _check(c.penalties, "penalties", f32, dev, (B, 3))
        p_counts, p_seen = counts.pointers(dev)
        n_slots = counts.n_slots
        if proposals is not None:
            n_props = proposals.shape[0]
            props = _check(proposals, "proposals", i32, dev, (n_props, B))
            if not 0 <= first_proposal <= n_props - rows_per_request + 1 or n_props > MAX_PROPOSALS:
                raise ValueError(f"rows see {first_proposal} to {first_proposal + rows_per_request - 1} "
                                 f"proposals of {n_props} (at most {MAX_PROPOSALS})")
            if n_props == 0:
                props = 0
    elif c.penalties is not None:
        raise ValueError("penalties need slots, penalties and token counts")
    if c.bias_start is not None:
        if c.bias_ids is None or c.bias_values is None:
            raise ValueError("bias_start needs bias_ids and bias_values")
        n_bias = c.bias_ids.numel()
        starts = _check(c.bias_start, "bias_start", i32, dev, (B + 1,))
        ids = _check(c.bias_ids, "bias_ids", i32, dev, (n_bias,))
        values = _check(c.bias_values, "bias_values", f32, dev, (n_bias,))
    if c.mask_rows is not None:
        if c.masks is None:
            raise ValueError("mask_rows needs masks")
        mask_rows = _check(c.mask_rows, "mask_rows", i32, dev, (rows,))
        n_masks = c.masks.shape[0]
        masks = _check(c.masks, "masks", i32, dev, (n_masks, mask_words(vocab)))
        if n_masks == 0:
            mask_rows = 0
    s = _PACK_CONTROLS(slots, penalties, p_counts, p_seen, n_slots, n_props, props,
                       first_proposal if props else 0, n_bias, starts, ids, values, mask_rows, masks,
                       n_masks, 0)
    in_ld, out_ld = logits.stride(0), out.stride(0)
    if rows == 1:  # the stride of a single row says nothing
        in_ld = out_ld = vocab
    _lib.launch_on(dev, "ms_apply_logit_controls", logits.data_ptr(), in_ld, out.data_ptr(), out_ld,
                   B, rows_per_request, vocab, s)
    return out


class RequestControls:
    """The controls of live requests, kept between steps (host side of the engine and of the
    speculative decoder).

    Each request with penalties holds a slot of a :class:`TokenCounts`, from its
    first step until :meth:`free`; the slots grow by doubling.  ``prepare``
    brings a batch's controls to the device; after its draws, ``drew`` counts
    the new tokens there, and ``confirm`` tells the host how many they were.  A
    request whose token lists do not have the length that was counted (its
    first step, or a caller that changed them) is counted afresh.
    """

    def __init__(self, vocab_size: int, device: torch.device) -> None:
        self.vocab_size = vocab_size
        self.device = device
        self.counts: TokenCounts | None = None
        self.version = 0  # of the uploaded controls: each prepare replaces them
        self._slot: dict[int, int] = {}
        self._counted: dict[int, int] = {}  # tokens counted, prompt included
        self._free: list[int] = []
        self._upload = HostStaging(device)
        self._recount_upload = HostStaging(device)

    def check(self, sampling: SamplingConfig) -> None:
        """Raise ``ValueError`` for biases of no token, that are no number or +inf, or that ban
        every token."""
        if sampling.logit_bias:
            self._check_bias(np.array(list(sampling.logit_bias)),
                             self._bias_values(sampling.logit_bias.values()), [len(sampling.logit_bias)])

    @staticmethod
    def _bias_values(values: Iterable[float]) -> np.ndarray:
        with np.errstate(over="ignore"):  # below float32's range: -inf, a ban
            return np.array(list(values), np.float32)

    def _check_bias(self, ids: np.ndarray, values: np.ndarray, counts: Sequence[int]) -> None:
        """Biases of requests that have ``counts`` of them each."""
        if ids.dtype.kind not in "iu" or ids.min() < 0 or ids.max() >= self.vocab_size:
            raise ValueError("logit_bias names a token outside the vocabulary")
        if not np.all(values < np.inf):
            raise ValueError("logit_bias values must be numbers below +inf")  # -inf bans a token
        end = 0
        for n in counts:
            end += n
            if n >= self.vocab_size and np.all(values[end - n : end] == -np.inf):
                raise ValueError("logit_bias bans every token")

    @staticmethod
    def wanted(requests: Sequence[Request]) -> bool:
        return any(r.sampling.controlled for r in requests)

    def masks_of(self, requests: Sequence[Request]) -> dict[int, np.ndarray]:
        """The allowed tokens of the requests that restrict them, by index.  Raises ``ValueError``
        for an array of the wrong shape or one that allows nothing the request's biases leave."""
        out: dict[int, np.ndarray] = {}
        for i, r in enumerate(requests):
            if r.sampling.allowed_tokens is None:
                continue
            got = r.sampling.allowed_tokens(list(r.output_ids))
            if got is None:
                continue
            allowed = np.asarray(got)
            if allowed.shape != (self.vocab_size,) or allowed.dtype != np.bool_:
                raise ValueError(f"request {r.request_id}: allowed_tokens must give a bool array of "
                                 f"{self.vocab_size} entries")
            left = allowed
            if r.sampling.logit_bias:
                ids = np.array(list(r.sampling.logit_bias))
                values = self._bias_values(r.sampling.logit_bias.values())
                self._check_bias(ids, values, [len(ids)])
                left = allowed.copy()
                left[ids[values == -np.inf]] = False
            if not left.any():
                raise ValueError(f"request {r.request_id}: allowed_tokens allows no token"
                                 + (" that logit_bias does not ban" if allowed.any() else ""))
            out[i] = allowed
        return out

    # -- token counts ------------------------------------------------------------
    def _grow(self, n: int) -> None:
        old = self.counts
        have = 0 if old is None else old.n_slots
        if len(self._free) >= n:
            return
        want = max(have + n - len(self._free), 2 * have)
        new = TokenCounts.empty(want, self.vocab_size, self.device)
        if old is not None:
            new.counts[:have].copy_(old.counts)
            new.seen[:have].copy_(old.seen)
        self._free += range(have, want)
        self.counts = new

    def _recount(self, requests: list[Request]) -> None:
        """Count the requests' tokens from the start."""
        slots = np.array([self._slot[r.request_id] for r in requests], np.int32)
        lens = np.array([r.num_tokens for r in requests], np.int32)
        prompts = np.array([len(r.prompt_ids) for r in requests], np.int32)
        start = (np.cumsum(lens, dtype=np.int64) - lens).view(np.int32)
        tokens = np.fromiter((t for r in requests for t in r.all_ids), np.int32, int(lens.sum()))
        blob, spans = pack_int32([start, slots, lens, prompts, tokens])
        dev = self._recount_upload.upload(blob)
        st, sl, ln, pr, tk = (dev[o : o + n] for o, n in spans)
        assert self.counts is not None
        self.counts.reset(sl)
        self.counts.append(sl, tk, ln, row_start=st.view(torch.int64), max_len=int(lens.max()),
                           n_prompt=pr)
        for r in requests:
            self._counted[r.request_id] = r.num_tokens

    def prepare(self, requests: Sequence[Request],
                masks: dict[int, np.ndarray] | None = None) -> LogitControls | None:
        """The batch's controls on the device (None: nothing to control), with ``masks`` (one
        row per request, from :meth:`masks_of`)."""
        if not self.wanted(requests):
            return None
        self.version += 1
        B = len(requests)
        parts: dict[str, np.ndarray] = {}
        if any(r.sampling.logit_bias for r in requests):
            lists = [sorted((r.sampling.logit_bias or {}).items()) for r in requests]
            ids = np.array([v for x in lists for v, _ in x])
            values = self._bias_values(b for x in lists for _, b in x)
            self._check_bias(ids, values, [len(x) for x in lists])
            parts["bias_start"] = np.cumsum([0] + [len(x) for x in lists]).astype(np.int32)
            parts["bias_ids"] = ids.astype(np.int32)
            parts["bias_values"] = values.view(np.int32)
        pen = [r for r in requests if r.sampling.penalised]
        if pen:
            new = [r for r in pen if r.request_id not in self._slot]
            self._grow(len(new))
            for r in new:
                self._slot[r.request_id] = self._free.pop()
            stale = [r for r in pen if self._counted.get(r.request_id) != r.num_tokens]
            if stale:
                self._recount(stale)
        if masks:
            parts["masks"] = pack_masks(np.stack([masks[i] for i in sorted(masks)]))
            rows = np.full(B, -1, np.int32)
            rows[sorted(masks)] = np.arange(len(masks))
            parts["mask_rows"] = rows
        if pen:
            parts["slots"] = np.array([self._slot[r.request_id] if r.sampling.penalised else -1
                                       for r in requests], np.int32)
            p = np.array([(s.repetition_penalty, s.presence_penalty, s.frequency_penalty)
                          for s in (r.sampling for r in requests)], np.float32)
            parts["penalties"] = p.view(np.int32)
        if not parts:  # allowed_tokens alone, and every one of them allowed everything
            return None
        blob, spans = pack_int32(list(parts.values()))
        dev = self._upload.upload(blob)
        t = {k: dev[o : o + n].view(parts[k].shape) for k, (o, n) in zip(parts, spans)}
        for k in ("penalties", "bias_values"):
            if k in t:
                t[k] = t[k].view(torch.float32)
        return LogitControls(**t)

    def drew(self, controls: LogitControls | None, tokens: torch.Tensor,
             lens: torch.Tensor | None = None, len_add: int = 0) -> None:
        """Count the drawn tokens, (B, width) with ``lens + len_add`` valid ones per request."""
        if controls is not None and controls.slots is not None:
            assert self.counts is not None
            self.counts.append(controls.slots, tokens, lens, len_add)

    def confirm(self, requests: Sequence[Request], drawn: Sequence[int]) -> None:
        """The batch's requests are getting ``drawn`` new tokens each."""
        for r, n in zip(requests, drawn, strict=True):
            if r.request_id in self._counted:
                self._counted[r.request_id] += int(n)

    def free(self, request_id: int) -> None:
        slot = self._slot.pop(request_id, None)
        self._counted.pop(request_id, None)
        if slot is not None:
            self._free.append(slot)

    def reset(self) -> None:
        for rid in list(self._slot):
            self.free(rid)

"""Inputs and a plain implementation in 64 bits for attention with score forms.

The reference goes by the definition: for each sequence, head and query the visible keys are
listed one by one, and only those enter any sum, so whatever stands elsewhere in the
pools (stale pages, other branches) cannot matter.

Tolerance, per output element.  With A = sum_j p_j |v_j| (p normalised) and x the
scores:
* a score is off by at most E = (dh + 8) 2^-23 max_j sum_d |q_d k_jd| scale (products summed
  with one rounding or truncation each, in float32) + 2^-21 max|x| + 2^-20 (scaling, cap,
  distance term, exponent: a few roundings of values of that size); that moves p by a factor
  within exp(2 E), so the result by at most 2 E A (1 + E) -- 2.1 E A for the small E here;
* float32: sums of n terms in any order, n 2^-23 A, and a few roundings of the result;
* bf16: each p may enter the product rounded (2^-8 A), the sum of the p then being of the
  rounded ones or of the others (2^-8 |o|), and the result is rounded (2^-8 |o|)."""

from __future__ import annotations

from dataclasses import dataclass

import numpy as np
import torch

DEV = "cuda"


@dataclass
class Inputs:
    q: torch.Tensor  # (T, hq, dh) on the CPU
    k: torch.Tensor  # (blocks, hkv, bs, dh)
    v: torch.Tensor
    tables: np.ndarray
    q_lens: list[int]
    context: list[int]
    positions: np.ndarray
    masks: np.ndarray | None  # (T, max_q) truth values
    slopes: np.ndarray | None
    prefix: np.ndarray | None
    softcap: float
    window: int
    scale: float

    @property
    def q_start(self) -> np.ndarray:
        return np.concatenate([[0], np.cumsum(self.q_lens)]).astype(np.int32)

    def batch(self, dev: str = DEV):
        from microserve_b200.model import PagedBatch

        t = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(dev)  # noqa: E731
        T = sum(self.q_lens)
        z = np.zeros(T, np.int32)
        return PagedBatch(input_ids=t(z), positions=t(self.positions), slot_mapping=t(z),
                          block_tables=t(self.tables), context_lens=t(self.context), q_lens=t(self.q_lens),
                          q_start=t(self.q_start), max_q=max(self.q_lens), n_tokens=T,
                          max_context=max(self.context))

    def form(self, dev: str = DEV):
        from microserve_b200.attention import AttentionForm

        f = lambda a, dt: None if a is None else torch.from_numpy(np.ascontiguousarray(a, dt)).to(dev)  # noqa: E731
        words = None
        if self.masks is not None:
            words = torch.from_numpy(pack_bits(self.masks).view(np.int32)).to(dev)
        return AttentionForm(softcap=self.softcap, slopes=f(self.slopes, np.float32), window=self.window,
                             prefix_lens=f(self.prefix, np.int32), tree_mask=words, scale=self.scale)


def pack_bits(flags: np.ndarray) -> np.ndarray:
    n, w = flags.shape
    words = -(-w // 32)
    full = np.zeros((n, words * 32), np.uint64)
    full[:, :w] = flags
    return (full.reshape(n, words, 32) << np.arange(32, dtype=np.uint64)).sum(-1).astype(np.uint32)


def tree_of(n: int, rng: np.random.Generator) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Parents, depths and the (n, n) ancestor matrix of a random tree."""
    parents, depths, sees = np.full(n, -1), np.zeros(n, int), np.eye(n, dtype=bool)
    for i in range(1, n):
        parents[i] = rng.integers(max(0, i - 6), i)
        depths[i] = depths[parents[i]] + 1
        sees[i] |= sees[parents[i]]
    return parents, depths, sees


def make(seed: int, dtype: torch.dtype, hq: int, hkv: int, dh: int, bs: int, cached: list[int], q_lens: list[int],
         *, tree: bool = False, softcap: float = 0.0, alibi: bool = False, window: int = 0,
         prefix: list[int] | None = None, scale: float = 0.0, spread: float = 2.0, stale: float = float("nan"),
         masks: np.ndarray | None = None) -> Inputs:
    """Random inputs; whatever no sequence holds is ``stale`` in both pools."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    context = [c + n for c, n in zip(cached, q_lens)]
    need = [-(-c // bs) for c in context]
    blocks = sum(need) + 3
    order = rng.permutation(blocks)
    tables = np.zeros((len(need), max(1, max(need))), np.int32)
    at = 0
    for b, n in enumerate(need):
        tables[b, :n] = order[at : at + n]
        tables[b, n:] = rng.integers(0, blocks, tables.shape[1] - n)  # ids left from earlier
        at += n
    k, v = (torch.full((blocks, hkv, bs, dh), stale, dtype=dtype) for _ in range(2))
    for b, c in enumerate(context):
        for p in range(need[b]):
            n = min(bs, c - p * bs)
            for t in (k, v):
                t[tables[b, p], :, :n] = torch.randn((hkv, n, dh), generator=g).to(dtype)
    T = sum(q_lens)
    q = (torch.randn((T, hq, dh), generator=g) * spread).to(dtype)
    positions, flags = [], np.zeros((T, max(q_lens)), bool)
    row = 0
    for c, n in zip(cached, q_lens):
        if tree:
            _, depths, sees = tree_of(n, rng)
            positions += (c + depths).tolist()
            flags[row : row + n, :n] = sees
        else:
            positions += range(c, c + n)
        row += n
    slopes = 2.0 ** (-8.0 * np.arange(1, hq + 1) / hq) if alibi else None
    return Inputs(q, k, v, tables, list(q_lens), context, np.array(positions, np.int32),
                  (flags if masks is None else masks) if tree else None, slopes,
                  None if prefix is None else np.array(prefix, np.int32), softcap, window, scale)


def visible(x: Inputs, b: int, i: int) -> tuple[np.ndarray, np.ndarray]:
    """The keys that query i of sequence b sees, and their distances."""
    t0, n, ctx = int(x.q_start[b]), x.q_lens[b], x.context[b]
    base, p = ctx - n, int(x.positions[int(x.q_start[b]) + i])
    j = np.arange(ctx)
    at = j.copy()
    if x.masks is not None:
        at[base:] = x.positions[t0 : t0 + n]
        seen = np.concatenate([np.ones(base, bool), x.masks[t0 + i, :n]])
    else:
        seen = at <= p
    if x.window:
        seen &= p - at < x.window
    if x.prefix is not None:
        seen |= j < x.prefix[b]
    return np.flatnonzero(seen), (p - at)[seen]


def reference(x: Inputs) -> tuple[torch.Tensor, torch.Tensor]:
    """The result in 64 bits and the tolerance for each element."""
    T, hq, dh = x.q.shape
    _, hkv, bs, _ = x.k.shape
    group = hq // hkv
    bf16 = x.q.dtype is torch.bfloat16
    out = torch.zeros((T, hq, dh), dtype=torch.float64)
    tol = torch.zeros_like(out)
    scale = x.scale or dh ** -0.5
    for b, n in enumerate(x.q_lens):
        pages = torch.from_numpy(x.tables[b, : -(-x.context[b] // bs)].astype(np.int64))
        k = x.k[pages].permute(1, 0, 2, 3).reshape(hkv, -1, dh).double()  # (hkv, keys, dh)
        v = x.v[pages].permute(1, 0, 2, 3).reshape(hkv, -1, dh).double()
        for i in range(n):
            row = int(x.q_start[b]) + i
            seen, away = visible(x, b, i)
            if not len(seen):
                continue
            j = torch.from_numpy(seen)
            kk, vv = k[:, j], v[:, j]
            qq = x.q[row].double().view(hkv, group, dh)
            s = torch.einsum("hgd,hjd->hgj", qq, kk) * scale
            size = torch.einsum("hgd,hjd->hgj", qq.abs(), kk.abs()) * scale
            if x.softcap:
                s = x.softcap * torch.tanh(s / x.softcap)
            if x.slopes is not None:
                f32 = torch.from_numpy(x.slopes.astype(np.float32).astype(np.float64)).view(hkv, group, 1)
                bias = f32 * torch.from_numpy(np.abs(away).astype(np.float64))
                s, size = s - bias, size
            p = torch.softmax(s, -1)
            o, a = p @ vv, p @ vv.abs()
            near = p > 2.0 ** -40  # what is far below the row's maximum does not matter
            big = torch.where(near, s.abs(), 0.0).amax(-1, keepdim=True)
            most = torch.where(near, size, 0.0).amax(-1, keepdim=True)
            e = (dh + 8) * 2.0 ** -23 * most + 2.0 ** -21 * big + 2.0 ** -20
            t = 2.1 * e * a + (len(seen) + 8) * 2.0 ** -23 * a
            if bf16:
                t = t + 2.0 ** -8 * (2 * o.abs() + a)
            out[row] = o.reshape(hq, dh)
            tol[row] = t.reshape(hq, dh)
    return out, tol


def run(x: Inputs, q: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    from microserve_b200.attention import paged_attention

    return paged_attention(x.q.to(DEV) if q is None else q, x.k.to(DEV), x.v.to(DEV), x.batch(), x.form(), out)


def check(got: torch.Tensor, x: Inputs, want: tuple[torch.Tensor, torch.Tensor] | None = None) -> None:
    from microserve_b200 import _lib

    assert _lib.device_error() == 0
    ref, tol = reference(x) if want is None else want
    g = got.detach().double().cpu()
    assert torch.equal(g.isfinite(), ref.isfinite())
    off = torch.where(ref.isfinite(), (g - ref).abs() - tol, 0.0)
    worst = int(off.argmax())
    assert float(off.max()) <= 0, (worst, float(g.flatten()[worst]), float(ref.flatten()[worst]),
                                   float(tol.flatten()[worst]))

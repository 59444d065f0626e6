"""Per-request logit controls and low-rank adapters restated in 64-bit numpy --
test infrastructure.  Each function also returns the sum of the
magnitudes that enter a result, from which rounding bounds are derived."""

from __future__ import annotations

import numpy as np

F64 = np.float64


def control_row(x: np.ndarray, counts: np.ndarray, seen: np.ndarray, said: list[int],
                penalty: tuple[float, float, float] | None, bias: dict[int, float],
                allowed: np.ndarray | None) -> tuple[np.ndarray, np.ndarray]:
    """One row: (controlled logits, magnitudes).  ``said`` are the proposals the
    row takes as generated; ``penalty`` = (repetition, presence, frequency)."""
    y = np.asarray(x, F64).copy()
    c = np.asarray(counts, F64).copy()
    s = np.asarray(seen, bool).copy()
    for v in said:
        c[v] += 1
        s[v] = True
    mag = np.abs(y)
    if penalty is not None:
        rep, pres, freq = (F64(np.float32(p)) for p in penalty)
        with np.errstate(invalid="ignore"):
            y = np.where(s, np.where(y > 0, y / rep, y * rep), y)
            mag = np.abs(y) + freq_abs(freq, c) + np.where(c > 0, abs(pres), 0.0)
            y = np.where(s, y - freq * c - np.where(c > 0, pres, 0.0), y)
    for v, b in bias.items():
        y[v] += F64(np.float32(b))
        mag[v] += abs(b)
    if allowed is not None:
        y[~np.asarray(allowed, bool)] = -np.inf
    return y, mag


def freq_abs(freq: float, c: np.ndarray) -> np.ndarray:
    return np.abs(freq) * c


def lora_row(x: np.ndarray, base: np.ndarray, a: np.ndarray, b: np.ndarray, scale: float,
             slice_of: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """One token: x (K,), base (N,), a (slices, r, K), b (r, N), the slice of each column:
    (y, the adapter's part, the magnitudes of its terms)."""
    low = np.asarray(a, F64) @ np.asarray(x, F64)  # (slices, r)
    mag = np.abs(np.asarray(a, F64)) @ np.abs(np.asarray(x, F64))
    bb = np.asarray(b, F64)
    part = F64(scale) * (low.T[:, slice_of] * bb).sum(0)
    terms = abs(F64(scale)) * (mag.T[:, slice_of] * np.abs(bb)).sum(0)
    return np.asarray(base, F64) + part, part, terms


def swiglu(y: np.ndarray) -> np.ndarray:
    """silu(gate) * up of columns interleaved in groups of 8."""
    v = y.reshape(-1, 2, 8)
    gate, up = v[:, 0].reshape(-1), v[:, 1].reshape(-1)
    return gate / (1.0 + np.exp(-gate)) * up

"""Paged-cache operators in 64 bits, sequence by sequence (numpy, CPU).

The definitions that the HIP kernels are held to: rotary with 64-bit angles,
attention of new tokens over their sequence's entries with a window and first
entries that stay visible, the weights that entries receive, and the choice of
those that stay.  Test infrastructure only.
"""

from __future__ import annotations

import math

import numpy as np


def rotate(x: np.ndarray, positions: np.ndarray, theta: float | None) -> np.ndarray:
    """``x[tokens, heads, dim]`` turned by ``positions[tokens]``."""

    x = np.asarray(x, dtype=np.float64)
    if theta is None:
        return x
    half = x.shape[-1] // 2
    angle = np.asarray(positions, dtype=np.float64)[:, None, None] * theta ** (-np.arange(half) / half)
    a, b = x[..., :half], x[..., half:]
    return np.concatenate((a * np.cos(angle) - b * np.sin(angle), b * np.cos(angle) + a * np.sin(angle)), -1)


def visible(first: int, tokens: int, length: int, window: int | None, sinks: int) -> np.ndarray:
    """[tokens, length]: what the token at entry first + t sees."""

    i = first + np.arange(tokens)[:, None]
    j = np.arange(length)[None]
    seen = j <= i
    if window is not None:
        seen &= (j > i - window) | (j < sinks)
    return seen


def attend(query: np.ndarray, keys: np.ndarray, values: np.ndarray, position: int, *, window: int | None, sinks: int,
           theta: float | None, scale: float | None = None) -> dict[str, np.ndarray]:
    """One sequence: ``query[T,QH,D]``, rotated ``keys``/``values``
    ``[L,KVH,D]``.  Unseen entries take part in nothing, whatever they hold.
    ``spread`` is sum p |v| and ``reach`` the largest scale * sum |q k| of a
    row: what roundings of p and q are amplified by."""

    tokens, qheads, dim = query.shape
    length, heads = keys.shape[:2]
    per = qheads // heads
    scale = dim ** -0.5 if scale is None else scale
    q = rotate(query, position + np.arange(tokens), theta)
    seen = visible(length - tokens, tokens, length, window, sinks)
    out = np.zeros((tokens, qheads, dim))
    spread = np.zeros((tokens, qheads, dim))
    reach = np.zeros((tokens, qheads))
    lse = np.full((tokens, qheads), -np.inf)
    weights = np.zeros((heads, length))
    for h in range(qheads):
        k, v = keys[:, h // per].astype(np.float64), values[:, h // per].astype(np.float64)
        for t in range(tokens):
            s = np.nonzero(seen[t])[0]
            if not len(s):
                continue
            with np.errstate(invalid="ignore", over="ignore"):
                logits = k[s] @ q[t, h] * scale
                top = logits.max()
                p = np.exp(logits - top)
                total = p.sum()
                p = p / total
                out[t, h] = p @ v[s]
                spread[t, h] = p @ np.abs(v[s])
                reach[t, h] = (np.abs(k[s]) @ np.abs(q[t, h])).max() * abs(scale)
                lse[t, h] = top + math.log(total) if total > 0 else np.nan
                weights[h // per, s] += p
    return {"out": out, "lse": lse, "weights": weights, "spread": spread, "reach": reach}


def select(weights: np.ndarray, budget: int, sinks: int, recent: int) -> np.ndarray:
    """The entries of one (sequence, head) that stay, ascending."""

    length = len(weights)
    if length <= budget:
        return np.arange(length)
    value = np.where(np.isnan(weights), -np.inf, weights.astype(np.float64) + 0.0)
    isnan = np.isnan(weights)
    inner = np.arange(sinks, length - recent)
    order = inner[np.lexsort((inner, isnan[inner], -value[inner]))]
    best = order[: budget - sinks - recent]
    return np.sort(np.concatenate((np.arange(sinks), best, np.arange(length - recent, length)))).astype(np.int64)

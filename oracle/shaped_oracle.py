"""Attention with shaped scores, its gradients, and rotary rules in 64 bits
(torch on the CPU).  The definitions that the HIP kernels are held to; test
infrastructure only.
"""

from __future__ import annotations

import math

import torch


def turn(x: torch.Tensor, positions, rates, *, layout: str = "half", magnitude: float = 1.0, sign: int = 1) -> torch.Tensor:
    """``x[N,H,D]`` with its first 2 len(rates) dims turned, as complex numbers."""

    x = x.double()
    n = len(rates)
    angle = torch.as_tensor(positions, dtype=torch.float64)[:, None] * torch.tensor(rates, dtype=torch.float64)
    spin = torch.polar(torch.full_like(angle, magnitude), sign * angle)[:, None]
    if layout == "half":
        z = torch.complex(x[..., :n].contiguous(), x[..., n : 2 * n].contiguous()) * spin
        turned = torch.cat((z.real, z.imag), -1)
    else:
        z = torch.view_as_complex(x[..., : 2 * n].contiguous().unflatten(-1, (-1, 2))) * spin
        turned = torch.view_as_real(z).flatten(-2)
    return torch.cat((turned, x[..., 2 * n :]), -1)


def rates(dims: int, theta: float, scaling: str | None = None, factor: float = 1.0, original: int = 0, low: float = 1.0,
          high: float = 4.0) -> list[float]:
    """Radians a position of each pair, written from the rules' words."""

    found = []
    for i in range(dims // 2):
        base = theta * factor ** (dims / (dims - 2)) if scaling == "base" else theta
        rate = math.exp(-2 * i / dims * math.log(base))
        if scaling == "linear":
            rate /= factor
        if scaling == "parts":
            turns = original / (2 * math.pi / rate)
            if turns < low:
                rate /= factor
            elif turns < high:
                keep = (turns - low) / (high - low)
                rate = keep * rate + (1 - keep) * rate / factor
        found.append(rate)
    return found


def visible(tokens: int, length: int, window: int | None, sinks: int, prefix: int) -> torch.Tensor:
    """[tokens, length]: what the last ``tokens`` of ``length`` entries see."""

    i = torch.arange(length - tokens, length)[:, None]
    j = torch.arange(length)[None]
    seen = ((j <= i) | (j < prefix)) & (i >= 0)
    if window is not None:
        seen &= (j > i - window) | (j < sinks)
    return seen


def scores(query, key, *, scale, cap, slope, first):
    """Shaped scores of one head, and the slope of the cap at each."""

    raw = query @ key.T * scale
    steep = torch.ones_like(raw)
    if cap:
        bent = torch.tanh(raw / cap)
        raw, steep = cap * bent, 1 - bent**2
    if slope is not None:
        i = torch.arange(query.shape[0])[:, None] + first
        raw = raw - slope * (i - torch.arange(key.shape[0])[None]).abs().double()
    return raw, steep


def attend(query, key, value, *, window=None, sinks=0, prefix=0, cap=None, slopes=None, scale=None, d_out=None) -> dict:
    """One sequence: ``query[T,QH,D]`` (its last T entries), ``key``/``value``
    ``[L,KVH,D]``, all as they enter the products.  Besides the results:
    ``spread`` sum p |v|, ``reach`` the largest scale sum |q k| of a row; with
    ``d_out`` the gradients, and what roundings of p and ds of h each change
    them by at most, per h."""

    query, key, value = query.double(), key.double(), value.double()
    tokens, qheads, dim = query.shape
    length, heads = key.shape[:2]
    per = qheads // heads
    scale = dim**-0.5 if scale is None else scale
    seen = visible(tokens, length, window, sinks, prefix)
    r = {n: torch.zeros(tokens, qheads, dim, dtype=torch.float64) for n in ("out", "spread")}
    r["lse"] = torch.full((tokens, qheads), -math.inf, dtype=torch.float64)
    r["reach"] = torch.zeros(tokens, qheads, dtype=torch.float64)
    r["weights"] = torch.zeros(heads, length, dtype=torch.float64)
    if d_out is not None:
        d_out = d_out.double()
        for n in ("dq", "dq_slack", "dq_size"):
            r[n] = torch.zeros(tokens, qheads, dim, dtype=torch.float64)
        for n in ("dk", "dv", "dk_slack", "dv_slack", "dk_size", "dv_size"):
            r[n] = torch.zeros(length, heads, dim, dtype=torch.float64)
    for h in range(qheads):
        q, k, v = query[:, h], key[:, h // per], value[:, h // per]
        x, steep = scores(q, k, scale=scale, cap=cap, slope=None if slopes is None else float(slopes[h]),
                          first=length - tokens)
        x = torch.where(seen, x, -math.inf)
        top = x.amax(-1, keepdim=True) if length else torch.full((tokens, 1), -math.inf, dtype=torch.float64)
        top = torch.where(torch.isinf(top) & (top < 0), torch.zeros_like(top), top)
        e = torch.where(seen, torch.exp(x - top), 0.0)
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total > 0, total, torch.ones_like(total))
        safe = torch.where(seen.any(0)[:, None], v, 0.0)
        r["out"][:, h] = p @ safe
        r["spread"][:, h] = p @ safe.abs()
        r["reach"][:, h] = torch.where(seen, q.abs() @ k.T.abs() * abs(scale), 0.0).amax(-1) if length else 0.0
        r["lse"][:, h] = (top + torch.log(total))[:, 0]
        r["weights"][h // per] += p.sum(0)
        if d_out is None:
            continue
        do, g = d_out[:, h], h // per
        dp = do @ v.T
        delta = (do * r["out"][:, h]).sum(-1, keepdim=True)
        slant = torch.where(seen, steep * scale, 0.0)
        ds = torch.where(seen, p * (dp - delta), 0.0) * slant
        # of ds: p and ds are rounded, delta takes the output's own rounding
        off = (p * ((do.abs() @ r["out"][:, h].abs().T).diagonal()[:, None] + 2 * (dp - delta).abs()) * slant.abs())
        size = p * (do.abs() @ v.T.abs() + (do.abs() @ r["out"][:, h].abs().T).diagonal()[:, None]) * slant.abs()
        r["dq"][:, h] = ds @ k
        r["dq_slack"][:, h] = off @ k.abs()
        r["dq_size"][:, h] = size @ k.abs()
        r["dk"][:, g] += ds.T @ q
        r["dk_slack"][:, g] += off.T @ q.abs()
        r["dk_size"][:, g] += size.T @ q.abs()
        r["dv"][:, g] += p.T @ do
        r["dv_slack"][:, g] += p.T @ do.abs()
        r["dv_size"][:, g] += p.T @ do.abs()
    return r

"""Rotary positions beyond one model's form.

The prefill, decode and paged operators turn queries and keys themselves: pairs
(i, i + D/2) of whole heads at plain frequencies, as the reference's model code
does (experiments_followup_mistral/evaluate_mistral_longbench.py:102,113,117).
:func:`rotary` is for models that do it otherwise: pairs side by side, part of a
head, frequencies scaled for contexts longer than the trained ones.  It turns
what :func:`jointkv_amd.packed_attention` takes, and what a paged cache takes
with ``rope_theta=None``; :class:`jointkv_amd.PagedKVCache` calls it where it is
given a :class:`RotaryRule`.
"""

from __future__ import annotations

import ctypes
import functools
import math
from dataclasses import dataclass

import torch

from . import _lib
from ._ops import _current, _overlaps, _plain, _refuse_second_derivative, _refuse_tangents, _written
from .attention import MISTRAL_ROPE_THETA

MOST_DIMS = 256
SCALINGS = (None, "linear", "base", "parts")


@dataclass(frozen=True)
class RotaryRule:
    """How a model's heads turn.

    Pair i of the first ``dims`` dims of a head (``None``: all) turns by
    ``theta^(-2i/dims)`` a position.  ``layout`` says which dims pair i is:
    ``"half"`` i and i + dims/2, ``"interleaved"`` 2i and 2i+1.  ``scaling``
    stretches a context by ``factor``:

    * ``"linear"``: every frequency divided by it;
    * ``"base"``: ``theta`` times ``factor^(dims/(dims-2))``, so the slowest pair
      is divided by it and the fastest keeps its frequency;
    * ``"parts"``: pairs that turn at least ``high`` times over
      ``original_length`` positions keep theirs, those below ``low`` turns are
      divided, a linear ramp over the turns between.

    Cosine and sine are multiplied by ``magnitude``.
    """

    theta: float = MISTRAL_ROPE_THETA
    layout: str = "half"
    dims: int | None = None
    scaling: str | None = None
    factor: float = 1.0
    original_length: int | None = None
    low: float = 1.0
    high: float = 4.0
    magnitude: float = 1.0

    def __post_init__(self) -> None:
        if not (self.theta > 0.0 and math.isfinite(self.theta)):
            raise ValueError("the rotary base must be positive")
        if self.layout not in ("half", "interleaved"):
            raise ValueError("the rotary layout must be 'half' or 'interleaved'")
        if self.dims is not None and (self.dims < 2 or self.dims % 2 or self.dims > MOST_DIMS):
            raise ValueError(f"the turned dims must be even, from 2 to {MOST_DIMS}")
        if self.scaling not in SCALINGS:
            raise ValueError(f"the rotary scaling must be one of {SCALINGS}")
        if not (self.factor > 0.0 and math.isfinite(self.factor)):
            raise ValueError("the scaling's factor must be positive")
        if self.scaling is None and self.factor != 1.0:
            raise ValueError("a factor needs a scaling")
        if self.scaling == "parts" and (self.original_length is None or self.original_length < 1
                                        or not 0.0 <= self.low < self.high):
            raise ValueError("scaling by parts needs the original length and 0 <= low < high")
        if not math.isfinite(self.magnitude):
            raise ValueError("the magnitude must be finite")

    def rates(self, head_dim: int) -> tuple[float, ...]:
        """Radians a position of every pair (64-bit)."""

        return _rates(self, head_dim)


@functools.lru_cache(maxsize=64)
def _rates(rule: RotaryRule, head_dim: int) -> tuple[float, ...]:
    dims = head_dim if rule.dims is None else rule.dims
    if dims > head_dim or dims % 2:
        raise ValueError(f"the turned dims must be even and at most the head's, got {dims} of {head_dim}")
    theta = rule.theta
    if rule.scaling == "base":
        if dims <= 2:
            raise ValueError("scaling the base needs more than one pair")
        grown = math.log(theta) + math.log(rule.factor) * dims / (dims - 2)
        if abs(grown) > 700.0:
            raise ValueError("the scaled rotary base passes 64 bits")
        theta *= rule.factor ** (dims / (dims - 2))
    rates = [theta ** (-2.0 * i / dims) for i in range(dims // 2)]
    if rule.scaling == "linear":
        rates = [r / rule.factor for r in rates]
    elif rule.scaling == "parts":
        for i, r in enumerate(rates):
            turns = rule.original_length * r / (2.0 * math.pi)
            keep = min(1.0, max(0.0, (turns - rule.low) / (rule.high - rule.low)))
            rates[i] = r * (keep + (1.0 - keep) / rule.factor)
    return tuple(rates)


@functools.lru_cache(maxsize=64)
def _rate_array(rule: RotaryRule, head_dim: int) -> tuple[ctypes.Array, int, int]:
    rates = _rates(rule, head_dim)
    return _lib.ptr_array(ctypes.c_double, rates), len(rates), int(rule.layout == "interleaved")


def _row_contiguous(tensor: torch.Tensor) -> torch.Tensor:
    return tensor if tensor.stride(2) == 1 else tensor.contiguous()


def _target(tensor: torch.Tensor, out: torch.Tensor | None) -> torch.Tensor:
    if out is None:
        return _plain(tensor)(tuple(tensor.shape))
    if out.dtype != tensor.dtype or out.shape != tensor.shape or out.stride(2) != 1:
        raise ValueError("outputs must match their inputs, with contiguous rows")
    if _overlaps(out):
        raise ValueError("outputs that are written must not overlap")
    return out


def _turn(query, key, rule, starts, positions, inverse, out=None, key_out=None):
    """One launch over one or two ``[N,H,D]`` tensors."""

    device = _lib.require_device(query, key, starts, positions, out, key_out)
    rows, heads, dim = query.shape
    source, target = _row_contiguous(query), _target(query, out)
    t, h, _d = source.stride()
    to_t, to_h, _d = target.stride()
    if key is None:
        key_args = (None, 0, 0, None, 0, 0, 0)
    else:
        key_source, key_target = _row_contiguous(key), _target(key, key_out)
        kt, kh, _d = key_source.stride()
        key_to_t, key_to_h, _d = key_target.stride()
        key_args = (key_source.data_ptr(), kt, kh, key_target.data_ptr(), key_to_t, key_to_h, key.shape[1])
    rates, pairs, interleaved = _rate_array(rule, dim)
    with _current(device):
        _lib.check(_lib.load().jkv_rotary(
            source.data_ptr(), t, h, target.data_ptr(), to_t, to_h, heads, *key_args, _lib.dtype_code(query.dtype), rows,
            dim, 2 * pairs, interleaved, rates, rule.magnitude, inverse, _lib.ptr(starts),
            0 if starts is None else starts.shape[0] - 1, _lib.ptr(positions), _lib.stream_handle(device)))
    return target if key is None else (target, key_target)


class _Rotary(torch.autograd.Function):
    """The gradient turns back: the same launch with the angles' signs changed."""

    @staticmethod
    def forward(ctx, query, key, rule, starts, positions):
        ctx.rule = rule
        ctx.with_key = key is not None
        ctx.shapes = query.shape, None if key is None else key.shape
        ctx.save_for_backward(starts, positions)
        return _turn(query, key, rule, starts, positions, False)

    @staticmethod
    def backward(ctx, d_query, d_key=None):
        _refuse_second_derivative("rotary")
        starts, positions = ctx.saved_tensors
        need = [ctx.needs_input_grad[0] and d_query is not None, ctx.needs_input_grad[1] and d_key is not None]
        if all(need):
            return (*_turn(d_query, d_key, ctx.rule, starts, positions, True), None, None, None)
        grads = [_turn(g, None, ctx.rule, starts, positions, True) if n else None for g, n in zip((d_query, d_key), need)]
        return (*grads, None, None, None)


def rotary(
    query: torch.Tensor,
    key: torch.Tensor | None = None,
    rule: RotaryRule = RotaryRule(),
    *,
    starts: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
    key_out: torch.Tensor | None = None,
):
    """``query`` ``[N,QH,D]`` and ``key`` ``[N,KVH,D]`` turned by ``rule`` at
    their rows' positions, in one launch.

    fp16, bf16 or fp32 (both alike), D even and at most 256, any strides of
    tokens and heads.  With ``starts`` (int32 ``[B+1]``, not decreasing) the rows
    are packed: row n of sequence b, ``starts[b] <= n < starts[b+1]``, has
    position ``positions[b] + n - starts[b]`` (``positions`` int32 ``[B]``;
    ``None``: zeros).  Without, ``positions`` is int32 ``[N]``, one a row
    (``None``: the row's number).  Rows that no sequence owns are copied as they
    are.  Angles are 64-bit products of position and frequency, the rotation
    fp32 with one rounding.

    Returns the turned query, or the pair (query, key); into ``out`` and
    ``key_out`` if given, which may be the inputs themselves but overlap them in
    no other way.  Differentiable in both (not with given outputs), once and in
    reverse: ``create_graph`` and tangents are refused.  A call repeats bit for bit.
    """

    if query.ndim != 3 or query.dtype not in (torch.float16, torch.bfloat16, torch.float32):
        raise ValueError("queries must be [N,QH,D] of fp16, bf16 or fp32")
    if key is not None and (key.ndim != 3 or key.dtype != query.dtype or key.shape[0] != query.shape[0]
                            or key.shape[2] != query.shape[2]):
        raise ValueError("keys must be [N,KVH,D] of the queries' type, rows and dims")
    if key is None and key_out is not None:
        raise ValueError("an output for keys without keys")
    if query.shape[2] % 2 or query.shape[2] > MOST_DIMS or query.shape[2] == 0:
        raise ValueError(f"rotary supports even head dims up to {MOST_DIMS}, got {query.shape[2]}")
    if starts is not None:
        if starts.dtype != torch.int32 or starts.ndim != 1 or starts.shape[0] < 1:
            raise ValueError("starts must be int32 [B+1]")
        starts = starts.contiguous()
    if positions is not None:
        count = query.shape[0] if starts is None else starts.shape[0] - 1
        if positions.dtype != torch.int32 or positions.shape != (count,):
            raise ValueError("positions must be int32 [N], or [B] beside starts")
        positions = positions.contiguous()
    _refuse_tangents("rotary", query, key)
    if torch.is_grad_enabled() and (query.requires_grad or (key is not None and key.requires_grad)):
        if out is not None or key_out is not None:
            raise ValueError("given outputs are not differentiable")
        return _Rotary.apply(query, key, rule, starts, positions)
    turned = _turn(query, key, rule, starts, positions, False, out, key_out)
    if out is not None or key_out is not None:
        _written(out, key_out)
    return turned

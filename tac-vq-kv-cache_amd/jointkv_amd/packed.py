"""Attention inside sequences that lie packed one behind another.

:func:`jointkv_amd.prefill_attention` takes one model's form: fp16 heads of 128
dims that it turns itself, sequences of one length, a causal window.
:func:`packed_attention` is for other models and other batches: texts of unequal
length packed without padding (each sees itself alone), fp16 or bf16, scores
capped or biased by distance, prefixes seen from both sides, first tokens that
stay visible behind a window.  Queries and keys come turned
(:func:`jointkv_amd.rotary`).  It is what a prompt needs before there is a cache,
and differentiable, for a caller's own training or calibration loop (the
closed-loop modules of this package call :func:`jointkv_amd.prefill_attention`).
"""

from __future__ import annotations

import torch

from . import _lib
from ._ops import _current, _overlaps, _plain, _refuse_second_derivative, _refuse_tangents, _written
from .paged import _rows, _shape_args

PACKED_TYPES = (torch.float16, torch.bfloat16)


def _place(tensor: torch.Tensor) -> tuple[torch.Tensor, tuple[int, int, int]]:
    """``tensor`` in rows that the kernels take, and its (address, token stride,
    head stride); a copy where its own are none."""

    tensor = _rows(tensor)
    if tensor.shape[0] > 1 and tensor.stride(0) >= 1 << 22:
        tensor = tensor.clone(memory_format=torch.contiguous_format)
    t, h, _d = tensor.stride()
    # (strides of one row or head say nothing)
    return tensor, (tensor.data_ptr(), t if tensor.shape[0] > 1 else 0, h if tensor.shape[1] > 1 else 0)


def _span(window: int | None, sinks: int) -> tuple[int, int]:
    return 0 if window is None else min(int(window), 0x7fffffff), min(int(sinks), 0x7fffffff)


def _forward(query, key, value, starts, prefixes, slopes, softcap, window, sinks, scale, lse, out, rest=None):
    device = _lib.require_device(query, key, value, starts, prefixes, slopes, lse, out)
    rows, qheads, dim = query.shape
    if out is None:
        out = _plain(query)((rows, qheads, dim))
    (query, q_at), (key, k_at), (value, v_at) = _place(query), _place(key), _place(value)
    with _current(device):
        _lib.check(_lib.load().jkv_packed_attention(
            *q_at, *k_at, *v_at, _lib.dtype_code(query.dtype), starts.data_ptr(), _lib.ptr(prefixes), rows,
            starts.shape[0] - 1, qheads, key.shape[1], dim, *_span(window, sinks), scale, softcap, _lib.ptr(slopes),
            out.data_ptr(), out.stride(0) if rows > 1 else 0, out.stride(1) if qheads > 1 else 0, _lib.ptr(lse),
            _lib.ptr(rest), _lib.stream_handle(device)))
    return out


class _PackedAttention(torch.autograd.Function):
    """The forward keeps each row's log-sum-exp and what the output's rounding took
    off; the backward forms the weights anew from them."""

    @staticmethod
    def forward(ctx, query, key, value, starts, prefixes, slopes, softcap, window, sinks, scale, lse):
        given, lse = lse, torch.empty(query.shape[:2], dtype=torch.float32, device=query.device)
        rest = _plain(query)(tuple(query.shape))
        out = _forward(query, key, value, starts, prefixes, slopes, softcap, window, sinks, scale, lse, None, rest)
        if given is not None:
            given.copy_(lse)  # (the caller may use its own again before the backward)
        ctx.params = (softcap, window, sinks, scale)
        ctx.save_for_backward(query, key, value, out, rest, lse, starts, prefixes, slopes)
        return out

    @staticmethod
    def backward(ctx, d_out):
        _refuse_second_derivative("packed_attention")
        query, key, value, out, rest, lse, starts, prefixes, slopes = ctx.saved_tensors
        softcap, window, sinks, scale = ctx.params
        rows, qheads, dim = query.shape
        device = query.device
        span, sinks = _span(window, sinks)
        grads = [_plain(x)(tuple(x.shape)) if need else None
                 for x, need in zip((query, key, value), ctx.needs_input_grad)]
        places = [_place(x) for x in (query, key, value, out, d_out)]  # (copies live until the launches are queued)
        with _current(device):
            ws_bytes = _lib.workspace_bytes("jkv_packed_backward_workspace_bytes", rows, starts.shape[0] - 1, qheads,
                                            key.shape[1], dim, span)
            workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
            _lib.check(_lib.load().jkv_packed_attention_backward(
                *(x for _tensor, at in places[:4] for x in at), rest.data_ptr(), *places[4][1], lse.data_ptr(),
                _lib.dtype_code(query.dtype), starts.data_ptr(), _lib.ptr(prefixes), rows, starts.shape[0] - 1, qheads, key.shape[1], dim,
                span, sinks, scale, softcap, _lib.ptr(slopes), *map(_lib.ptr, grads), workspace.data_ptr(),
                ws_bytes, _lib.stream_handle(device)))
        return (*grads, *(None,) * 8)


def packed_attention(
    query: torch.Tensor,
    key: torch.Tensor,
    value: torch.Tensor,
    starts: torch.Tensor,
    *,
    prefixes: torch.Tensor | None = None,
    window: int | None = None,
    sinks: int = 0,
    softcap: float | None = None,
    slopes: torch.Tensor | None = None,
    scale: float | None = None,
    lse: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of every row over its own sequence.

    ``query`` ``[N,QH,D]``, ``key``/``value`` ``[N,KVH,D]``, fp16 or bf16, D 64 or
    128, turned already where the model turns them; any whole number of query
    heads shares a kv head, any strides of tokens and heads.  ``starts`` (int32
    ``[B+1]``, not decreasing): sequence b is rows ``starts[b]`` to
    ``starts[b+1]``.  Its row i sees its row j if ``j <= i`` or ``j <
    prefixes[b]`` (int32 ``[B]``; a prefix as long as the sequence makes it see
    itself whole), and if ``j > i - window`` (``None``: all) or ``j < sinks``.

    A score is ``scale`` (default ``D ** -0.5``) times the product; ``softcap`` c
    (0.001 to 1024) bends it to ``c tanh(s / c)``, and ``slopes`` (fp32 ``[QH]``,
    without gradients) then takes ``slopes[h] |i - j|`` off.  ``lse`` (fp32
    ``[N,QH]``) receives each row's log-sum-exp.

    Returns ``[N,QH,D]`` (``out``, if given, which must not share memory with the
    inputs); rows that no sequence owns are 0, their ``lse`` and gradients -inf
    and 0.  Rows and gradients depend on what they see alone, whatever lies in
    other places; infinite and NaN elements reach what the formulas say.  Scores
    and sums are 32-bit, a cap c within 2e-7 c.  Weights enter the second product
    rounded once to the inputs' type, and their sum as rounded divides it; so they
    do in the values' gradient, and score gradients enter theirs as two parts:
    outputs and gradients are at most about 1.5 times as far off, in norm, as
    their own rounding.
    Differentiable in ``query``, ``key`` and ``value`` (not with a given ``out``), once
    and in reverse: ``create_graph`` and tangents are refused.  A call repeats bit for
    bit, its gradients too.
    """

    if query.ndim != 3 or query.dtype not in PACKED_TYPES:
        raise ValueError("queries must be [N,QH,D] of fp16 or bf16")
    rows, qheads, dim = query.shape
    if key.ndim != 3 or key.shape != value.shape or key.shape[0] != rows or key.shape[2] != dim:
        raise ValueError("keys and values must be [N,KVH,D] of the queries' rows and dims")
    if key.dtype != query.dtype or value.dtype != query.dtype:
        raise ValueError("queries, keys and values must be of one type")
    heads = key.shape[1]
    if heads == 0 or qheads == 0 or qheads % heads:
        raise ValueError("query heads must be a multiple of kv heads")
    if starts.dtype != torch.int32 or starts.ndim != 1 or starts.shape[0] < 1:
        raise ValueError("starts must be int32 [B+1]")
    if window is not None and window < 1:
        raise ValueError("window must be positive")
    if sinks < 0:
        raise ValueError("sinks must not be negative")
    softcap, slopes, prefixes = _shape_args(softcap, slopes, prefixes, qheads, starts.shape[0] - 1)
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (rows, qheads) or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous fp32 [N,QH] tensor")
    if out is not None:
        if out.dtype != query.dtype or out.shape != query.shape or out.stride(2) != 1 or out.stride(0) % 8 or (
                out.stride(1) % 8 or out.data_ptr() % 16 or (rows > 1 and out.stride(0) >= 1 << 22)):
            raise ValueError("out must match the queries, with contiguous 16-byte aligned rows")
        if _overlaps(out):
            raise ValueError("an out that is written must not overlap")
    scale = dim ** -0.5 if scale is None else float(scale)
    starts = starts.contiguous()
    args = (starts, prefixes, slopes, softcap, window, sinks, scale, lse)
    _refuse_tangents("packed_attention", query, key, value, slopes)
    if torch.is_grad_enabled() and (query.requires_grad or key.requires_grad or value.requires_grad):
        if out is not None:
            raise ValueError("a given out is not differentiable")
        _lib.require_device(query, key, value, starts, prefixes, slopes, lse)
        return _PackedAttention.apply(query, key, value, *args)
    result = _forward(query, key, value, *args, out)
    if out is not None or lse is not None:
        _written(out, lse)
    return result

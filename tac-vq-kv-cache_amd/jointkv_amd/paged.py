"""A paged K/V cache for batches whose sequences differ in length.

The reference's LongBench loop keeps one cache a sequence and attends a
prefill chunk over itself only (experiments_followup_mistral/
evaluate_mistral_longbench.py:29-124).  Here the (codec's) keys and values of
many sequences share one pool of pages:

* :func:`paged_append` writes new tokens into their pages, keys rotated;
* :func:`paged_attention` attends new tokens, single ones or chunks, over all
  that is cached, in a sliding window beside a few first entries that stay
  visible, and can sum up the softmax weight that every entry received;
* :func:`select_entries` and :func:`compact_pages` drop the entries that
  received least;
* :class:`PagedKVCache` keeps the pages, tables and lengths of a model's
  layers.

New tokens of a batch are packed ``[tokens, heads, dim]``: sequence b owns
rows ``starts[b]`` to ``starts[b+1]``, and they are its last entries.  Without
``starts`` there is one token a sequence, row b.  An entry's index and its
rotary position are the same until entries are evicted; from then on
``positions`` (of each sequence's first new token) runs ahead of the lengths.
Keys are stored rotated, so attention never needs a cached entry's position.

No function here synchronises, and none is differentiable (calibration trains
through :func:`jointkv_amd.prefill_attention`).
"""

from __future__ import annotations

import contextlib
from dataclasses import dataclass
from typing import Sequence

import torch

from . import _lib
from ._ops import _plain
from .attention import MISTRAL_ROPE_THETA, MISTRAL_WINDOW

PAGE_TYPES = (torch.float16, torch.bfloat16)


_NO_CHANGE = contextlib.nullcontext()


def _current(device: torch.device):
    """The device's own context where another device is current."""

    if torch._C._cuda_getDevice() == device.index:
        return _NO_CHANGE
    return torch.cuda.device(device)


def _rows(tensor: torch.Tensor) -> torch.Tensor:
    """``tensor`` with contiguous 16-byte aligned rows (a copy if need be)."""

    t, h, d = tensor.stride()
    if d != 1 or t % 8 or h % 8 or tensor.data_ptr() % 16:
        return tensor.clone(memory_format=torch.contiguous_format)  # (contiguous ones may be misaligned)
    return tensor


def _overlaps(tensor: torch.Tensor) -> bool:
    """Whether two elements of ``tensor`` share memory (strides that nest)."""

    if tensor.is_contiguous():
        return False
    span = 1
    for stride, extent in sorted(zip(tensor.stride(), tensor.shape)):
        if extent > 1 and stride < span:
            return True
        span = max(span, stride * extent)
    return False


def _pool_args(key_pages: torch.Tensor, value_pages: torch.Tensor, written: bool) -> tuple:
    if key_pages.ndim != 4 or key_pages.shape != value_pages.shape:
        raise ValueError("key and value pages must be two [pages,KVH,page_size,D] tensors of one shape")
    if key_pages.dtype not in PAGE_TYPES or key_pages.dtype != value_pages.dtype:
        raise ValueError("pages must be fp16 or bf16, keys and values alike")
    strides = key_pages.stride()
    if strides != value_pages.stride():
        raise ValueError("key and value pages need identical strides")
    if strides[3] != 1:
        raise ValueError("page rows must be contiguous")
    pages, heads, size, dim = key_pages.shape
    if written and (_overlaps(key_pages) or _overlaps(value_pages)):
        raise ValueError("pages that are written must not overlap")
    return (strides[0], strides[1], strides[2], pages, size), heads, dim


def _batch_args(block_tables, lengths, starts, positions, rows: int) -> tuple:
    if block_tables.dtype != torch.int32 or block_tables.ndim != 2:
        raise ValueError("block tables must be int32 [B,pages] with contiguous rows")
    batch, width = block_tables.shape
    row, step = block_tables.stride()
    if step != 1 and width > 1:
        raise ValueError("block tables must be int32 [B,pages] with contiguous rows")
    if lengths.dtype != torch.int32 or lengths.shape != (batch,):
        raise ValueError("lengths must be int32 [B]")
    if starts is None:
        if rows != batch:
            raise ValueError("without starts there is one new token a sequence")
    else:
        if starts.dtype != torch.int32 or starts.shape != (batch + 1,):
            raise ValueError("starts must be int32 [B+1]")
        starts = starts.contiguous()
    if positions is not None:
        if positions.dtype != torch.int32 or positions.shape != (batch,):
            raise ValueError("positions must be int32 [B]")
        positions = positions.contiguous()
    return batch, (block_tables.data_ptr(), row, width), (lengths.contiguous(), starts, positions)


def _theta(rope_theta: float | None) -> float:
    if rope_theta is None:
        return 0.0
    if not rope_theta > 0.0:
        raise ValueError("the rotary base must be positive")
    return float(rope_theta)


def paged_append(
    key: torch.Tensor,
    value: torch.Tensor,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    *,
    starts: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    rope_theta: float | None = MISTRAL_ROPE_THETA,
) -> None:
    """Write new tokens' keys, rotated, and values into their pages.

    ``key``/``value`` ``[N,KVH,D]`` (pre-RoPE, e.g. the codec's
    reconstructions) of the pages' type; ``key_pages``/``value_pages``
    ``[pages,KVH,page_size,D]`` fp16 or bf16, D 64 or 128, page sizes powers of
    two from 16; ``block_tables`` int32 ``[B,W]``; ``lengths`` int32 ``[B]``,
    the new tokens counted.  Angles are 64-bit products of position and
    frequency, the rotation fp32 with one rounding; ``rope_theta=None`` stores
    the keys as they are.  Entries whose page number lies outside the pool are
    not written, nor are packed rows that no sequence owns.
    """

    device = _lib.require_device(key, value, key_pages, value_pages, block_tables, lengths, starts, positions)
    strides, heads, dim = _pool_args(key_pages, value_pages, written=True)
    if key.ndim != 3 or key.shape != value.shape or key.shape[1:] != (heads, dim):
        raise ValueError("new keys and values must be [N,KVH,D] of the pages' heads and dims")
    if key.dtype != key_pages.dtype or value.dtype != key_pages.dtype:
        raise ValueError("new keys and values must have the pages' type")
    rows = key.shape[0]
    batch, table, (lengths, starts, positions) = _batch_args(block_tables, lengths, starts, positions, rows)
    key, value = _rows(key), _rows(value)
    with _current(device):
        _lib.check(_lib.load().jkv_paged_append(
            key.data_ptr(), key.stride(0), key.stride(1), value.data_ptr(), value.stride(0), value.stride(1),
            _lib.dtype_code(key.dtype), key_pages.data_ptr(), value_pages.data_ptr(), *strides, *table,
            lengths.data_ptr(), _lib.ptr(starts), _lib.ptr(positions), rows, batch, heads, dim, _theta(rope_theta),
            _lib.stream_handle(device)))


def paged_attention(
    query: torch.Tensor,
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    block_tables: torch.Tensor,
    lengths: torch.Tensor,
    *,
    starts: torch.Tensor | None = None,
    positions: torch.Tensor | None = None,
    window: int | None = MISTRAL_WINDOW,
    sinks: int = 0,
    rope_theta: float | None = MISTRAL_ROPE_THETA,
    scale: float | None = None,
    max_new: int | None = None,
    max_length: int | None = None,
    weights: torch.Tensor | None = None,
    accumulate: bool = False,
    lse: torch.Tensor | None = None,
    out: torch.Tensor | None = None,
) -> torch.Tensor:
    """Attention of new tokens over the cached entries of their sequences.

    ``query`` ``[N,QH,D]`` pre-RoPE, of the pages' type; the token at entry i
    of its sequence sees the entries ``j <= i`` that lie in its ``window``
    (``j > i - window``; ``None``: all) or among the first ``sinks``.  Any
    whole number of query heads shares a kv head.  ``max_new`` and
    ``max_length`` bound a sequence's new tokens and entries (defaults: all
    packed rows, the table's room); closer bounds make for a better division
    of the work.  They are promises: entries past ``max_length`` take no part,
    and rows past ``max_new`` hold anything.

    ``weights`` (fp32 ``[B,KVH,C]``, C at least ``max_length``): entry j below
    ``lengths[b]`` receives the sum of its softmax weights over the sequence's
    new tokens and the heads of its group, added to what is there with
    ``accumulate``, stored without; entries behind are left as they were.
    ``lse`` (fp32 ``[N,QH]``) receives each row's log-sum-exp.

    Returns ``[N,QH,D]`` (``out``, if given).  Rows that no sequence owns are
    left as they were; a token with no entry to see (a length below the number
    of new tokens) gets zeros and an ``lse`` of ``-inf``; a page number outside
    the pool reads as zeros.  Infinite and NaN keys and values count for the rows
    that see them alone: a score of -infinity weighs nothing, an infinite value
    makes its dim infinite.  A call repeats bit for bit; how the work is
    divided follows from the sizes and bounds, so a row may differ in its last
    bits between calls of other ones.  Calls whose ``max_new`` times the heads of
    a group is at most 32 (steps of single tokens, small chunks) keep queries and
    weights in two 16-bit parts before the matrix products, 2^-17 of each or
    better.  All sequences of other calls, single tokens among them, have both
    rounded once to the pages' type; ask for ``lse`` to keep the queries in two
    parts there (a sixth to a third slower), as they are where ``weights``
    are asked for.
    """

    device = _lib.require_device(query, key_pages, value_pages, block_tables, lengths, starts, positions, weights,
                                 lse, out)
    strides, heads, dim = _pool_args(key_pages, value_pages, written=False)
    if query.ndim != 3 or query.dtype != key_pages.dtype:
        raise ValueError("queries must be [N,QH,D] of the pages' type and dims")
    rows, qheads, query_dim = query.shape
    if query_dim != dim:
        raise ValueError("queries must be [N,QH,D] of the pages' type and dims")
    if heads == 0 or qheads == 0 or qheads % heads:
        raise ValueError("query heads must be a multiple of kv heads")
    batch, table, (lengths, starts, positions) = _batch_args(block_tables, lengths, starts, positions, rows)
    room = table[2] * strides[4]
    if window is not None and window < 1:
        raise ValueError("window must be positive")
    if sinks < 0 or (max_new is not None and max_new < 0) or (max_length is not None and max_length < 0):
        raise ValueError("sinks, max_new and max_length must not be negative")
    weight_args = (None, 0, 0, 0)
    if weights is not None:
        if weights.dtype != torch.float32 or weights.ndim != 3 or weights.shape[:2] != (batch, heads) or (
                weights.shape[2] > 1 and weights.stride(2) != 1):
            raise ValueError("weights must be fp32 [B,KVH,C] with contiguous rows")
        width, (per_batch, per_head, _one) = weights.shape[2], weights.stride()
        if max_length is None:
            max_length = min(room, width)
        elif min(max_length, room) > width:
            raise ValueError("weights have fewer entries than max_length")
        if _overlaps(weights):
            raise ValueError("weights that are written must not overlap")
        weight_args = (weights.data_ptr(), per_batch, per_head, width)
    max_length = room if max_length is None else min(int(max_length), room)
    max_new = 1 if starts is None else (rows if max_new is None else min(int(max_new), rows))
    if lse is not None and (lse.dtype != torch.float32 or lse.shape != (rows, qheads) or not lse.is_contiguous()):
        raise ValueError("lse must be a contiguous fp32 [N,QH] tensor")
    if out is None:
        out = _plain(query)((rows, qheads, dim))
    elif out.dtype != query.dtype or out.shape != query.shape or out.stride(2) != 1 or out.stride(0) % 8 or (
            out.stride(1) % 8 or out.data_ptr() % 16):
        raise ValueError("out must match the queries, with contiguous 16-byte aligned rows")
    elif _overlaps(out):
        raise ValueError("an out that is written must not overlap")
    query = _rows(query)
    span = 0 if window is None else min(int(window), 0x7fffffff)
    sinks = min(int(sinks), 0x7fffffff)
    with _current(device):
        ws_bytes = _lib.workspace_bytes("jkv_paged_attention_workspace_bytes", rows, batch, qheads, heads, dim, max_new,
                                        max_length, span, sinks, int(weights is not None))
        workspace = torch.empty(ws_bytes, dtype=torch.uint8, device=device) if ws_bytes else None
        _lib.check(_lib.load().jkv_paged_attention(
            query.data_ptr(), query.stride(0), query.stride(1), _lib.dtype_code(query.dtype), key_pages.data_ptr(),
            value_pages.data_ptr(), *strides, *table, lengths.data_ptr(), _lib.ptr(starts), _lib.ptr(positions), rows,
            batch, qheads, heads, dim, max_new, max_length, span, sinks, _theta(rope_theta),
            dim ** -0.5 if scale is None else float(scale), out.data_ptr(), out.stride(0), out.stride(1),
            _lib.ptr(lse), *weight_args, int(accumulate), _lib.ptr(workspace), ws_bytes, _lib.stream_handle(device)))
    return out


def select_entries(
    weights: torch.Tensor,
    lengths: torch.Tensor,
    budget: int,
    *,
    sinks: int = 0,
    recent: int = 0,
) -> tuple[torch.Tensor, torch.Tensor]:
    """Which entries of each sequence and kv head stay when ``budget`` may.

    Of ``lengths[b]`` entries with weights ``[B,KVH,C]`` (fp32) the first
    ``sinks`` and the last ``recent`` stay, and of the others those with the
    largest weights, the lower index first among equals (NaN below every
    number).  Returns their indices, ascending, int32 ``[B,KVH,budget]`` with
    -1 behind the last, and the new lengths ``min(lengths, budget)``.
    """

    device = _lib.require_device(weights, lengths)
    if weights.dtype != torch.float32 or weights.ndim != 3 or (weights.shape[2] > 1 and weights.stride(2) != 1):
        raise ValueError("weights must be fp32 [B,KVH,C] with contiguous rows")
    batch, heads, width = map(int, weights.shape)
    if lengths.dtype != torch.int32 or tuple(lengths.shape) != (batch,):
        raise ValueError("lengths must be int32 [B]")
    if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
        raise ValueError("the budget must be positive and hold the first and the last entries that stay")
    lengths = lengths.contiguous()
    kept = torch.empty((batch, heads, budget), dtype=torch.int32, device=device)
    new_lengths = torch.empty(batch, dtype=torch.int32, device=device)
    with _current(device):
        _lib.check(_lib.load().jkv_paged_select(
            weights.data_ptr(), weights.stride(0), weights.stride(1), lengths.data_ptr(), batch, heads, width,
            int(budget), int(sinks), int(recent), kept.data_ptr(), new_lengths.data_ptr(), _lib.stream_handle(device)))
    return kept, new_lengths


def compact_pages(
    key_pages: torch.Tensor,
    value_pages: torch.Tensor,
    block_tables: torch.Tensor,
    kept: torch.Tensor,
    new_tables: torch.Tensor,
    *,
    weights: torch.Tensor | None = None,
) -> torch.Tensor | None:
    """Copy the entries that stay into new pages of the same pool.

    Entry ``kept[b,h,j]`` (int32 ``[B,KVH,budget]``, negative: nothing) of a
    sequence's pages becomes entry j of its ``new_tables`` row.  The new pages
    must be none that are read, of this or another sequence (other sequences
    may share the old ones); an entry that stays where it is costs nothing.  With
    ``weights`` ``[B,KVH,C]`` returns those of the entries that stay, in their
    new order, zeros behind.
    """

    device = _lib.require_device(key_pages, value_pages, block_tables, kept, new_tables, weights)
    strides, heads, dim = _pool_args(key_pages, value_pages, written=True)
    tables = []
    for t in (block_tables, new_tables):
        if t.dtype != torch.int32 or t.ndim != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
            raise ValueError("block tables must be int32 [B,pages] with contiguous rows")
        tables.append((t.data_ptr(), t.stride(0), int(t.shape[1])))
    batch = int(block_tables.shape[0])
    if int(new_tables.shape[0]) != batch or kept.dtype != torch.int32 or kept.ndim != 3 or tuple(
            kept.shape[:2]) != (batch, heads):
        raise ValueError("kept entries must be int32 [B,KVH,budget] beside tables of B rows")
    kept = kept.contiguous()
    weight_args, moved = (None, 0, 0, 0), None
    if weights is not None:
        if weights.dtype != torch.float32 or weights.ndim != 3 or tuple(weights.shape[:2]) != (batch, heads) or (
                weights.shape[2] > 1 and weights.stride(2) != 1):
            raise ValueError("weights must be fp32 [B,KVH,C] with contiguous rows")
        moved = torch.empty(weights.shape, dtype=torch.float32, device=device)
        weight_args = (weights.data_ptr(), weights.stride(0), weights.stride(1), int(weights.shape[2]))
    with _current(device):
        _lib.check(_lib.load().jkv_paged_compact(
            key_pages.data_ptr(), value_pages.data_ptr(), _lib.dtype_code(key_pages.dtype), *strides, *tables[0],
            kept.data_ptr(), int(kept.shape[2]), *tables[1], batch, heads, dim, *weight_args, _lib.ptr(moved),
            _lib.stream_handle(device)))
    return moved


@dataclass(frozen=True)
class PagedStep:
    """One step's sequences as the kernels take them: every layer of the step
    appends and attends with it (until the next eviction or release).

    A captured step is replayed with ``lengths`` and ``positions`` (and
    ``starts``) refilled from a later ``begin``; give it the cache's
    ``max_length`` first (``dataclasses.replace``), as entries past the bound
    take no part."""

    block_tables: torch.Tensor
    lengths: torch.Tensor
    starts: torch.Tensor | None
    positions: torch.Tensor
    tokens: int
    max_new: int
    max_length: int


class PagedKVCache:
    """Pages, tables and lengths of a model's layers for up to ``sequences``
    sequences at once.

    Replaces one ``LayerCache`` a layer and sequence
    (evaluate_mistral_longbench.py:29-78).  All layers share one table (their
    entries are as many), each has its own pool.  A step is
    ``begin([new tokens of each sequence])``, then per layer ``append`` and
    ``attention``.  With ``track_weights`` attention adds up what every entry
    receives, and :meth:`evict` brings sequences down to a budget by it.
    """

    def __init__(
        self,
        layers: int,
        sequences: int,
        pages: int,
        kv_heads: int,
        *,
        max_length: int,
        page_size: int = 64,
        head_dim: int = 128,
        dtype: torch.dtype = torch.float16,
        track_weights: bool = False,
        device: torch.device | str = "cuda",
    ) -> None:
        if min(layers, sequences, pages, kv_heads, max_length) <= 0 or head_dim not in (64, 128):
            raise ValueError("invalid paged-cache geometry")
        if page_size < 16 or page_size > 4096 or page_size & (page_size - 1):
            raise ValueError("the page size must be a power of two from 16 to 4096")
        if dtype not in PAGE_TYPES:
            raise ValueError("pages must be fp16 or bf16")
        shape = (layers, pages, kv_heads, page_size, head_dim)
        self.key = torch.empty(shape, dtype=dtype, device=device)
        self.value = torch.empty(shape, dtype=dtype, device=device)
        self.page_size, self.max_length = page_size, max_length
        width = -(-max_length // page_size)
        device = self.key.device
        self.block_tables = torch.full((sequences, width), -1, dtype=torch.int32, device=device)
        self.weights = ([torch.zeros(sequences, kv_heads, max_length, dtype=torch.float32, device=device)
                         for _ in range(layers)] if track_weights else None)
        self._free = list(range(pages - 1, -1, -1))
        self._pages: list[list[int]] = [[] for _ in range(sequences)]
        self._lengths = [0] * sequences
        self._positions = [0] * sequences
        self._begun: tuple | None = None  # the latest step's lengths tensor, and what it is taken back to

    @property
    def lengths(self) -> tuple[int, ...]:
        """Entries of every sequence."""

        return tuple(self._lengths)

    @property
    def positions(self) -> tuple[int, ...]:
        """Position that every sequence's next token takes."""

        return tuple(self._positions)

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def _on_device(self, values: list) -> torch.Tensor:
        # a pinned copy does not wait for the device's queued work
        host = torch.tensor(values, dtype=torch.int32, pin_memory=True)
        return host.to(self.key.device, non_blocking=True)

    def _upload(self, rows: list[list[int]]) -> None:
        """The block tables on the device, in their place (steps and captured
        graphs hold the tensor)."""

        width = self.block_tables.shape[1]
        self.block_tables.copy_(self._on_device([row + [-1] * (width - len(row)) for row in rows]))

    def begin(self, new_tokens: Sequence[int]) -> PagedStep:
        """Take pages for ``new_tokens[b]`` more entries of every sequence b
        (0: none this step).  The entries count from here on: a step whose
        appends or attention fail is taken back with :meth:`cancel`."""

        new = [int(n) for n in new_tokens]
        if len(new) != len(self._lengths) or any(n < 0 for n in new):
            raise ValueError("one count of new tokens per sequence")
        after = [length + n for length, n in zip(self._lengths, new)]
        if max(after) > self.max_length:
            raise ValueError(f"a sequence would have {max(after)} entries, the cache holds {self.max_length}")
        more = [-(-a // self.page_size) - len(row) for a, row in zip(after, self._pages)]
        if sum(more) > len(self._free):
            raise ValueError(f"the step needs {sum(more)} pages, {len(self._free)} are free")
        before = self._lengths, self._positions, self._pages
        if sum(more):
            free = iter(reversed(self._free))
            pages = [row + [next(free) for _ in range(n)] for row, n in zip(self._pages, more)]
            self._upload(pages)
            self._pages = pages
            del self._free[-sum(more) :]
        starts = [0]
        for n in new:
            starts.append(starts[-1] + n)
        batch = len(new)
        ints = self._on_device(after + self._positions + starts)
        single = all(n == 1 for n in new)
        self._lengths = after
        self._positions = [p + n for p, n in zip(self._positions, new)]
        step = PagedStep(self.block_tables, ints[:batch], None if single else ints[2 * batch :],
                         ints[batch : 2 * batch], starts[-1], max(new), max(after))
        self._begun = (step.lengths, *before)
        return step

    def cancel(self, step: PagedStep) -> None:
        """Take back ``step``, the latest one, before an eviction or release:
        lengths, positions and pages are again those before it, and its own
        entries' weights 0.  What its attention added to the weights of earlier
        entries stays."""

        if self._begun is None or step.lengths is not self._begun[0]:
            raise ValueError("only the latest step can be taken back, before an eviction or release")
        lengths, positions, pages = self._begun[1:]
        taken = [page for old, now in zip(pages, self._pages) for page in now[len(old) :]]
        if taken:
            self._upload(pages)
        if self.weights is not None:
            for weights in self.weights:
                for b, (old, now) in enumerate(zip(lengths, self._lengths)):
                    if now > old:
                        weights[b, :, old:now].zero_()
        self._free.extend(reversed(taken))
        self._lengths, self._positions, self._pages, self._begun = lengths, positions, pages, None

    def append(self, layer: int, step: PagedStep, key: torch.Tensor, value: torch.Tensor, *,
               rope_theta: float | None = MISTRAL_ROPE_THETA) -> None:
        """The step's packed ``[tokens,KVH,D]`` keys and values into ``layer``'s pages."""

        if key.shape[0] != step.tokens:
            raise ValueError(f"the step has {step.tokens} new tokens, got {key.shape[0]}")
        paged_append(key, value, self.key[layer], self.value[layer], step.block_tables, step.lengths,
                     starts=step.starts, positions=step.positions, rope_theta=rope_theta)

    def attention(self, layer: int, step: PagedStep, query: torch.Tensor, *, window: int | None = MISTRAL_WINDOW,
                  sinks: int = 0, rope_theta: float | None = MISTRAL_ROPE_THETA,
                  scale: float | None = None) -> torch.Tensor:
        """:func:`paged_attention` of the step's packed queries over ``layer``,
        adding to its weights if the cache tracks them."""

        if query.shape[0] != step.tokens:
            raise ValueError(f"the step has {step.tokens} new tokens, got {query.shape[0]}")
        return paged_attention(query, self.key[layer], self.value[layer], step.block_tables, step.lengths,
                               starts=step.starts, positions=step.positions, window=window, sinks=sinks,
                               rope_theta=rope_theta, scale=scale, max_new=step.max_new, max_length=step.max_length,
                               weights=None if self.weights is None else self.weights[layer], accumulate=True)

    def evict(self, budget: int, *, sinks: int = 0, recent: int = 0) -> None:
        """Bring every sequence of more than ``budget`` entries down to it, in
        all layers: the first ``sinks``, the last ``recent`` and those between
        that received most stay.  They move to free pages (what else reads the
        old ones, a shared prompt, is not disturbed) and the old pages are
        freed.  The pages of one sequence's ``budget`` have to be free; where
        those of all do not fit, sequences follow one another into the pages
        that the ones before left."""

        if self.weights is None:
            raise ValueError("the cache does not track weights")
        if budget < 1 or sinks < 0 or recent < 0 or sinks + recent > budget:
            raise ValueError("the budget must be positive and hold the first and the last entries that stay")
        over = [b for b, length in enumerate(self._lengths) if length > budget]
        each = -(-budget // self.page_size)
        if over and each > len(self._free):
            raise ValueError(f"the eviction needs {each} pages, {len(self._free)} are free")
        while over:  # (what a round frees is at least what it takes)
            now = over[: len(self._free) // each]
            self._evict(now, each, budget, sinks, recent)
            over = over[len(now) :]

    def _evict(self, over: list[int], each: int, budget: int, sinks: int, recent: int) -> None:
        taken = self._free[-each * len(over) :]
        pages = list(self._pages)
        for n, b in enumerate(over):
            pages[b] = taken[n * each : (n + 1) * each]
        lengths = self._on_device([self._lengths[b] for b in over])
        rows = self._on_device(over)
        old_tables = self.block_tables.clone()
        try:
            self._upload(pages)
            tables = [t.index_select(0, rows) for t in (old_tables, self.block_tables)]
            moved = []
            for layer, weights in enumerate(self.weights):
                received = weights.index_select(0, rows)
                kept, _ = select_entries(received, lengths, budget, sinks=sinks, recent=recent)
                moved.append(compact_pages(self.key[layer], self.value[layer], tables[0], kept, tables[1],
                                           weights=received))
            rows = rows.long()
        except BaseException:
            self.block_tables.copy_(old_tables)  # nothing is taken: the old pages are as they were
            raise
        self._begun = None
        for weights, left in zip(self.weights, moved):
            weights.index_copy_(0, rows, left)  # in their place: captured graphs hold them
        del self._free[-each * len(over) :]
        for b in over:
            self._free.extend(reversed(self._pages[b]))
            self._lengths[b] = budget
        self._pages = pages

    def release(self, sequence: int) -> None:
        """Drop a sequence: its pages are free and its slot empty."""

        self._begun = None
        self._free.extend(reversed(self._pages[sequence]))
        self._pages[sequence] = []
        self._lengths[sequence] = self._positions[sequence] = 0
        self._upload(self._pages)
        if self.weights is not None:
            for weights in self.weights:
                weights[sequence].zero_()

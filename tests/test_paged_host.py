"""Paged-cache checks that need no GPU: the definitions against one another,
the host's page accounting, and what the C entry points refuse."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

import jointkv_amd as jkv
from jointkv_amd import _lib
from oracle import paged_oracle as ref


def test_attend_is_a_softmax_over_what_is_seen():
    rng = np.random.default_rng(1)
    q, k, v = rng.standard_normal((5, 4, 8)), rng.standard_normal((11, 2, 8)), rng.standard_normal((11, 2, 8))
    got = ref.attend(q, k, v, 30, window=4, sinks=2, theta=100.0)
    turned = ref.rotate(q, 30 + np.arange(5), 100.0)
    for t in range(5):
        at = 6 + t
        seen = [j for j in range(11) if j <= at and (j > at - 4 or j < 2)]
        for h in range(4):
            e = np.exp([turned[t, h] @ k[j, h // 2] / np.sqrt(8) for j in seen])
            want = sum(x * v[j, h // 2] for x, j in zip(e / e.sum(), seen))
            assert np.allclose(got["out"][t, h], want)
            assert np.isclose(got["lse"][t, h], np.log(e.sum()))
    assert np.allclose(got["weights"].sum(), 5 * 4)


def test_rotation_keeps_products_of_equal_distance():
    rng = np.random.default_rng(2)
    a, b = rng.standard_normal((2, 1, 1, 16))
    near = (ref.rotate(a, [7], 10000.0) * ref.rotate(b, [4], 10000.0)).sum()
    far = (ref.rotate(a, [1_000_003], 10000.0) * ref.rotate(b, [1_000_000], 10000.0)).sum()
    assert np.isclose(near, far, rtol=1e-8)


def test_select_prefers_weight_then_the_lower_index():
    w = np.array([0.0, 5.0, 1.0, 1.0, np.nan, 1.0, 0.0, 0.0], dtype=np.float32)
    assert ref.select(w, 4, 1, 1).tolist() == [0, 1, 2, 7]
    assert ref.select(w, 8, 1, 1).tolist() == list(range(8))
    assert ref.select(w, 7, 0, 0).tolist() == [0, 1, 2, 3, 5, 6, 7]


def _attention_call(**overrides):
    args = dict(q=16, qst=512, qsh=128, dtype=0, k=16, v=16, page=4096, head=2048, slot=128, n_pages=4, page_size=16,
                tables=1, tstride=4, twidth=4, lengths=1, starts=None, positions=None, N=2, B=2, QH=4, KVH=2, D=128,
                max_new=1, max_length=64, window=0, sinks=0, theta=10000.0, scale=0.1, out=16, ost=512, osh=128,
                lse=None, weights=None, wsb=0, wsh=0, width=0, accumulate=0, ws=None, ws_bytes=0, stream=None)
    args.update(overrides)
    return _lib.load().jkv_paged_attention(*args.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), b"fp16 or bf16"), (dict(D=96), b"head_dim"), (dict(QH=3), b"multiple"), (dict(B=-1), b"geometry"),
    (dict(N=3), b"one new token"), (dict(page_size=8), b"power of two"), (dict(page_size=48), b"power of two"),
    (dict(page=4097), b"strides"), (dict(page=-4096), b"negative"), (dict(head=-2048), b"negative"), (dict(slot=64), b"strides"), (dict(k=8), b"aligned"), (dict(window=-1), b"negative"),
    (dict(max_new=-1), b"negative"), (dict(sinks=-1), b"negative"), (dict(theta=-2.0), b"rotary"),
    (dict(theta=float("nan")), b"rotary"), (dict(scale=float("nan")), b"scale"), (dict(qst=12), b"multiples of 8"),
    (dict(out=8), b"aligned"), (dict(weights=16, width=10), b"fewer entries"), (dict(lengths=None), b"null"),
    (dict(out=None), b"null"), (dict(weights=16, width=64, wsb=128, wsh=64), b"workspace"), (dict(n_pages=-1), b"page"),
])
def test_attention_refuses_before_the_device_is_touched(change, message):
    # only calls that fail their checks: one that passes would launch
    assert _attention_call(**change) == _lib.JKV_EINVAL
    assert message in _lib.load().jkv_last_error(), _lib.load().jkv_last_error()


def test_workspaces_that_no_memory_holds_are_refused():
    # scores of 2^24 sequences of 2^29 entries: their bytes would wrap
    batch = (1 << 24) - 1
    sizes = dict(N=batch, B=batch, max_length=1 << 29, twidth=1 << 20, page_size=1024,
                 page=1 << 20, head=1 << 17, tstride=0, weights=16, width=1 << 29, wsb=1 << 30, wsh=1 << 29)
    assert _attention_call(**sizes) == _lib.JKV_EINVAL
    assert b"workspace" in _lib.load().jkv_last_error()


@pytest.mark.parametrize("scale", [3e38, -3e38, 1e30, float("inf")])
def test_scales_whose_base_2_form_overflows_are_refused(scale):
    assert _attention_call(scale=scale) == _lib.JKV_EINVAL
    assert b"scale" in _lib.load().jkv_last_error()


@pytest.mark.parametrize("change", [dict(D=0), dict(D=-64), dict(D=256), dict(N=1 << 62), dict(B=1 << 62),
                                    dict(QH=1 << 20), dict(max_length=-1), dict(window=-1), dict(sinks=-1)])
def test_workspaces_of_refused_sizes_are_none(change):
    sizes = dict(N=2, B=2, QH=4, KVH=2, D=128, max_new=1, max_length=4096, window=0, sinks=0, weights=1)
    query = _lib.load().jkv_paged_attention_workspace_bytes
    assert query(*sizes.values()) > 0
    assert query(*{**sizes, **change}.values()) == 0


def test_empty_calls_are_no_ops():
    assert _attention_call(N=0, B=0) == _lib.JKV_OK
    lib = _lib.load()
    assert lib.jkv_paged_append(16, 256, 128, 16, 256, 128, 0, 16, 16, 4096, 2048, 128, 4, 16, 1, 4, 4, 1, None, None, 0,
                                0, 2, 128, 1e4, None) == _lib.JKV_OK
    assert lib.jkv_paged_select(16, 0, 0, 1, 0, 2, 5, 4, 1, 1, 1, 1, None) == _lib.JKV_OK
    assert lib.jkv_paged_compact(16, 16, 0, 4096, 2048, 128, 4, 16, 1, 4, 4, 1, 4, 1, 4, 4, 0, 2, 128, None, 0, 0, 0,
                                 None, None) == _lib.JKV_OK


def test_other_entries_refuse_before_the_device_is_touched():
    lib = _lib.load()
    append = [16, 256, 128, 16, 256, 128, 0, 16, 16, 4096, 2048, 128, 4, 16, 1, 4, 4, 1, None, None, 2, 2, 2, 128, 1e4, None]
    for at, value, message in ((0, None, b"null"), (0, 8, b"aligned"), (1, 100, b"multiples"), (23, 32, b"head_dim"),
                               (24, -1.0, b"rotary"), (13, 17, b"power of two"), (20, 3, b"one new token")):
        call = list(append)
        call[at] = value
        assert lib.jkv_paged_append(*call) == _lib.JKV_EINVAL and message in lib.jkv_last_error()
    for budget, sinks, recent in ((0, 0, 0), (4, 3, 2), (4, 5, 0), (4, -1, 0), (4, 0, -1)):
        assert lib.jkv_paged_select(16, 8, 4, 1, 2, 2, 4, budget, sinks, recent, 1, 1, None) == _lib.JKV_EINVAL
    assert lib.jkv_paged_select(16, 8, 4, 1, 2, 2, 4, 2, 0, 0, None, 1, None) == _lib.JKV_EINVAL
    assert lib.jkv_paged_compact(16, 16, 0, 4096, 2048, 128, 4, 16, 1, 4, 4, None, 4, 1, 4, 4, 2, 2, 128, None, 0, 0, 0,
                                 None, None) == _lib.JKV_EINVAL


def test_copies_that_pass_32_bits_of_threads_are_refused():
    assert _lib.load().jkv_paged_compact(16, 16, 0, 4096, 2048, 128, 4, 16, 1, 4, 4, 1, (1 << 30) - 1, 1, 4, 4, 1, 2, 128,
                                         None, 0, 0, 0, None, None) == _lib.JKV_EINVAL
    assert b"grid" in _lib.load().jkv_last_error()


def test_operators_refuse_cpu_tensors():
    pages = torch.zeros(4, 2, 16, 64, dtype=torch.float16)
    ints = torch.zeros(2, 4, dtype=torch.int32)
    lengths = torch.ones(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="MI355X"):
        jkv.paged_attention(torch.zeros(2, 2, 64, dtype=torch.float16), pages, pages, ints, lengths)
    with pytest.raises(ValueError, match="MI355X"):
        jkv.paged_append(torch.zeros(2, 2, 64, dtype=torch.float16), torch.zeros(2, 2, 64, dtype=torch.float16), pages,
                         pages, ints, lengths)
    with pytest.raises(ValueError, match="MI355X"):
        jkv.select_entries(torch.zeros(2, 2, 8), lengths, 4)
    with pytest.raises(ValueError, match="MI355X"):
        jkv.compact_pages(pages, pages, ints, torch.zeros(2, 2, 4, dtype=torch.int32), ints)


@pytest.mark.parametrize("make", [
    lambda: torch.arange(2 * 3 * 64 + 1).half()[1:].view(2, 3, 64), lambda: torch.zeros(2, 3, 65).half()[:, :, 1:],
    lambda: torch.zeros(3, 2, 64).half().transpose(0, 1), lambda: torch.zeros(2, 64, 3).half().transpose(1, 2),
    lambda: torch.zeros(2, 3, 68).half()[:, :, :64], lambda: torch.zeros(1, 64).half().expand(2, 3, 64)])
def test_rows_are_aligned_or_copied(make):
    rows = make()
    got = jkv.paged._rows(rows)
    t, h, d = got.stride()
    assert got.data_ptr() % 16 == 0 and d == 1 and t % 8 == 0 and h % 8 == 0
    assert torch.equal(got, rows)


class _HostCache(jkv.PagedKVCache):
    def _on_device(self, values):
        return torch.tensor(values, dtype=torch.int32)


def test_page_accounting():
    cache = _HostCache(1, 3, 10, 1, max_length=100, page_size=16, head_dim=64, device="cpu")
    step = cache.begin([33, 1, 0])
    assert cache.free_pages == 6 and step.tokens == 34 and step.max_new == 33 and step.max_length == 33
    assert step.starts.tolist() == [0, 33, 34, 34] and step.positions.tolist() == [0, 0, 0]
    assert step.lengths.tolist() == [33, 1, 0]
    pages = step.block_tables.tolist()
    assert [sum(p >= 0 for p in row) for row in pages] == [3, 1, 0]
    assert len({p for row in pages for p in row if p >= 0}) == 4
    step = cache.begin([1, 1, 1])
    assert step.starts is None and cache.free_pages == 5 and step.positions.tolist() == [33, 1, 0]
    with pytest.raises(ValueError, match="are free"):
        cache.begin([0, 0, 99])
    with pytest.raises(ValueError, match="holds 100"):
        cache.begin([0, 0, 100])
    with pytest.raises(ValueError, match="one count"):
        cache.begin([1, 1])
    assert cache.lengths == (34, 2, 1) and cache.free_pages == 5, "a refused step changes nothing"
    with pytest.raises(ValueError, match="does not track"):
        cache.evict(4)
    cache.release(0)
    assert cache.lengths == (0, 2, 1) and cache.free_pages == 8 and cache.positions == (0, 2, 1)


def _plain_eviction(monkeypatch, seen):
    """Selection and compaction in plain form (the oracle's choice), for caches
    on the host; ``seen`` collects the rows of each call."""

    def select_entries(weights, lengths, budget, *, sinks, recent):
        kept = torch.full((*weights.shape[:2], budget), -1, dtype=torch.int32)
        for b, length in enumerate(lengths.tolist()):
            for h in range(weights.shape[1]):
                stay = ref.select(weights[b, h, :length].numpy(), budget, sinks, recent)
                kept[b, h, : len(stay)] = torch.from_numpy(stay).int()
        return kept, lengths.clamp(max=budget)

    def compact_pages(key, value, tables, kept, new_tables, *, weights):
        seen.append(tables.shape[0])
        size, moved = key.shape[2], torch.zeros_like(weights)
        for pool in (key, value):
            before = pool.clone()
            for b, h, j in (kept >= 0).nonzero().tolist():
                e = int(kept[b, h, j])
                pool[new_tables[b, j // size], h, j % size] = before[tables[b, e // size], h, e % size]
                moved[b, h, j] = weights[b, h, e]
        return moved

    monkeypatch.setattr(jkv.paged, "select_entries", select_entries)
    monkeypatch.setattr(jkv.paged, "compact_pages", compact_pages)


def _filled(pages, lengths):
    """A cache on the host whose entries hold their sequence and index."""

    cache = _HostCache(2, len(lengths), pages, 2, max_length=100, page_size=16, head_dim=64, track_weights=True,
                       device="cpu")
    cache.key.zero_()
    cache.value.zero_()
    cache.begin(lengths)
    gen = torch.Generator().manual_seed(len(lengths))
    for layer in range(2):
        for b, length in enumerate(lengths):
            cache.weights[layer][b, :, :length] = torch.rand(2, length, generator=gen)
            for j in range(length):
                page = cache.block_tables[b, j // 16]
                cache.key[layer][page, :, j % 16] = 1000 * b + j
                cache.value[layer][page, :, j % 16] = -1000 * b - j
    return cache


def _entries(cache, layer, b):
    """Keys, values and weights of a sequence: [KVH, length] each (one dim stands for all)."""

    length = cache.lengths[b]
    pages = cache.block_tables[b, : -(-length // 16)].long()
    k, v = (pool[layer][pages].transpose(0, 1).reshape(2, -1, 64)[:, :length, 0] for pool in (cache.key, cache.value))
    return k, v, cache.weights[layer][b, :, :length].clone()


@pytest.mark.parametrize("spare", [2, 3, 4, 20])
def test_eviction_touches_only_sequences_over_the_budget_and_reuses_pages(monkeypatch, spare):
    """With pages for one sequence's budget free, or more: the same entries
    stay, the others' pages and weights are not passed on at all."""

    seen = []
    _plain_eviction(monkeypatch, seen)
    lengths = [70, 20, 33, 97, 0]
    cache = _filled(5 + 2 + 3 + 7 + spare, lengths)
    before = [[_entries(cache, layer, b) for b in range(5)] for layer in range(2)]
    pages = cache.block_tables.clone()
    cache.evict(30, sinks=2, recent=8)
    assert cache.lengths == (30, 20, 30, 30, 0) and cache.positions == tuple(lengths)
    assert cache.free_pages == 5 + 2 + 3 + 7 + spare - 4 * 2
    assert sum(seen) == 2 * 3, "rows of sequences within the budget were passed on"
    table = cache.block_tables.tolist()
    used = [p for row in table for p in row if p >= 0]
    assert len(set(used)) == len(used) == 8 and not set(used) & set(cache._free)
    assert torch.equal(cache.block_tables[1], pages[1])
    for layer in range(2):
        for b, length in enumerate(lengths):
            for h in range(2):
                k, v, w = (x[h] for x in before[layer][b])
                stay = torch.from_numpy(ref.select(w.numpy(), 30, 2, 8))
                for got, want in zip(_entries(cache, layer, b), (k, v, w)):
                    assert torch.equal(got[h], want[stay])
                assert bool((cache.weights[layer][b, h, len(stay) :] == 0).all())


def test_eviction_without_pages_for_one_budget_is_refused(monkeypatch):
    _plain_eviction(monkeypatch, [])
    cache = _filled(5 + 7 + 1, [70, 97])
    before, weights = cache.block_tables.clone(), cache.weights[0].clone()
    with pytest.raises(ValueError, match="needs 2 pages, 1 are free"):
        cache.evict(30)
    assert cache.lengths == (70, 97) and cache.free_pages == 1
    assert torch.equal(cache.block_tables, before) and torch.equal(cache.weights[0], weights)


def test_an_eviction_that_fails_leaves_the_cache_as_it_was(monkeypatch):
    _plain_eviction(monkeypatch, [])
    cache = _filled(5 + 7 + 4, [70, 97])
    before, weights = cache.block_tables.clone(), [w.clone() for w in cache.weights]
    entries = [_entries(cache, 1, b) for b in range(2)]
    plain, calls = jkv.paged.select_entries, []

    def failing(*args, **kwargs):
        calls.append(1)
        if len(calls) == 2:
            raise RuntimeError("second layer")
        return plain(*args, **kwargs)

    monkeypatch.setattr(jkv.paged, "select_entries", failing)
    with pytest.raises(RuntimeError, match="second layer"):
        cache.evict(30)
    assert cache.lengths == (70, 97) and cache.free_pages == 4 and torch.equal(cache.block_tables, before)
    assert all(torch.equal(a, b) for a, b in zip(cache.weights, weights))
    for b in range(2):
        assert all(torch.equal(x, y) for x, y in zip(entries[b], _entries(cache, 1, b)))


def test_a_step_that_failed_is_taken_back(monkeypatch):
    _plain_eviction(monkeypatch, [])
    cache = _filled(20, [40, 16, 0])
    tables, weights = cache.block_tables.clone(), [w.clone() for w in cache.weights]
    state = cache.lengths, cache.positions, cache.free_pages, list(cache._free)
    step = cache.begin([30, 1, 2])
    assert cache.lengths == (70, 17, 2) and cache.free_pages == 20 - 5 - 2 - 1
    with pytest.raises(ValueError, match="33 new tokens"):
        cache.append(0, step, torch.zeros(32, 2, 64), torch.zeros(32, 2, 64))
    for w in cache.weights:  # a layer's attention before the failure
        w[0, :, 40:70] = 3.0
    cache.cancel(step)
    assert (cache.lengths, cache.positions, cache.free_pages, cache._free) == state
    assert torch.equal(cache.block_tables, tables)
    assert all(torch.equal(a, b) for a, b in zip(cache.weights, weights))
    with pytest.raises(ValueError, match="latest step"):
        cache.cancel(step)
    # the same step again finds what the first one found
    again = cache.begin([30, 1, 2])
    for name in ("block_tables", "lengths", "starts", "positions"):
        assert torch.equal(getattr(again, name), getattr(step, name))
    with pytest.raises(ValueError, match="latest step"):
        cache.cancel(step)
    cache.cancel(dataclasses.replace(again, max_length=100))
    assert (cache.lengths, cache.positions, cache.free_pages, cache._free) == state
    for end in (lambda: cache.release(1), lambda: cache.evict(30)):
        step = cache.begin([1, 0, 0])
        end()
        with pytest.raises(ValueError, match="before an eviction or release"):
            cache.cancel(step)


@pytest.mark.parametrize("change", [dict(layers=0), dict(head_dim=32), dict(page_size=24), dict(page_size=8),
                                    dict(dtype=torch.float32), dict(max_length=0)])
def test_cache_refuses_geometry(change):
    args = dict(layers=1, sequences=1, pages=2, kv_heads=1, max_length=32, device="cpu")
    args.update(change)
    with pytest.raises(ValueError):
        jkv.PagedKVCache(**args)


def test_a_call_without_tokens_checks_what_it_reads():
    # it stores zero weights below the lengths
    assert _attention_call(N=0, starts=1, lengths=None, weights=16, wsb=128, wsh=64, width=64) == _lib.JKV_EINVAL
    assert b"null" in _lib.load().jkv_last_error()
    assert _attention_call(N=0, starts=1, lengths=None) == _lib.JKV_OK
    assert _attention_call(N=0, starts=1, lengths=None, weights=16, wsb=128, wsh=64, width=64, accumulate=1) == _lib.JKV_OK

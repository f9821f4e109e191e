"""Checks of rotary rules, packed and shaped attention, copied pages and forked
sequences that need no GPU: the definitions against one another and against
differences, what is refused, the host's page accounting."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

import jointkv_amd as jkv
from jointkv_amd import _lib
from oracle import shaped_oracle as ref


def test_shaped_attention_is_a_softmax_over_what_is_seen():
    gen = torch.Generator().manual_seed(1)
    q, k, v = (torch.randn(n, h, 8, generator=gen, dtype=torch.float64) for n, h in ((5, 4), (9, 2), (9, 2)))
    slopes = [0.5, 0.1, 0.0, -0.2]
    got = ref.attend(q, k, v, window=4, sinks=1, prefix=7, cap=1.5, slopes=slopes)
    for t in range(5):
        i = 4 + t
        seen = [j for j in range(9) if (j <= i or j < 7) and (j > i - 4 or j < 1)]
        for h in range(4):
            x = [1.5 * math.tanh(float(q[t, h] @ k[j, h // 2]) / math.sqrt(8) / 1.5) - slopes[h] * abs(i - j) for j in seen]
            e = [math.exp(s) for s in x]
            want = sum(w * v[j, h // 2] for w, j in zip(e, seen)) / sum(e)
            assert torch.allclose(got["out"][t, h], want)
            assert math.isclose(got["lse"][t, h], math.log(sum(e)))
    assert math.isclose(float(got["weights"].sum()), 5 * 4)


@pytest.mark.parametrize("form", [dict(), dict(cap=0.7), dict(slopes=[0.3, 0.05]), dict(prefix=5), dict(window=3, sinks=1, cap=2.0)])
def test_gradients_are_the_formulas_and_the_differences(form):
    gen = torch.Generator().manual_seed(2)
    q, k, v, d = (torch.randn(7, h, 6, generator=gen, dtype=torch.float64) for h in (2, 1, 1, 2))
    got = ref.attend(q, k, v, d_out=d, **form)
    for name, x in (("dq", q), ("dk", k), ("dv", v)):
        flat = x.view(-1)
        for at in range(0, flat.numel(), 5):
            old = float(flat[at])
            values = []
            for step in (1e-6, -1e-6):
                flat[at] = old + step
                values.append(float((ref.attend(q, k, v, **form)["out"] * d).sum()))
            flat[at] = old
            assert math.isclose((values[0] - values[1]) / 2e-6, float(got[name].view(-1)[at]), rel_tol=1e-5, abs_tol=1e-8)


@pytest.mark.parametrize("rule,args", [
    (dict(), dict()), (dict(dims=20), dict()), (dict(theta=500000.0), dict()),
    (dict(scaling="linear", factor=8.0), dict(scaling="linear", factor=8.0)),
    (dict(scaling="base", factor=4.0), dict(scaling="base", factor=4.0)),
    (dict(scaling="parts", factor=8.0, original_length=8192), dict(scaling="parts", factor=8.0, original=8192)),
    (dict(scaling="parts", factor=0.5, original_length=100, low=0.0, high=2.0), dict(scaling="parts", factor=0.5, original=100, low=0.0, high=2.0)),
])
def test_rates(rule, args):
    made = jkv.RotaryRule(**rule)
    dims = made.dims or 64
    got = made.rates(64)
    want = ref.rates(dims, made.theta, **args)
    assert len(got) == dims // 2 and all(math.isclose(a, b, rel_tol=1e-12) for a, b in zip(got, want))


def test_scalings_do_what_they_say():
    plain, linear = jkv.RotaryRule().rates(128), jkv.RotaryRule(scaling="linear", factor=4.0).rates(128)
    assert all(math.isclose(a, 4 * b) for a, b in zip(plain, linear))
    base = jkv.RotaryRule(scaling="base", factor=4.0).rates(128)
    assert base[0] == plain[0] and math.isclose(base[-1] * 4, plain[-1], rel_tol=1e-12)
    parts = jkv.RotaryRule(scaling="parts", factor=4.0, original_length=2048, low=1.0, high=4.0).rates(128)
    for a, b in zip(plain, parts):
        turns = 2048 * a / (2 * math.pi)
        assert math.isclose(b, a) if turns >= 4 else math.isclose(b, a / 4) if turns <= 1 else a / 4 < b < a


@pytest.mark.parametrize("change", [
    dict(theta=0.0), dict(theta=-1.0), dict(theta=float("inf")), dict(layout="pairs"), dict(dims=0), dict(dims=7),
    dict(dims=258), dict(scaling="ntk"), dict(scaling="linear", factor=0.0), dict(factor=2.0),
    dict(scaling="parts", factor=2.0), dict(scaling="parts", factor=2.0, original_length=10, low=4.0, high=4.0),
    dict(magnitude=float("nan"))])
def test_rules_that_make_no_sense_are_refused(change):
    with pytest.raises(ValueError):
        jkv.RotaryRule(**change)


def test_rules_that_do_not_fit_a_head_are_refused():
    with pytest.raises(ValueError, match="at most the head"):
        jkv.RotaryRule(dims=128).rates(64)
    with pytest.raises(ValueError, match="one pair"):
        jkv.RotaryRule(dims=2, scaling="base", factor=2.0).rates(64)
    with pytest.raises(ValueError, match="64 bits"):
        jkv.RotaryRule(dims=4, scaling="base", factor=1e200).rates(64)


ints = lambda *v: torch.tensor(v, dtype=torch.int32)


@pytest.mark.parametrize("change,message", [
    (dict(query=torch.zeros(4, 2, 64, dtype=torch.float64)), "fp16"), (dict(query=torch.zeros(4, 128)), "fp16"),
    (dict(query=torch.zeros(4, 2, 63)), "even"), (dict(query=torch.zeros(4, 2, 258)), "even"),
    (dict(key=torch.zeros(3, 2, 64)), "keys"), (dict(key=torch.zeros(4, 2, 64).half()), "keys"),
    (dict(key_out=torch.zeros(4, 2, 64)), "without keys"), (dict(starts=torch.zeros(3)), "starts"),
    (dict(starts=ints()), "starts"), (dict(positions=ints(1, 2)), "positions"),
    (dict(positions=torch.zeros(4)), "positions"), (dict(starts=ints(0, 4), positions=ints(1, 2)), "positions"),
    (dict(), "HIP"),
])
def test_rotary_refuses(change, message):
    args = dict(query=torch.zeros(4, 2, 64))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        jkv.rotary(args.pop("query"), args.pop("key", None), **args)


def test_given_outputs_are_not_differentiable():
    x = torch.zeros(4, 2, 64, requires_grad=True)
    with pytest.raises(ValueError, match="differentiable"):
        jkv.rotary(x, out=torch.zeros(4, 2, 64))


@pytest.mark.parametrize("change,message", [
    (dict(query=torch.zeros(6, 4, 64)), "fp16 or bf16"), (dict(key=torch.zeros(5, 2, 64).half()), "rows and dims"),
    (dict(key=torch.zeros(6, 2, 64).bfloat16(), value=torch.zeros(6, 2, 64).bfloat16()), "one type"),
    (dict(key=torch.zeros(6, 3, 64).half(), value=torch.zeros(6, 3, 64).half()), "multiple"),
    (dict(key=torch.zeros(6, 0, 64).half(), value=torch.zeros(6, 0, 64).half()), "multiple"),
    (dict(starts=torch.zeros(3)), "starts"), (dict(window=0), "window"), (dict(sinks=-1), "sinks"),
    (dict(softcap=0.0), "cap"), (dict(softcap=float("nan")), "cap"), (dict(softcap=2000.0), "cap"),
    (dict(slopes=torch.zeros(3)), "slopes"), (dict(slopes=torch.zeros(4).half()), "slopes"),
    (dict(slopes=torch.zeros(4, requires_grad=True)), "gradient"), (dict(prefixes=ints(1)), "prefixes"),
    (dict(prefixes=torch.zeros(2)), "prefixes"), (dict(lse=torch.zeros(6, 4).half()), "lse"),
    (dict(out=torch.zeros(6, 4, 64)), "out"), (dict(out=torch.zeros(6, 1, 64).half().expand(6, 4, 64)), "overlap"), (dict(), "HIP"),
])
def test_packed_attention_refuses(change, message):
    args = dict(query=torch.zeros(6, 4, 64).half(), key=torch.zeros(6, 2, 64).half(), value=torch.zeros(6, 2, 64).half(),
                starts=ints(0, 2, 6))
    args.update(change)
    with pytest.raises(ValueError, match=message):
        jkv.packed_attention(args.pop("query"), args.pop("key"), args.pop("value"), args.pop("starts"), **args)


def test_paged_shapes_are_refused():
    pages = torch.zeros(4, 2, 16, 64).half()
    args = (torch.zeros(2, 4, 64).half(), pages, pages, torch.zeros(2, 4, dtype=torch.int32), ints(5, 6))
    with pytest.raises(ValueError, match="HIP"):
        jkv.paged_attention(*args, softcap=30.0)
    with pytest.raises(ValueError, match="HIP"):
        jkv.copy_pages(pages, pages, ints(0), ints(1))


def _packed_call(**overrides):
    args = dict(q=16, qst=256, qsh=64, k=16, kst=128, ksh=64, v=16, vst=128, vsh=64, dtype=0, starts=16, prefixes=None, N=6,
                B=2, QH=4, KVH=2, D=64, window=0, sinks=0, scale=0.125, softcap=0.0, slopes=None, out=16, ost=256, osh=64,
                lse=None, rest=None, stream=None)
    args.update(overrides)
    return _lib.load().jkv_packed_attention(*args.values())


def _backward_call(**overrides):
    args = dict(q=16, qst=256, qsh=64, k=16, kst=128, ksh=64, v=16, vst=128, vsh=64, o=16, ost=256, osh=64, rest=None, d=16,
                dst=256, dsh=64, lse=16, dtype=0, starts=16, prefixes=None, N=6, B=2, QH=4, KVH=2, D=64, window=0, sinks=0,
                scale=0.125, softcap=0.0, slopes=None, dq=16, dk=16, dv=16, ws=16, ws_bytes=0, stream=None)
    args.update(overrides)
    return _lib.load().jkv_packed_attention_backward(*args.values())


PACKED = [(dict(dtype=2), b"fp16 or bf16"), (dict(D=96), b"head_dim"), (dict(QH=3), b"multiple"), (dict(KVH=0), b"multiple"),
          (dict(N=-1), b"rows"), (dict(N=1 << 30), b"rows"), (dict(B=-1), b"rows"), (dict(N=1 << 29, QH=8), b"rows"),
          (dict(window=-1), b"window"), (dict(sinks=-1), b"window"), (dict(scale=float("nan")), b"scale"),
          (dict(scale=1e30), b"scale"), (dict(softcap=-1.0), b"cap"), (dict(softcap=1e-4), b"cap"),
          (dict(softcap=float("inf")), b"cap"), (dict(softcap=float("nan")), b"cap"), (dict(qst=12), b"strides"), (dict(kst=1 << 22), b"strides"),
          (dict(vsh=-64), b"strides"), (dict(q=None), b"null"), (dict(starts=None), b"null"), (dict(k=8), b"aligned")]


@pytest.mark.parametrize("change,message", PACKED + [(dict(out=None), b"null"), (dict(rest=8), b"aligned")])
def test_packed_entry_refuses_before_the_device_is_touched(change, message):
    assert _packed_call(**change) == _lib.JKV_EINVAL
    assert message in _lib.load().jkv_last_error(), _lib.load().jkv_last_error()


@pytest.mark.parametrize("change,message", PACKED + [
    (dict(), b"workspace"), (dict(lse=None), b"null"), (dict(d=None), b"null"), (dict(dk=8), b"aligned"),
    (dict(ws=None, ws_bytes=1 << 30), b"workspace"), (dict(ws=8, ws_bytes=1 << 30), b"workspace")])
def test_backward_entry_refuses_before_the_device_is_touched(change, message):
    assert _backward_call(**change) == _lib.JKV_EINVAL
    assert message in _lib.load().jkv_last_error(), _lib.load().jkv_last_error()


def test_empty_calls_are_no_ops_and_refused_sizes_need_no_workspace():
    assert _packed_call(N=0) == _lib.JKV_OK and _backward_call(N=0) == _lib.JKV_OK
    size = _lib.load().jkv_packed_backward_workspace_bytes
    good = dict(N=100, B=2, QH=8, KVH=2, D=128, window=0)
    assert size(*good.values()) >= 2 * 100 * 8 * 4
    for change in (dict(N=0), dict(N=1 << 62), dict(B=-1), dict(QH=7), dict(KVH=0), dict(D=96), dict(window=-1), dict(QH=1 << 20)):
        assert size(*{**good, **change}.values()) == 0
    # heads in splits keep their sums
    assert size(8192, 1, 32, 8, 128, 0) > 2 * 2 * 8192 * 8 * 128 * 4


def _rotary_call(**overrides):
    rates = (ctypes.c_double * 32)(*([0.5] * 32))
    args = dict(q=16, qst=256, qsh=64, qo=16, qost=256, qosh=64, QH=4, k=16, kst=128, ksh=64, ko=16, kost=128, kosh=64, KVH=2,
                dtype=0, N=6, D=64, dims=64, side=0, rates=rates, magnitude=1.0, inverse=0, starts=None, B=0, positions=None,
                stream=None)
    args.update(overrides)
    return _lib.load().jkv_rotary(*args.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=3), b"fp16"), (dict(D=63), b"head dims"), (dict(D=258), b"head dims"), (dict(D=0), b"head dims"),
    (dict(dims=66), b"turned"), (dict(dims=0), b"turned"), (dict(dims=31), b"turned"), (dict(N=-1), b"rows"),
    (dict(B=-1), b"rows"), (dict(QH=0, KVH=0), b"heads"), (dict(QH=-1), b"heads"), (dict(QH=1 << 16), b"heads"),
    (dict(rates=None), b"null"), (dict(magnitude=float("inf")), b"magnitude"), (dict(q=None), b"null"),
    (dict(ko=None), b"null"), (dict(q=17), b"aligned"), (dict(rates=(ctypes.c_double * 32)(*([float("nan")] * 32))), b"rates")])
def test_rotary_entry_refuses_before_the_device_is_touched(change, message):
    assert _rotary_call(**change) == _lib.JKV_EINVAL
    assert message in _lib.load().jkv_last_error(), _lib.load().jkv_last_error()


def test_rotary_of_no_rows():
    assert _rotary_call(N=0, q=None, qo=None, k=None, ko=None) == _lib.JKV_OK


def _copy_call(**overrides):
    args = dict(k=16, v=16, dtype=0, layers=2, layer=1 << 16, page=4096, head=2048, slot=128, n_pages=4, size=16, KVH=2, D=128,
                src=16, dst=16, entries=None, pairs=3, stream=None)
    args.update(overrides)
    return _lib.load().jkv_paged_copy(*args.values())


@pytest.mark.parametrize("change,message", [
    (dict(dtype=2), b"fp16"), (dict(D=96), b"head_dim"), (dict(size=24), b"power of two"), (dict(layers=-1), b"layers"),
    (dict(layers=1 << 16), b"layers"), (dict(layer=12), b"layers"), (dict(layer=-8), b"layers"), (dict(pairs=-1), b"pages"),
    (dict(pairs=1 << 24), b"pages"), (dict(src=None), b"null"), (dict(dst=None), b"null"), (dict(k=8), b"aligned"),
    (dict(page=4100), b"strides"), (dict(size=4096, KVH=60000), b"large"), (dict(size=4096, KVH=8192, pairs=1 << 20), b"grid")])
def test_copy_entry_refuses_before_the_device_is_touched(change, message):
    assert _copy_call(**change) == _lib.JKV_EINVAL
    assert message in _lib.load().jkv_last_error(), _lib.load().jkv_last_error()


def test_copies_of_nothing():
    assert _copy_call(pairs=0) == _lib.JKV_OK and _copy_call(layers=0) == _lib.JKV_OK and _copy_call(n_pages=0) == _lib.JKV_OK


class _HostCache(jkv.PagedKVCache):
    """Page accounting without a device: copies of pages are made on the CPU."""

    def _on_device(self, values):
        return torch.tensor(values, dtype=torch.int32)


@pytest.fixture
def copies(monkeypatch):
    made = []

    def copy_pages(key, value, sources, targets, *, entries=None):
        made.append(list(zip(sources.tolist(), targets.tolist(), entries.tolist())))
        for s, d, n in made[-1]:
            key[:, d, :, :n] = key[:, s, :, :n]

    monkeypatch.setattr(jkv.paged, "copy_pages", copy_pages)
    return made


def cache_of(**change):
    args = dict(layers=2, sequences=4, pages=12, kv_heads=1, max_length=100, page_size=16, head_dim=64, device="cpu")
    args.update(change)
    return _HostCache(args.pop("layers"), args.pop("sequences"), args.pop("pages"), args.pop("kv_heads"), **args)


def listed(cache):
    """Pages that the tables list, and how often: what the accounting must hold."""

    count = [0] * len(cache._uses)
    for row, pages, length in zip(cache.block_tables.tolist(), cache._pages, cache.lengths):
        assert row[: len(pages)] == pages and set(row[len(pages) :]) <= {-1} and len(pages) == -(-length // cache.page_size)
        for page in pages:
            count[page] += 1
    assert count == cache._uses
    assert sorted(cache._free) == [p for p, n in enumerate(count) if not n]


def test_a_fork_shares_and_a_write_copies(copies):
    cache = cache_of()
    cache.begin([40, 0, 0, 0])
    cache.fork(0, 1)
    cache.fork(0, 2, 33)
    cache.fork(0, 3, 32)
    listed(cache)
    assert cache.free_pages == 9 and not copies and cache.positions == (40, 40, 33, 32)
    third = cache._pages[0][2]
    cache.begin([1, 1, 1, 0])
    listed(cache)
    # all but the last of the sharers of the half-written page copied what it holds
    assert copies == [[(third, cache._pages[0][2], 8), (third, cache._pages[1][2], 8)]] and cache._pages[2][2] == third
    cache.begin([1, 1, 1, 1])
    listed(cache)
    assert len(copies) == 1 and cache.lengths == (42, 42, 35, 33)
    cache.release(0)
    listed(cache)
    cache.release(1)
    cache.release(2)
    cache.release(3)
    assert cache.free_pages == 12


def test_a_whole_page_is_shared_for_good(copies):
    cache = cache_of()
    cache.begin([32, 0, 0, 0])
    cache.fork(0, 1)
    cache.begin([1, 1, 0, 0])
    listed(cache)
    assert not copies and cache._pages[0][:2] == cache._pages[1][:2] and cache._pages[0][2] != cache._pages[1][2]


def test_a_step_that_copied_is_taken_back(copies):
    cache = cache_of()
    cache.begin([20, 5, 0, 0])
    cache.fork(0, 2)
    before = [list(x) for x in cache._pages], list(cache._free), list(cache._uses), cache.lengths, cache.block_tables.clone()
    for _ in range(2):
        step = cache.begin([20, 1, 3, 0])
        listed(cache)
        assert copies
        cache.cancel(step)
        listed(cache)
        assert before[:4] == ([list(x) for x in cache._pages], cache._free, cache._uses, cache.lengths)
        assert torch.equal(before[4], cache.block_tables)


def test_forks_that_are_refused(copies):
    cache = cache_of(pages=4)
    cache.begin([20, 3, 0, 0])
    for args, message in (((0, 0), "empty"), ((0, 1), "empty"), ((0, 2, 21), "up to 20"), ((0, 2, -1), "up to 20")):
        with pytest.raises(ValueError, match=message):
            cache.fork(*args)
    cache._positions = [50, 3, 0, 0]  # (as an eviction leaves them)
    with pytest.raises(ValueError, match="evicted"):
        cache.fork(0, 2, 10)
    cache.fork(0, 2)
    assert cache.positions[2] == 50
    cache.fork(0, 3, 20)
    cache.release(1)
    state = [list(x) for x in cache._pages], list(cache._free), list(cache._uses)
    with pytest.raises(ValueError, match="needs 3 pages, 2 are free"):
        cache.begin([1, 0, 1, 13])  # two copies and a new page
    assert state == ([list(x) for x in cache._pages], cache._free, cache._uses)
    listed(cache)
    step = cache.begin([0, 0, 1, 0])
    cache.fork(2, 1)
    with pytest.raises(ValueError, match="latest"):
        cache.cancel(step)


def test_a_fork_of_nothing_and_its_weights(copies):
    cache = cache_of(track_weights=True)
    cache.fork(0, 1)
    assert cache.lengths == (0, 0, 0, 0) and cache.free_pages == 12
    cache.begin([20, 0, 0, 0])
    for w in cache.weights:
        w[0, :, :20] = torch.arange(20.0)
    cache.fork(0, 2, 7)
    for w in cache.weights:
        assert w[2, 0, :7].tolist() == list(range(7)) and not w[2, 0, 7:].any()


def test_an_eviction_of_shared_pages_counts_what_it_frees(copies, monkeypatch):
    monkeypatch.setattr(jkv.paged, "select_entries", lambda w, n, budget, **_: (torch.zeros(len(n), 1, budget, dtype=torch.int32), n))
    monkeypatch.setattr(jkv.paged, "compact_pages", lambda k, v, old, kept, new, weights: weights.clone())
    cache = cache_of(track_weights=True, pages=9)
    cache.begin([96, 0, 0, 0])  # six pages, three are free
    cache.fork(0, 1)
    cache.fork(0, 2)
    state = [list(x) for x in cache._pages], list(cache._free), list(cache._uses), cache.lengths
    with pytest.raises(ValueError, match="needs 2 pages, 1 are free"):
        cache.evict(32)  # the first to move frees nothing: the others still read its pages
    assert state == ([list(x) for x in cache._pages], cache._free, cache._uses, cache.lengths)
    cache.evict(16)
    listed(cache)
    assert cache.lengths == (16, 16, 16, 0) and cache.free_pages == 6


def test_distances_and_prefixes_after_an_eviction_are_refused(copies):
    cache = cache_of()
    step = cache.begin([20, 0, 0, 0])
    cache._positions = [25, 0, 0, 0]
    for form in (dict(slopes=torch.zeros(2)), dict(prefixes=ints(0, 0, 0, 0))):
        with pytest.raises(ValueError, match="evicted"):
            cache.attention(0, step, torch.zeros(20, 2, 64).half(), **form)


def rows_of(cache, sequence):
    """A sequence's stored keys of all layers, entry after entry (the copies made on the
    CPU are of keys)."""

    at = [(page, slot) for page in cache._pages[sequence] for slot in range(cache.page_size)][: cache.lengths[sequence]]
    return torch.stack([cache.key[:, page, 0, slot] for page, slot in at])


def write(cache, step, before, marks):
    """What a step's appends do: sequence b's new rows, all of the number ``marks[b]``."""

    tables = step.block_tables.tolist()
    for b, (old, now) in enumerate(zip(before, cache.lengths)):
        for j in range(old, now):
            cache.key[:, tables[b][j // cache.page_size], :, j % cache.page_size] = marks[b]


@pytest.mark.parametrize("order", [(0, 1, 2), (2, 1, 0), (1, 2, 0), (2, 0, 1)])
@pytest.mark.parametrize("new", [(1, 1, 1), (9, 1, 4), (1, 14, 2), (1, 1, 0), (0, 3, 1)])
def test_a_cancelled_step_leaves_the_entries_of_all_sharers(copies, order, new):
    """A prompt's owner and forks of parts of it, in every order of their lengths:
    what a step wrote before it was taken back is nobody's."""

    owner, part, less = order
    cache = cache_of(dtype=torch.bfloat16)
    cache.key.zero_()
    count = [0, 0, 0, 0]
    count[owner] = 40
    cache.begin(count)
    for j in range(40):
        cache.key[:, cache._pages[owner][j // 16], :, j % 16] = 100 + j
    cache.fork(owner, part, 35)
    cache.fork(owner, less, 33)
    held = [rows_of(cache, b).clone() for b in range(3)]
    lengths = cache.lengths
    for _ in range(2):
        step = cache.begin([*new, 0])
        listed(cache)
        write(cache, step, lengths, [1, 2, 3, 0])
        for b in range(3):  # each has its own rows behind what it had
            rows = rows_of(cache, b)
            assert torch.equal(rows[: lengths[b]], held[b]) and (rows[lengths[b] :] == b + 1).all()
        cache.cancel(step)
        listed(cache)
        assert cache.lengths == lengths
        for b in range(3):
            assert torch.equal(rows_of(cache, b), held[b]), b
    # and taken up again
    step = cache.begin([*new, 0])
    write(cache, step, lengths, [1, 2, 3, 0])
    for b in range(3):
        rows = rows_of(cache, b)
        assert torch.equal(rows[: lengths[b]], held[b]) and (rows[lengths[b] :] == b + 1).all()


@pytest.mark.parametrize("private", [0, 2])
def test_an_eviction_begins_with_what_frees_pages(copies, monkeypatch, private):
    """Sharers of a prompt beside a sequence with pages of its own, two pages free: the
    latter's move makes room for the others', whatever their order."""

    monkeypatch.setattr(jkv.paged, "select_entries", lambda w, n, budget, **_: (torch.zeros(len(n), 1, budget, dtype=torch.int32), n))
    monkeypatch.setattr(jkv.paged, "compact_pages", lambda k, v, old, kept, new, weights: weights.clone())
    cache = cache_of(track_weights=True, pages=13)
    owner, fork = [b for b in range(3) if b != private]
    count = [0] * 4
    count[owner], count[private] = 96, 80
    cache.begin(count)
    cache.fork(owner, fork)
    assert cache.free_pages == 2
    cache.evict(32)
    listed(cache)
    assert cache.lengths == (32, 32, 32, 0) and cache.free_pages == 13 - 6


def test_an_eviction_finishes_one_prompts_sharers_first(copies, monkeypatch):
    """Two prompts with sharers each and pages for three moves: the last sharer's is
    what frees a prompt."""

    monkeypatch.setattr(jkv.paged, "select_entries", lambda w, n, budget, **_: (torch.zeros(len(n), 1, budget, dtype=torch.int32), n))
    monkeypatch.setattr(jkv.paged, "compact_pages", lambda k, v, old, kept, new, weights: weights.clone())
    cache = cache_of(track_weights=True, pages=14, sequences=5)
    cache.begin([64, 64, 0, 0, 0])
    cache.fork(0, 2)
    cache.fork(0, 3)
    cache.fork(1, 4)
    assert cache.free_pages == 6
    cache.evict(32)  # (the first three to move would free nothing)
    listed(cache)
    assert cache.lengths == (32,) * 5 and cache.free_pages == 4


def test_tangents_are_refused():
    """Forward mode: a dual tensor would give a result without its tangent."""

    q, k = torch.zeros(4, 2, 64).half(), torch.zeros(4, 1, 64).half()
    with torch.autograd.forward_ad.dual_level():
        dual = lambda x: torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for args in ((dual(q),), (q, dual(k)), (dual(q), k)):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    jkv.rotary(*args)
        for args in ((dual(q), k, k), (q, dual(k), k), (q, k, dual(k))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                jkv.packed_attention(*args, ints(0, 4))
        with pytest.raises(RuntimeError, match="forward-mode"):
            jkv.packed_attention(q, k, k, ints(0, 4), slopes=dual(torch.zeros(2)))
        with pytest.raises(ValueError, match="HIP"):  # (none has a tangent)
            jkv.packed_attention(q, k, k, ints(0, 4))
        with pytest.raises(ValueError, match="HIP"):
            jkv.rotary(q, k)
    with pytest.raises(RuntimeError, match="forward-mode"):
        torch.func.jvp(lambda x: jkv.rotary(x), (q,), (q,))


def test_distances_beside_an_idle_sequence_with_evicted_entries(copies, monkeypatch):
    """Only the sequences that a step attends for must have all their entries."""

    calls = []
    monkeypatch.setattr(jkv.paged, "paged_attention", lambda *args, **form: calls.append(form))
    cache = cache_of()
    cache.begin([20, 20, 0, 0])
    cache._positions = [25, 20, 0, 0]  # (as an eviction leaves them)
    step = cache.begin([0, 3, 5, 0])
    for form in (dict(slopes=torch.zeros(2)), dict(prefixes=ints(0, 0, 0, 0))):
        cache.attention(0, step, torch.zeros(8, 2, 64).half(), **form)
    assert len(calls) == 2
    step = cache.begin([1, 0, 1, 0])
    for form in (dict(slopes=torch.zeros(2)), dict(prefixes=ints(0, 0, 0, 0))):
        with pytest.raises(ValueError, match="evicted"):
            cache.attention(0, step, torch.zeros(2, 2, 64).half(), **form)

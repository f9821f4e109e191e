"""Paged attention with capped, biased and prefix-masked scores on the MI355X
against 64-bit definitions; copied pages and forked sequences."""

from __future__ import annotations

import numpy as np
import pytest
import torch

import jointkv_amd as jkv
from oracle import shaped_oracle as ref
from tests.test_gpu_paged import Batch, half_step

pytestmark = pytest.mark.gpu


def slopes_of(heads):
    return (2.0 ** (-8.0 * torch.arange(1, heads + 1, dtype=torch.float64) / heads)).float()


def expect(batch, **form):
    prefixes = form.pop("prefixes", None) or [0] * len(batch.lengths)
    return [ref.attend(q, k, v, prefix=min(n, p), **form)
            for q, k, v, n, p in zip(batch.queries, batch.keys, batch.values, batch.lengths, prefixes)]


def score_slack(r, dim, cap, slopes, length):
    """How far a score of each row may be off: 32-bit sums of D products
    (2 roundings of a term's size each), the cap's 2e-7, the bias's own
    rounding, the base-2 score's, and the exponential's 2^-22."""

    bias = 0.0 if slopes is None else float(slopes.abs().max()) * length
    size = (r["reach"] if not cap else r["reach"].clamp_max(1e30)) * dim * 2.0**-23
    return size + (4e-7 * cap if cap else 0.0) + 4 * (bias + (cap or 0.0)) * 2.0**-23 + r["reach"] * 2.0**-22 + 2.0**-21


def check(out, results, dtype, dim, cap=None, slopes=None, few=False, length=1, lse=None):
    """Rounding h of the result and of each weight (few rows keep weights in two
    parts, h^2 or 2^-17), scores off by ``score_slack``, which a weight and the
    sum that divides it take on both."""

    h = half_step(dtype)
    at = 0
    for r in results:
        n = r["out"].shape[0]
        got = out[at : at + n].cpu().double()
        off = (score_slack(r, dim, cap, slopes, length) * 2)[..., None]
        p = max(h * h, 2.0**-17) if few else h
        bound = h * r["out"].abs() + (p + off) * r["spread"] * 1.01 + 1e-6 * r["spread"] + 2.0**-24
        assert ((got - r["out"]).abs() <= bound).all(), ((got - r["out"]).abs() - bound).max()
        if lse is not None:
            want = r["lse"]
            mine = lse[at : at + n].cpu().double()
            seen = torch.isfinite(want)
            assert torch.equal(torch.isfinite(mine), seen)
            # (the logarithm's base changes once more)
            assert ((mine - want).abs()[seen] <= (off[..., 0] + 2.0**-21 * (1 + want.abs()))[seen]).all()
        at += n


FORMS = [dict(cap=20.0), dict(bias=True), dict(prefix=True), dict(cap=30.0, bias=True, prefix=True)]
NAMES = ["cap", "bias", "prefix", "all"]


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("lengths,new,qh,kvh,dim,page,window,sinks", [
    ([1], [1], 4, 4, 128, 16, None, 0),                              # one token alone
    ([33, 1, 700, 64], [1, 1, 1, 1], 8, 2, 128, 16, None, 0),         # single tokens
    ([333, 40, 1000], [1, 1, 1], 12, 4, 64, 32, 100, 5),              # a window and first entries
    ([3000, 17], [1, 1], 8, 2, 128, 64, None, 0),                     # splits that are joined
    ([90, 7, 0, 300], [5, 7, 0, 8], 4, 1, 64, 16, None, 0),           # small chunks, few rows, one idle
    ([200, 131, 65], [130, 1, 65], 8, 2, 128, 16, None, 0),           # chunks
    ([500, 77, 3], [129, 64, 3], 7, 1, 64, 32, 50, 3),                # 7 heads to one, a window and first entries
    ([900, 400], [300, 299], 16, 16, 128, 256, None, 0),              # blocks of 256 rows, one head each
])
def test_against_the_definition(device, form, dtype, lengths, new, qh, kvh, dim, page, window, sinks):
    batch = Batch(sum(lengths) + qh, lengths, new, qh=qh, kvh=kvh, dim=dim, page=page, dtype=dtype, theta=None, gain=2.0)
    cap = form.get("cap")
    slopes = slopes_of(qh) if form.get("bias") else None
    prefixes = [n * 2 // 3 for n in lengths] if form.get("prefix") else None
    lse = torch.full((sum(new), qh), 7.0, device=device)
    args = dict(window=window, sinks=sinks, rope_theta=None, softcap=cap, max_new=max(new),
                slopes=None if slopes is None else slopes.to(device),
                prefixes=None if prefixes is None else torch.tensor(prefixes, dtype=torch.int32, device=device))
    on = batch.on(device)
    out = jkv.paged_attention(batch.query.to(device), **on, **args)
    results = expect(batch, window=window, sinks=sinks, cap=cap, slopes=slopes, prefixes=prefixes)
    few = max(new) * (qh // kvh) <= 32
    check(out, results, dtype, dim, cap, slopes, few, max(lengths))
    again = jkv.paged_attention(batch.query.to(device), **on, **args, lse=lse)
    check(again, results, dtype, dim, cap, slopes, few, max(lengths), lse)
    assert torch.equal(jkv.paged_attention(batch.query.to(device), **on, **args), out)


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
@pytest.mark.parametrize("lengths,new,qh,kvh,dim", [
    ([200, 45, 1], [1, 1, 1], 8, 2, 128), ([150, 6], [4, 6], 8, 2, 64), ([400, 90], [200, 90], 4, 2, 128),
    ([700], [600], 3, 3, 64)])
def test_weights_received(device, form, lengths, new, qh, kvh, dim):
    batch = Batch(77 + sum(new), lengths, new, qh=qh, kvh=kvh, dim=dim, theta=None)
    cap, bias, prefix = form.get("cap"), form.get("bias"), form.get("prefix")
    slopes = slopes_of(qh) if bias else None
    prefixes = [n // 2 + 1 for n in lengths] if prefix else None
    weights = torch.full((len(lengths), kvh, max(lengths) + 3), 5.0, device=device)
    jkv.paged_attention(batch.query.to(device), **batch.on(device), window=64, sinks=2, rope_theta=None, softcap=cap,
                        slopes=None if slopes is None else slopes.to(device), weights=weights, max_new=max(new),
                        prefixes=None if prefixes is None else torch.tensor(prefixes, dtype=torch.int32, device=device))
    results = expect(batch, window=64, sinks=2, cap=cap, slopes=slopes, prefixes=prefixes)
    for b, (r, n) in enumerate(zip(results, lengths)):
        slack = float(score_slack(r, dim, cap, slopes, n).max()) * 2 + new[b] * 2.0**-22
        assert ((weights[b, :, :n].cpu().double() - r["weights"]).abs() <= slack * r["weights"] + 1e-9).all()
        assert (weights[b, :, n:] == 5.0).all()


def test_rotation_beside_shaped_scores(device):
    """rope_theta still turns queries, rounded once before the products."""

    batch = Batch(5, [300, 40], [1, 1], qh=8, kvh=2, theta=10000.0, ahead=7)
    out = jkv.paged_attention(batch.query.to(device), **batch.on(device), window=None, softcap=25.0)
    at = torch.tensor([p for p in batch.positions])
    rates = ref.rates(128, 10000.0)
    batch.queries = [ref.turn(q, [int(p)], rates) for q, p in zip(batch.queries, at)]
    # two parts of a query: 2^-17 of a score's terms
    for n, r in enumerate(expect(batch, cap=25.0)):
        off = 2 * (score_slack(r, 128, 25.0, None, 300) + r["reach"] * 2.0**-17)[..., None]
        assert ((out[n : n + 1].cpu().double() - r["out"]).abs() <= 2.0**-11 * r["out"].abs() + (2.0**-17 + off) * r["spread"] + 2.0**-24).all()


@pytest.mark.parametrize("new", [1, 100])
def test_masked_places_may_hold_anything(device, new):
    """Infinite and NaN keys and values of entries that no row sees change
    nothing; a seen infinite key weighs as the cap says."""

    batch = Batch(6, [260], [new], qh=4, kvh=1, dim=64, theta=None)
    args = dict(window=32, rope_theta=None, softcap=10.0)
    clean = jkv.paged_attention(batch.query.to(device), **batch.on(device), **args)
    for j, value in ((0, float("inf")), (50, float("nan")), (100, float("-inf"))):
        batch.k_pool[batch.tables[0, j // 16], :, j % 16] = value
        batch.v_pool[batch.tables[0, j // 16], :, j % 16] = value
    assert torch.equal(jkv.paged_attention(batch.query.to(device), **batch.on(device), **args), clean)
    one = Batch(7, [3], [1], qh=1, kvh=1, dim=64, theta=None)
    one.query.fill_(1.0)
    one.queries = [one.query]
    one.keys[0][0] = float("inf")
    one.write(0, one.keys[0], one.values[0])
    out = jkv.paged_attention(one.query.to(device), **one.on(device), window=None, rope_theta=None, softcap=2.0)
    x = torch.tanh((one.keys[0][:, 0].double() @ one.query[0, 0].double()) / 8 / 2.0) * 2.0
    want = torch.softmax(x, 0) @ one.values[0][:, 0].double()
    assert x[0] == 2.0 and torch.allclose(out[0, 0].cpu().double(), want, atol=2e-3)


def test_slopes_of_every_size(device):
    batch = Batch(8, [500], [1], qh=4, kvh=1, theta=None)
    slopes = torch.tensor([0.0, -0.01, 3.0, 1e30])
    out = jkv.paged_attention(batch.query.to(device), **batch.on(device), window=None, rope_theta=None,
                              slopes=slopes.to(device))
    r = expect(batch, slopes=slopes[:3].tolist() + [1e30])[0]
    off = torch.tensor([2.0**-16, 2.0**-16, 2.0**-14, 2.0**-16])[None, :, None]
    assert ((out.cpu().double() - r["out"]).abs() <= 2.0**-11 * r["out"].abs() + (2.0**-17 + off) * r["spread"] + 2.0**-24).all()
    assert torch.equal(out[0, 3].cpu(), batch.values[0][-1, 0])  # sees itself alone


def test_plain_calls_are_what_they_were(device):
    """No form asked for: the plain kernels, whose scores start from the
    reference; a form that does nothing agrees within both bounds."""

    batch = Batch(9, [400, 30], [60, 30], qh=8, kvh=2, theta=None)
    on = batch.on(device)
    plain = jkv.paged_attention(batch.query.to(device), **on, window=None, rope_theta=None)
    none = jkv.paged_attention(batch.query.to(device), **on, window=None, rope_theta=None,
                               prefixes=torch.zeros(2, dtype=torch.int32, device=device))
    check(none, expect(batch), torch.float16, 128)
    assert (plain.float() - none.float()).abs().max() < 2e-2


def pools(device, layers, pages, dtype=torch.float16, kvh=2, page=16, dim=64, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(layers, pages, kvh, page, dim, generator=gen).to(dtype).to(device) for _ in range(2)]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("layers,page,dim,kvh", [(1, 16, 64, 1), (3, 64, 128, 8), (2, 256, 128, 3)])
def test_copy_pages(device, dtype, layers, page, dim, kvh):
    k, v = pools(device, layers, 9, dtype, kvh, page, dim)
    want = [x.clone() for x in (k, v)]
    src, dst, count = [3, 3, 8, 0, 5, 99, 6, 7], [1, 2, 4, 0, -1, 6, 77, 7], [page, 1, 0, page, page, page, page, page - 1]
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device=device)
    for x in want:
        for s, d, n in zip(src, dst, count):
            if 0 <= s < 9 and 0 <= d < 9:
                x[:, d, :, :n] = x[:, s, :, :n]
    jkv.copy_pages(k, v, ints(src), ints(dst), entries=ints(count))
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    jkv.copy_pages(k[0], v[0], ints([3]), ints([5]))  # one layer, whole pages
    want[0][0, 5], want[1][0, 5] = want[0][0, 3], want[1][0, 3]
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])
    jkv.copy_pages(k, v, ints([]), ints([]))
    # heads inside slots, and counts past a page
    kt, vt = (x.transpose(2, 3).contiguous().transpose(2, 3) for x in (k, v))
    jkv.copy_pages(kt, vt, ints([1, 2]), ints([6, 8]), entries=ints([page + 5, -3]))
    want[0][:, 6], want[1][:, 6] = want[0][:, 1], want[1][:, 1]
    assert torch.equal(kt, want[0]) and torch.equal(vt, want[1])


def test_copy_of_far_pages(device):
    """Offsets past 32 bits."""

    pages = (1 << 31) // (16 * 64 * 2) + 3
    k = torch.empty(pages, 1, 16, 64, dtype=torch.float16, device=device)
    v = torch.empty_like(k)
    k[pages - 1], v[pages - 1], k[0], v[0] = 1.0, 2.0, 0.0, 0.0
    ints = lambda *x: torch.tensor(x, dtype=torch.int32, device=device)
    jkv.copy_pages(k, v, ints(pages - 1), ints(0))
    assert (k[0] == 1).all() and (v[0] == 2).all()
    jkv.copy_pages(k, v, ints(0), ints(pages - 2), entries=ints(7))
    assert (k[pages - 2, :, :7] == 1).all() and (v[pages - 2, :, :7] == 2).all()


class Twin:
    """A PagedKVCache beside each sequence's own lists of keys and values."""

    def __init__(self, device, sequences=5, pages=60, layers=2, track=True, max_length=200):
        self.cache = jkv.PagedKVCache(layers, sequences, pages, 2, max_length=max_length, page_size=16, head_dim=64,
                                      track_weights=track, device=device)
        self.layers, self.device, self.gen = layers, device, torch.Generator().manual_seed(11)
        self.held = [[[] for _ in range(sequences)] for _ in range(layers)]

    def step(self, new, **form):
        step = self.cache.begin(new)
        outs = []
        for layer in range(self.layers):
            k, v = (torch.randn(step.tokens, 2, 64, generator=self.gen).half() for _ in range(2))
            q = torch.randn(step.tokens, 4, 64, generator=self.gen).half()
            self.cache.append(layer, step, k.to(self.device), v.to(self.device), rope_theta=None)
            out = self.cache.attention(layer, step, q.to(self.device), window=None, rope_theta=None, **form)
            at = 0
            for b, n in enumerate(new):
                self.held[layer][b] = self.held[layer][b] + [(k[at + t], v[at + t]) for t in range(n)]
                if n:
                    keys, values = (torch.stack(x) for x in zip(*self.held[layer][b]))
                    r = ref.attend(q[at : at + n], keys, values, cap=form.get("softcap"))
                    check(out[at : at + n], [r], torch.float16, 64, form.get("softcap"), length=200)
                at += n
            outs.append(out)
        return step, outs

    def fork(self, source, target, length=None):
        self.cache.fork(source, target, length)
        for layer in self.held:
            layer[target] = list(layer[source] if length is None else layer[source][:length])


def test_forked_sequences_go_their_own_ways(device):
    twin = Twin(device)
    twin.step([40, 0, 0, 7, 0])
    free = twin.cache.free_pages
    twin.fork(0, 1)
    twin.fork(0, 2, 35)
    twin.fork(0, 4, 32)  # whole pages
    assert twin.cache.free_pages == free and twin.cache.lengths == (40, 40, 35, 7, 32)
    twin.step([1, 1, 1, 1, 1], softcap=30.0)
    # two of the three sharers of the half-written page copied it, the last one wrote in place; one new page
    assert twin.cache.free_pages == free - 3
    twin.step([3, 30, 1, 0, 20])
    twin.cache.release(0)
    twin.held = [[[] if b == 0 else x for b, x in enumerate(layer)] for layer in twin.held]
    twin.step([5, 2, 2, 2, 2])
    for b in range(5):
        twin.cache.release(b)
    assert twin.cache.free_pages == 60


def test_cancel_after_a_copied_page(device):
    twin = Twin(device)
    twin.step([20, 0, 0, 0, 0])
    twin.fork(0, 1)
    before = (twin.cache.free_pages, twin.cache.lengths, list(twin.cache._free), list(twin.cache._uses),
              twin.cache.block_tables.clone())
    held = [[list(x) for x in layer] for layer in twin.held]
    step, _ = twin.step([1, 2, 0, 0, 0])
    assert twin.cache.free_pages == before[0] - 1
    twin.cache.cancel(step)
    twin.held = held
    assert (twin.cache.free_pages, twin.cache.lengths, twin.cache._free, twin.cache._uses) == before[:4]
    assert torch.equal(twin.cache.block_tables, before[4])
    twin.step([1, 2, 0, 0, 0])


def test_eviction_of_forked_sequences(device):
    twin = Twin(device, pages=30)
    twin.step([100, 0, 0, 0, 0])
    twin.cache.fork(0, 1)
    for w in twin.cache.weights:
        assert torch.equal(w[0], w[1])
    old = [twin.cache.key[layer].clone() for layer in range(2)]
    twin.cache.evict(32, sinks=4, recent=8)
    assert twin.cache.lengths == (32, 32, 0, 0, 0) and twin.cache.free_pages == 30 - 4
    for layer in range(2):
        rows = [twin.cache.key[layer][twin.cache.block_tables[b, :2].long()] for b in (0, 1)]
        assert torch.equal(rows[0], rows[1])
    del old


def test_rule_in_a_cache(device):
    """Keys and queries turned by a rule: what attention over turned rows gives,
    each rounded once more."""

    rule = jkv.RotaryRule(layout="interleaved", dims=32, scaling="linear", factor=2.0)
    cache = jkv.PagedKVCache(1, 2, 20, 2, max_length=100, page_size=16, head_dim=64, device=device)
    gen = torch.Generator().manual_seed(3)
    held = [[], []]
    for new in ([30, 5], [1, 1], [0, 3]):
        step = cache.begin(new)
        q, k, v = (torch.randn(step.tokens, h, 64, generator=gen).half().to(device) for h in (4, 2, 2))
        cache.append(0, step, k, v, rule=rule)
        out = cache.attention(0, step, q, window=None, rule=rule, softcap=40.0)
        at = 0
        for b, n in enumerate(new):
            first = len(held[b])
            pos = list(range(first, first + n))
            rates = ref.rates(32, 10000.0, "linear", 2.0)
            turned = [ref.turn(x[at : at + n].cpu(), pos, rates, layout="interleaved").half() for x in (q, k)]
            held[b] = held[b] + list(zip(turned[1], v[at : at + n].cpu()))
            if n:
                keys, values = (torch.stack(x) for x in zip(*held[b]))
                r = ref.attend(turned[0], keys, values, cap=40.0)
                # a turned value next to a border may round the other way: h of a score's terms, twice
                slack = 2 * (r["reach"] * 2.0**-10)[..., None] * r["spread"]
                assert ((out[at : at + n].cpu().double() - r["out"]).abs() <= 2.0**-10 * r["spread"] + slack + 1e-6).all()
            at += n


@pytest.mark.parametrize("owner", [0, 1])
def test_cancel_after_a_shorter_sharer_kept_the_page(device, owner):
    """What a cancelled step wrote over entries that others have is undone, in both
    pools and all layers: every later attention still matches its own rows."""

    twin = Twin(device)
    new = [0] * 5
    new[owner] = 40
    twin.step(new)
    twin.fork(owner, 1 - owner, 35)
    twin.fork(owner, 2, 33)
    held = [[list(x) for x in layer] for layer in twin.held]
    for count in ([1, 1, 1, 0, 0], [2, 9, 4, 0, 0], [1, 1, 0, 0, 0]):
        step, _ = twin.step(count)
        twin.cache.cancel(step)
        twin.held = [[list(x) for x in layer] for layer in held]
    twin.step([1, 1, 1, 0, 0])
    twin.step([2, 1, 3, 0, 0])

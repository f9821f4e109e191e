"""The paged K/V cache on the MI355X against 64-bit definitions."""

from __future__ import annotations

import dataclasses

import numpy as np
import pytest
import torch

import jointkv_amd as jkv
from oracle import paged_oracle as ref

pytestmark = pytest.mark.gpu

THETA = 10000.0


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


class Batch:
    """Random sequences in a pool whose other slots hold NaN."""

    def __init__(self, seed, lengths, new, *, qh, kvh, dim=128, page=16, dtype=torch.float16, theta=THETA, ahead=0,
                 gain=1.0, layout="phsd", spare=2):
        rng = np.random.default_rng(seed)
        gen = torch.Generator().manual_seed(seed)
        self.lengths, self.new, self.qh, self.kvh, self.dim, self.page = lengths, new, qh, kvh, dim, page
        self.dtype, self.theta = dtype, theta
        counts = [-(-x // page) for x in lengths]
        self.width = max(max(counts), 1)
        pages = sum(counts) + spare
        order = rng.permutation(pages)
        self.tables = np.full((len(lengths), self.width), -1, dtype=np.int32)
        at = 0
        for b, n in enumerate(counts):
            self.tables[b, :n] = order[at : at + n]
            at += n
        shapes = {"phsd": ((pages, kvh, page, dim), (0, 1, 2, 3)), "pshd": ((pages, page, kvh, dim), (0, 2, 1, 3))}
        shape, axes = shapes[layout]
        self.k_pool = torch.full(shape, float("nan"), dtype=dtype).permute(axes)
        self.v_pool = torch.full(shape, float("nan"), dtype=dtype).permute(axes)
        self.positions = [x - n + ahead * (b + 1) for b, (x, n) in enumerate(zip(lengths, new))]
        self.keys, self.values, self.queries = [], [], []
        for b, length in enumerate(lengths):
            k = (torch.randn(length, kvh, dim, generator=gen) * gain).to(dtype)
            v = torch.randn(length, kvh, dim, generator=gen).to(dtype)
            self.keys.append(k)
            self.values.append(v)
            self.write(b, k, v)
            self.queries.append((torch.randn(new[b], qh, dim, generator=gen) * gain).to(dtype))
        self.query = torch.cat(self.queries)
        self.starts = np.concatenate(([0], np.cumsum(new))).astype(np.int32)

    def write(self, b, k, v):
        for j in range(len(k)):
            page, slot = self.tables[b, j // self.page], j % self.page
            self.k_pool[page, :, slot] = k[j]
            self.v_pool[page, :, slot] = v[j]

    def on(self, device):
        def ints(x):
            return torch.tensor(np.asarray(x), dtype=torch.int32, device=device)

        # Tensor.to keeps the permuted strides
        return {"key_pages": self.k_pool.to(device), "value_pages": self.v_pool.to(device),
                "block_tables": ints(self.tables), "lengths": ints(self.lengths), "starts": ints(self.starts),
                "positions": ints(self.positions)}

    def expect(self, window, sinks, scale=None):
        return [ref.attend(q.double().numpy(), k.double().numpy(), v.double().numpy(), p, window=window, sinks=sinks,
                           theta=self.theta, scale=scale)
                for q, k, v, p in zip(self.queries, self.keys, self.values, self.positions)]


def check_out(out, expect, dtype, rows=None):
    """|error| against its bound: the result's own rounding h, and what a p and
    a rotated q of 16 bits are off by: h each of p's terms and up to
    exp(2 h reach) - 1 of all (reach = scale sum |q k| bounds how far h of q
    moves a score); 32-bit sums add 2^-20 of sum p |v| and scores."""

    h = half_step(dtype)
    got = out.detach().double().cpu().numpy()
    want = np.concatenate([e["out"] for e in expect])
    spread = np.concatenate([e["spread"] for e in expect])
    reach = np.concatenate([e["reach"] for e in expect])[..., None]
    slack = 2.0 ** -20
    tol = h * np.abs(want) + spread * (h + np.expm1(2 * (h + slack) * reach) + slack) * (1 + h)
    tol = tol + float(torch.finfo(dtype).tiny)
    err = np.abs(got - want)
    assert np.isfinite(got).all()
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol).all(), f"error {err[worst]} over {tol[worst]} at {worst}"
    # the roundings are independent: their sum is a fraction of their bound
    norm = np.linalg.norm(want)
    if norm > 0 and want.size >= 512:
        rms_reach = float(np.sqrt(np.mean(reach ** 2)))
        rel = np.linalg.norm(err) / norm
        assert rel <= 2 * h * (1 + rms_reach), f"relative error {rel}"


def check_weights(got, expect, lengths):
    """fp32 weights: scores of 32-bit sums over exact products with a query
    held to 2^-16 or better, so a weight is off by at most 2 (2^-17 reach) of
    itself, and the sums by 2^-20."""

    for b, e in enumerate(expect):
        w = got[b, :, : lengths[b]].double().cpu().numpy()
        reach = float(e["reach"].max()) if e["reach"].size else 0.0
        tol = e["weights"] * (np.expm1(2 * 2.0 ** -17 * reach) + 2.0 ** -18) + 1e-30
        assert (np.abs(w - e["weights"]) <= tol).all(), float((np.abs(w - e["weights"]) - tol).max())


CASES = [
    # lengths, new tokens, heads, dims, page, window, sinks
    pytest.param([1], [1], 1, 1, 64, 16, None, 0, id="one-entry"),
    pytest.param([1, 2, 17, 16, 15], [1, 1, 1, 1, 1], 4, 1, 128, 16, None, 0, id="page-edges"),
    pytest.param([300], [1], 32, 8, 128, 16, None, 0, id="one-sequence"),
    pytest.param([65, 64, 63, 700, 129], [1] * 5, 8, 2, 128, 64, None, 0, id="tile-edges"),
    pytest.param([65, 64, 63, 700, 129], [1] * 5, 14, 2, 64, 32, 50, 4, id="window-sinks"),
    pytest.param([500, 40, 33], [1] * 3, 16, 1, 128, 32, 16, 100, id="sinks-over-window"),
    pytest.param([300, 5], [1] * 2, 24, 1, 64, 16, 1, 0, id="window-of-one"),
    pytest.param([600, 3], [1] * 2, 40, 1, 128, 128, None, 0, id="many-heads"),
    pytest.param([1300], [1], 4, 4, 128, 256, 1000, 70, id="multi-head"),
    pytest.param([7, 130, 260], [7, 2, 3], 8, 2, 128, 16, None, 0, id="small-chunks"),
    pytest.param([128], [128], 4, 1, 128, 64, None, 0, id="whole-prompt"),
    pytest.param([333, 70, 200, 9], [129, 1, 200, 0], 12, 4, 64, 16, None, 0, id="mixed"),
    pytest.param([333, 70, 200, 9], [129, 1, 200, 0], 10, 2, 128, 32, 40, 3, id="mixed-window-sinks"),
    pytest.param([450, 64], [300, 64], 7, 1, 64, 64, 64, 65, id="chunk-tile-sinks"),
    pytest.param([700], [513], 3, 3, 128, 16, 200, 0, id="chunk-window"),
    pytest.param([0, 5, 0], [0, 2, 0], 2, 1, 128, 16, None, 0, id="empty-sequences"),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("lengths,new,qh,kvh,dim,page,window,sinks", CASES)
def test_attention_lse_and_weights(device, lengths, new, qh, kvh, dim, page, window, sinks, dtype):
    print(f"paged L={lengths} T={new} heads={qh}/{kvh} D={dim} page={page} window={window} sinks={sinks} {dtype}",
          flush=True)
    batch = Batch(sum(lengths) + dim, lengths, new, qh=qh, kvh=kvh, dim=dim, page=page, dtype=dtype, ahead=1000)
    args = batch.on(device)
    expect = batch.expect(window, sinks)
    query = batch.query.to(device)
    single = all(n == 1 for n in new)
    if single:
        args["starts"] = None
    bounds = dict(max_new=max(new), max_length=max(lengths))
    out = jkv.paged_attention(query, **args, window=window, sinks=sinks, **bounds)
    check_out(out, expect, dtype)
    # with what else it can give, and without the caller's bounds
    width = batch.width * page
    weights = torch.full((len(lengths), kvh, width), 7.0, device=device)
    lse = torch.empty(len(query), qh, device=device)
    out2 = jkv.paged_attention(query, **args, window=window, sinks=sinks, weights=weights, lse=lse)
    check_out(out2, expect, dtype)
    check_weights(weights, expect, lengths)
    for b, length in enumerate(lengths):
        assert bool((weights[b, :, length:] == 7.0).all()), "weights behind the last entry were written"
    want = np.concatenate([e["lse"] for e in expect])
    reach = np.concatenate([e["reach"] for e in expect])
    assert (np.abs(lse.double().cpu().numpy() - want) <= 2.0 ** -17 * reach + 2.0 ** -19 * (1 + np.abs(want))).all()
    # added to what is there: two equal calls give exactly twice one
    once = weights.clone()
    jkv.paged_attention(query, **args, window=window, sinks=sinks, weights=weights, accumulate=True)
    for b, length in enumerate(lengths):
        assert torch.equal(weights[b, :, :length], 2 * once[b, :, :length])
    # the same call repeats bit for bit
    assert torch.equal(out, jkv.paged_attention(query, **args, window=window, sinks=sinks, **bounds))
    if single:  # one token a sequence, said with starts
        args["starts"] = torch.arange(len(lengths) + 1, dtype=torch.int32, device=device)
        assert torch.equal(out, jkv.paged_attention(query, **args, window=window, sinks=sinks, **bounds))


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("theta", [THETA, None, 500000.0])
def test_append_rotates_and_places(device, dim, dtype, theta):
    lengths, new = [40, 17, 1, 64, 9], [7, 1, 1, 64, 0]
    batch = Batch(dim, lengths, new, qh=2, kvh=2, dim=dim, dtype=dtype)
    # far positions: angles that 32 bits lose
    batch.positions = [33, 1_000_003, 0, 2 ** 30 - 5, 4]
    args = batch.on(device)
    gen = torch.Generator().manual_seed(9)
    rows = sum(new)
    # rows behind the last sequence are nobody's
    key = torch.randn(rows + 3, 2, dim, generator=gen).to(dtype)
    value = torch.randn(rows + 3, 2, dim, generator=gen).to(dtype)
    before_k, before_v = batch.k_pool.clone(), batch.v_pool.clone()
    jkv.paged_append(key.to(device), value.to(device), **args, rope_theta=theta)
    h = half_step(dtype)
    at = 0
    for b, (length, n) in enumerate(zip(lengths, new)):
        want = ref.rotate(key[at : at + n].double().numpy(), batch.positions[b] + np.arange(n), theta)
        size = np.abs(key[at : at + n].double().numpy()).max(initial=0)
        for t in range(n):
            j = length - n + t
            page, slot = batch.tables[b, j // 16], j % 16
            got = args["key_pages"][page, :, slot].double().cpu().numpy()
            # one rounding of the result, 32-bit products and the hardware's sine and cosine (2^-19 of the pair)
            assert (np.abs(got - want[t]) <= h * np.abs(want[t]) + 2.0 ** -18 * size).all()
            assert torch.equal(args["value_pages"][page, :, slot].cpu(), value[at + t])
            before_k[page, :, slot] = args["key_pages"][page, :, slot].cpu()
            before_v[page, :, slot] = args["value_pages"][page, :, slot].cpu()
        at += n
    # nothing else was written
    for pool, before in ((args["key_pages"], before_k), (args["value_pages"], before_v)):
        assert torch.equal(pool.cpu().view(torch.int16), before.view(torch.int16))


def test_append_then_attend_a_prompt_in_chunks(device):
    """A run of the operators as a server makes it: prompts in chunks beside
    single tokens, in another memory layout of the pool."""

    kvh, qh, dim, dtype = 2, 8, 128, torch.float16
    final = [150, 61, 99]
    batch = Batch(5, final, [0, 0, 0], qh=qh, kvh=kvh, dim=dim, dtype=dtype, layout="pshd")
    gen = torch.Generator().manual_seed(6)
    raw = [(torch.randn(n, kvh, dim, generator=gen).to(dtype), torch.randn(n, kvh, dim, generator=gen).to(dtype),
            torch.randn(n, qh, dim, generator=gen).to(dtype)) for n in final]
    pools = batch.on(device)
    done = [0, 0, 0]
    for step in ([64, 0, 1], [60, 33, 97], [1, 1, 1], [25, 27, 0]):
        after = [d + n for d, n in zip(done, step)]
        key, value, query = (torch.cat([x[i][d:a] for x, d, a in zip(raw, done, after)]).to(device) for i in range(3))
        starts = torch.tensor(np.concatenate(([0], np.cumsum(step))), dtype=torch.int32, device=device)
        lengths = torch.tensor(after, dtype=torch.int32, device=device)
        where = (pools["key_pages"], pools["value_pages"], pools["block_tables"], lengths)
        jkv.paged_append(key, value, *where, starts=starts)
        out = jkv.paged_attention(query, *where, starts=starts, window=50, sinks=2)
        expect = []
        for b in range(3):
            # what the cache holds: the rotation rounded once
            k = ref.rotate(raw[b][0][: after[b]].double().numpy(), np.arange(after[b]), THETA)
            k = torch.from_numpy(k).to(dtype).double().numpy()
            expect.append(ref.attend(raw[b][2][done[b] : after[b]].double().numpy(), k,
                                     raw[b][1][: after[b]].double().numpy(), done[b], window=50, sinks=2, theta=THETA))
        check = np.concatenate([e["reach"] for e in expect])
        assert check.shape[0] == sum(step)
        # a rotated key on a rounding's edge may fall either way: one more half step of the keys
        for e in expect:
            e["reach"] = e["reach"] * 2
        check_out(out, expect, dtype)
        done = after


def test_unseen_entries_may_hold_anything(device):
    """NaN and infinities outside a row's window, behind it, and behind the
    length reach no output and no weight."""

    for dtype in (torch.float16, torch.bfloat16):
        for qh, new, window, sinks in ((4, 1, 33, 2), (4, 20, 33, 2), (4, 150, 40, 3), (2, 150, 1, 0)):
            lengths = [200, 163]
            batch = Batch(3, lengths, [new, new], qh=qh, kvh=2, dim=128, dtype=dtype)
            expect = batch.expect(window, sinks)
            bad = [float("nan"), float("inf"), float("-inf")]
            for b, length in enumerate(lengths):
                seen = ref.visible(length - new, new, length, window, sinks).any(0)
                for n, j in enumerate(np.nonzero(~seen)[0]):
                    batch.keys[b][j] = bad[n % 3]
                    batch.values[b][j] = bad[(n + 1) % 3]
                batch.write(b, batch.keys[b], batch.values[b])
            args = batch.on(device)
            weights = torch.zeros(2, 2, 256, device=device)
            out = jkv.paged_attention(batch.query.to(device), **args, window=window, sinks=sinks, weights=weights)
            check_out(out, expect, dtype)
            check_weights(weights, expect, lengths)


@pytest.mark.parametrize("new", [3, 40, 200])
def test_non_finite_values_reach_only_the_rows_that_see_them(device, new):
    """An infinite value is seen by the tokens from its own on, while it lies
    in their window: those get infinity or NaN as their sums do, the others
    their finite results."""

    length, window = 260, 90
    batch = Batch(new, [length], [new], qh=2, kvh=1, dim=64)
    j = length - new + new // 2  # one of the new tokens
    clean = batch.expect(window, 0)[0]
    batch.values[0][j, 0, 5] = float("inf")
    batch.values[0][j, 0, 9] = float("nan")
    batch.write(0, batch.keys[0], batch.values[0])
    args = batch.on(device)
    out = jkv.paged_attention(batch.query.to(device), **args, window=window).double().cpu().numpy()
    seen = ref.visible(length - new, new, length, window, 0)[:, j]
    assert (out[seen][:, :, 5] == np.inf).all() and np.isnan(out[seen][:, :, 9]).all()
    for e in ("out", "spread", "reach"):
        clean[e] = clean[e][~seen]
    check_out(torch.from_numpy(out[~seen]).half(), [clean], torch.float16)


def test_rows_that_see_nothing_and_rows_of_nobody(device):
    batch = Batch(1, [3, 40], [3, 2], qh=4, kvh=2, dim=128)
    args = batch.on(device)
    # five packed rows for a sequence of three entries: the first two see none
    query = torch.randn(10, 4, 128, generator=torch.Generator().manual_seed(2)).half()
    args["starts"] = torch.tensor([0, 5, 7], dtype=torch.int32, device=device)
    out = torch.full((10, 4, 128), 9.0, dtype=torch.float16, device=device)
    lse = torch.full((10, 4), 9.0, device=device)
    weights = torch.zeros(2, 2, 64, device=device)
    jkv.paged_attention(query.to(device), **args, out=out, lse=lse, weights=weights)
    assert bool((out[:2] == 0).all()) and bool((lse[:2] == float("-inf")).all())
    assert bool((out[7:] == 9.0).all()) and bool((lse[7:] == 9.0).all())
    assert bool(torch.isfinite(lse[2:7]).all())
    # every visible token's weights sum to one a head
    assert torch.allclose(weights.sum(-1).cpu(), torch.tensor([[6.0, 6.0], [4.0, 4.0]]), atol=1e-4)
    # starts that begin behind row 0, and a sequence of no entries with a token
    args["starts"] = torch.tensor([4, 5, 5], dtype=torch.int32, device=device)
    args["lengths"] = torch.tensor([0, 40], dtype=torch.int32, device=device)
    out.fill_(9.0)
    jkv.paged_attention(query.to(device), **args, out=out)
    assert bool((out[4] == 0).all()) and bool((out[:4] == 9.0).all()) and bool((out[5:] == 9.0).all())


@pytest.mark.parametrize("new", [1, 70])
def test_pages_outside_the_pool_read_as_zeros(device, new):
    """A table that names no page of the pool: nothing is read there."""

    batch = Batch(4, [100], [new], qh=4, kvh=2, dim=128)
    bad = {1: -1, 3: 10 ** 9, 4: batch.k_pool.shape[0]}
    for at, page in bad.items():
        batch.tables[0, at] = page
        batch.keys[0][16 * at : 16 * at + 16] = 0
        batch.values[0][16 * at : 16 * at + 16] = 0
    args = batch.on(device)
    out = jkv.paged_attention(batch.query.to(device), **args, window=None)
    check_out(out, batch.expect(None, 0), torch.float16)
    before = args["key_pages"].clone()
    jkv.paged_append(torch.ones(16, 2, 128, dtype=torch.float16, device=device),
                     torch.ones(16, 2, 128, dtype=torch.float16, device=device), args["key_pages"],
                     args["value_pages"], args["block_tables"], torch.tensor([32], dtype=torch.int32, device=device),
                     starts=torch.tensor([0, 16], dtype=torch.int32, device=device))
    assert torch.equal(args["key_pages"].view(torch.int16), before.view(torch.int16))


def test_strided_queries_outputs_and_tables(device):
    batch = Batch(8, [90, 200], [5, 150], qh=6, kvh=2, dim=64, layout="pshd")
    args = batch.on(device)
    rows = len(batch.query)
    wide = torch.zeros(6, rows, 64 + 8, dtype=torch.float16, device=device)
    wide[:, :, :64] = batch.query.to(device).permute(1, 0, 2)
    query = wide.permute(1, 0, 2)[:, :, :64]  # heads outermost, rows further apart
    held = torch.zeros(rows, 12, 64, dtype=torch.float16, device=device)
    args["block_tables"] = torch.cat((args["block_tables"], args["block_tables"]), 1)[:, : batch.width]
    jkv.paged_attention(query, **args, out=held[:, ::2])
    check_out(held[:, ::2], batch.expect(jkv.attention.MISTRAL_WINDOW, 0), torch.float16)
    assert bool((held[:, 1::2] == 0).all())
    odd = torch.zeros(rows, 6, 65, dtype=torch.float16, device=device)
    odd[:, :, 1:] = batch.query.to(device)  # rows that 16-byte loads cannot take
    assert torch.equal(jkv.paged_attention(odd[:, :, 1:], **args), held[:, ::2].contiguous())


def test_scale_and_large_scores(device):
    """Scores of hundreds: the running maximum moves from tile to tile."""

    for new in (1, 100):
        batch = Batch(11, [700], [new], qh=4, kvh=2, dim=128, gain=6.0, dtype=torch.float16)
        args = batch.on(device)
        for scale in (None, 0.02, 0.0):
            out = jkv.paged_attention(batch.query.to(device), **args, window=None, scale=scale)
            check_out(out, batch.expect(None, 0, scale), torch.float16)


def test_long_cache_is_split_and_joined(device):
    """Many entries of one sequence: the work is divided over them."""

    for new, dtype in ((1, torch.float16), (1, torch.bfloat16), (5, torch.float16), (64, torch.bfloat16)):
        batch = Batch(12, [9000], [new], qh=4, kvh=1, dim=64, page=128, dtype=dtype)
        args = batch.on(device)
        out = jkv.paged_attention(batch.query.to(device), **args, window=None)
        check_out(out, batch.expect(None, 0), dtype)
        out = jkv.paged_attention(batch.query.to(device), **args, window=5000, sinks=130)
        check_out(out, batch.expect(5000, 130), dtype)


def test_blocks_between_one_and_two_a_cu_are_split(device):
    """520 tokens of 64 heads over 4,900 entries: 264 blocks of rows with chains
    long enough to be split in two."""

    batch = Batch(45, [4900], [520], qh=64, kvh=8, dim=64, page=64)
    weights = torch.full((1, 8, 4900), -1.0, device=device)
    query, args = batch.query.to(device), batch.on(device)
    plain = jkv.paged_attention(query, **args, window=None, max_length=4900, max_new=520)
    exact = jkv.paged_attention(query, **args, window=None, max_length=4900, max_new=520, weights=weights)
    for h in (0, 7):
        heads = slice(8 * h, 8 * h + 8)
        expect = [ref.attend(batch.queries[0][:, heads].double().numpy(), batch.keys[0][:, h : h + 1].double().numpy(),
                             batch.values[0][:, h : h + 1].double().numpy(), batch.positions[0], window=None, sinks=0,
                             theta=THETA)]
        check_out(plain[:, heads], expect, torch.float16)
        check_out(exact[:, heads], expect, torch.float16)
        check_weights(weights[:, h : h + 1], expect, [4900])


@pytest.mark.parametrize("length,budget,sinks,recent", [
    (10, 20, 0, 0), (20, 20, 2, 3), (21, 20, 0, 0), (100, 20, 4, 16), (100, 20, 20, 0), (100, 20, 0, 20),
    (5000, 1024, 4, 256), (4097, 4096, 0, 0), (12345, 1, 0, 0), (9000, 8000, 1, 1),
])
def test_select_entries(device, length, budget, sinks, recent):
    rng = np.random.default_rng(length + budget)
    other = max(1, length // 3)
    w = np.exp(2 * rng.standard_normal((2, 3, length + 5))).astype(np.float32)
    w[0, 0, : length // 2] = 0.0
    w[0, 0, 1::2] = -0.0
    w[0, 1] = np.round(w[0, 1])  # many equal
    w[0, 2, ::7] = np.nan
    w[0, 2, 3::11] = np.inf
    w[1, 0] = 1.0
    w[1, 1] = -w[1, 1]
    w[1, 2, ::5] = -np.inf
    lengths = [length, other]
    kept, new_lengths = jkv.select_entries(torch.from_numpy(w).to(device),
                                           torch.tensor(lengths, dtype=torch.int32, device=device), budget,
                                           sinks=sinks, recent=recent)
    assert new_lengths.tolist() == [min(x, budget) for x in lengths]
    for b in range(2):
        for h in range(3):
            want = ref.select(w[b, h, : lengths[b]], budget, sinks, recent)
            got = kept[b, h].cpu().numpy()
            assert (got[: len(want)] == want).all() and (got[len(want) :] == -1).all()


@pytest.mark.parametrize("dim,page,layout", [(128, 16, "phsd"), (64, 64, "pshd")])
def test_compact_pages(device, dim, page, layout):
    lengths, budget = [200, 30], 77
    batch = Batch(dim, lengths, [0, 0], qh=2, kvh=2, dim=dim, page=page, layout=layout, spare=2 + 2 * -(-budget // page))
    args = batch.on(device)
    weights = torch.rand(2, 2, 220, generator=torch.Generator().manual_seed(1)).to(device)
    kept, new_lengths = jkv.select_entries(weights, args["lengths"], budget, sinks=2, recent=9)
    used = set(batch.tables[batch.tables >= 0].tolist())
    free = [p for p in range(batch.k_pool.shape[0]) if p not in used]
    per = -(-budget // page)
    new_tables = np.array([free[:per], [*batch.tables[1, : -(-30 // page)], *([-1] * per)][:per]], dtype=np.int32)
    before_k, before_v = args["key_pages"].clone().cpu(), args["value_pages"].clone().cpu()
    moved = jkv.compact_pages(args["key_pages"], args["value_pages"], args["block_tables"], kept,
                              torch.from_numpy(new_tables).to(device), weights=weights)
    for b in range(2):
        for h in range(2):
            stay = ref.select(weights[b, h, : lengths[b]].cpu().numpy(), budget, 2, 9)
            for j, e in enumerate(stay):
                before_k[new_tables[b, j // page], h, j % page] = batch.keys[b][e, h]
                before_v[new_tables[b, j // page], h, j % page] = batch.values[b][e, h]
            assert torch.equal(moved[b, h, : len(stay)].cpu(), weights[b, h].cpu()[torch.from_numpy(stay)])
            assert bool((moved[b, h, len(stay) :] == 0).all())
    assert torch.equal(args["key_pages"].cpu().view(torch.int16), before_k.view(torch.int16))
    assert torch.equal(args["value_pages"].cpu().view(torch.int16), before_v.view(torch.int16))


def test_cache_serves_two_layers_evicts_and_goes_on(device):
    """The class, as a server uses it: prompts, single tokens, an eviction, the
    steps after it and a sequence that leaves, against plain caches."""

    layers, kvh, qh, dim, dtype = 2, 2, 4, 64, torch.float16
    cache = jkv.PagedKVCache(layers, 3, 24, kvh, max_length=160, page_size=16, head_dim=dim, dtype=dtype,
                             track_weights=True, device=device)
    gen = torch.Generator().manual_seed(3)
    keys = [[np.zeros((0, kvh, dim)) for _ in range(3)] for _ in range(layers)]
    values = [[np.zeros((0, kvh, dim)) for _ in range(3)] for _ in range(layers)]
    weights = [[np.zeros((kvh, 0)) for _ in range(3)] for _ in range(layers)]
    position = [0, 0, 0]

    def step(new):
        plan = cache.begin(new)
        for layer in range(layers):
            k, v = (torch.randn(sum(new), kvh, dim, generator=gen).to(dtype) for _ in range(2))
            q = torch.randn(sum(new), qh, dim, generator=gen).to(dtype)
            cache.append(layer, plan, k.to(device), v.to(device))
            out = cache.attention(layer, plan, q.to(device), window=60, sinks=2)
            expect, at = [], 0
            for b, n in enumerate(new):
                turned = ref.rotate(k[at : at + n].double().numpy(), position[b] + np.arange(n), THETA)
                turned = torch.from_numpy(turned).to(dtype).double().numpy()
                keys[layer][b] = np.concatenate((keys[layer][b], turned))
                values[layer][b] = np.concatenate((values[layer][b], v[at : at + n].double().numpy()))
                e = ref.attend(q[at : at + n].double().numpy(), keys[layer][b], values[layer][b], position[b],
                               window=60, sinks=2, theta=THETA)
                grown = np.zeros((kvh, len(keys[layer][b])))
                grown[:, : weights[layer][b].shape[1]] = weights[layer][b]
                weights[layer][b] = grown + e["weights"]
                e["reach"] = e["reach"] * 2  # a key on a rounding's edge may fall either way
                expect.append(e)
                at += n
            check_out(out, expect, dtype)
        for b, n in enumerate(new):
            position[b] += n

    step([100, 40, 3])
    step([1, 1, 1])
    step([1, 70, 0])
    assert cache.lengths == (102, 111, 4) and cache.positions == (102, 111, 4)
    free = cache.free_pages
    tracked = [[w[b].cpu().numpy() for b in range(3)] for w in cache.weights]
    for layer in range(layers):
        for b in range(3):
            n = weights[layer][b].shape[1]
            assert np.allclose(tracked[layer][b][:, :n], weights[layer][b], rtol=2e-2, atol=1e-6)
            assert (tracked[layer][b][:, n:] == 0).all()
    cache.evict(48, sinks=2, recent=16)
    assert cache.lengths == (48, 48, 4) and cache.positions == (102, 111, 4)
    assert cache.free_pages == free + 7 + 7 - 3 - 3
    for layer in range(layers):
        for b in range(3):
            stay = [ref.select(tracked[layer][b][h, : len(keys[layer][b])], 48, 2, 16) for h in range(kvh)]
            keys[layer][b], values[layer][b] = (np.stack([x[stay[h], h] for h in range(kvh)], 1)
                                                for x in (keys[layer][b], values[layer][b]))
            weights[layer][b] = np.stack([weights[layer][b][h, stay[h]] for h in range(kvh)])
    step([1, 1, 1])
    step([5, 0, 60])
    cache.release(1)
    for layer in range(layers):
        keys[layer][1] = values[layer][1] = np.zeros((0, kvh, dim))
        weights[layer][1] = np.zeros((kvh, 0))
    position[1] = 0
    step([1, 20, 1])
    assert cache.lengths == (55, 20, 66)
    with pytest.raises(ValueError, match="holds 160"):
        cache.begin([200, 0, 0])
    with pytest.raises(ValueError, match="are free"):
        cache.begin([105, 140, 94])


def test_captured_steps_outlive_an_eviction(device):
    """A step captured once and replayed, its tensors refilled, before and after
    an eviction, against a second cache that is stepped eagerly."""

    kvh, qh, dim = 2, 4, 64
    gen = torch.Generator().manual_seed(43)

    def new_cache():
        return jkv.PagedKVCache(1, 2, 20, kvh, max_length=128, page_size=16, head_dim=dim, track_weights=True,
                                device=device)

    def randn(n, heads):
        return torch.randn(n, heads, dim, generator=gen).half().to(device)

    def run(cache, step, k, v, q):
        cache.append(0, step, k, v)
        return cache.attention(0, step, q, window=50, sinks=2)

    caches = [new_cache(), new_cache()]
    prompt = randn(120, kvh), randn(120, kvh), randn(120, qh)
    for cache in caches:
        run(cache, cache.begin([70, 50]), *prompt)
    # replays of longer sequences than now: the bound is the cache's
    held = dataclasses.replace(caches[0].begin([1, 1]), max_length=128)
    k, v, q = randn(2, kvh), randn(2, kvh), randn(2, qh)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = run(caches[0], held, k, v, q)
    for turn in range(4):
        if turn == 2:
            for cache in caches:
                cache.evict(32, sinks=2, recent=8)
        if turn > 0:
            step = caches[0].begin([1, 1])
            held.lengths.copy_(step.lengths)
            held.positions.copy_(step.positions)
            for t, heads in ((k, kvh), (v, kvh), (q, qh)):
                t.copy_(randn(2, heads))
        want = run(caches[1], caches[1].begin([1, 1]), k, v, q)
        other = torch.full((2, kvh, 128), -1.0, device=device)  # takes what memory is free
        graph.replay()
        torch.cuda.synchronize()
        assert torch.allclose(out.float(), want.float(), rtol=2 * half_step(torch.float16), atol=2.0 ** -20)
        assert torch.allclose(caches[0].weights[0], caches[1].weights[0], rtol=2.0 ** -18, atol=0)
        assert (other == -1.0).all()
    assert caches[0].lengths == (34, 34)


def test_codec_reconstructions_through_pages_match_the_prefill(device):
    """The codec's reconstructions of a prompt, appended and attended through
    pages, agree with the prefill over the same chunk: both are held to the
    same fp16 bounds, the prefill's rotary and rounding of keys included."""

    gen = torch.Generator().manual_seed(2)
    tables = [torch.randn(2, 16, 2, 256, 8, generator=gen) for _ in range(2)]
    states = [torch.randn(1, 2, 70, 128, generator=gen).half().to(device) for _ in range(2)]
    exits = [jkv.hard_grouped_residual_vq(s, t.to(device), prefixes=(2,))[0][2] for s, t in zip(states, tables)]
    query = torch.randn(1, 8, 70, 128, generator=gen).half().to(device)
    want = jkv.prefill_attention(query, exits[0], exits[1], 0, window=30)
    cache = jkv.PagedKVCache(1, 1, 8, 2, max_length=128, page_size=16, device=device)
    plan = cache.begin([70])
    cache.append(0, plan, *(e[0].transpose(0, 1) for e in exits))
    out = cache.attention(0, plan, query[0].transpose(0, 1), window=30)
    err = (out.float() - want[0].transpose(0, 1).float()).norm() / want.float().norm()
    assert float(err) <= 8 * half_step(torch.float16)


def test_streams_devices_and_graphs(device):
    """On another stream than the default one, and captured: two graphs of one
    pool of memory replayed in turn, with eager work between."""

    batch = Batch(21, [700, 90], [1, 1], qh=8, kvh=2, dim=128)
    args = batch.on(device)
    args["starts"] = None
    chunk = Batch(22, [300, 200], [100, 7], qh=8, kvh=2, dim=128)
    chunk_args = chunk.on(device)
    q1, q2 = batch.query.to(device), chunk.query.to(device)
    w1 = torch.zeros(2, 2, 704, device=device)
    w2 = torch.zeros(2, 2, 304, device=device)

    def one():
        return jkv.paged_attention(q1, **args, window=500, sinks=3, weights=w1, max_length=700)

    def two():
        return jkv.paged_attention(q2, **chunk_args, weights=w2, max_new=100, max_length=300)

    eager = [(f().clone(), w.clone()) for f, w in ((one, w1), (two, w2))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        w1.zero_()
        assert torch.equal(one(), eager[0][0]) and torch.equal(w1, eager[0][1])
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    pool = torch.cuda.graph_pool_handle()
    for f in (one, two):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, pool=pool):
            outs.append(f())
        graphs.append(g)
    for _ in range(4):
        for i, (g, w) in enumerate(zip(graphs, (w1, w2))):
            w.fill_(3.0)
            one() if i else two()
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(outs[i], eager[i][0])
            for b, length in enumerate((batch, chunk)[i].lengths):
                assert torch.equal(w[b, :, :length], eager[i][1][b, :, :length])


def test_pages_beyond_four_gigabytes(device):
    """Offsets that pass 32 bits: the sequence lies at the end of a large pool."""

    page, kvh, dim = 64, 8, 128
    pages = (1 << 32) // (page * kvh * dim * 2) + 40
    print(f"pool of {pages} pages, {2 * pages * page * kvh * dim * 2 >> 30} GiB", flush=True)
    pools = [torch.empty(pages, kvh, page, dim, dtype=torch.float16, device=device) for _ in range(2)]
    length = 300
    for new in (1, 30):
        batch = Batch(31, [length], [new], qh=16, kvh=kvh, dim=dim, page=page)
        count = -(-length // page)
        tables = torch.tensor([[pages - 1 - 7 * i for i in range(count)]], dtype=torch.int32, device=device)
        for pool in pools:
            pool[tables[0].long()] = float("nan")
        lengths = torch.tensor([length], dtype=torch.int32, device=device)
        starts = torch.tensor([0, length], dtype=torch.int32, device=device)
        jkv.paged_append(batch.keys[0].to(device), batch.values[0].to(device), *pools, tables, lengths, starts=starts,
                         rope_theta=None)
        starts = torch.tensor([0, new], dtype=torch.int32, device=device)
        weights = torch.zeros(1, kvh, length, device=device)
        out = jkv.paged_attention(batch.query.to(device), *pools, tables, lengths, starts=starts, window=None,
                                  weights=weights)
        expect = batch.expect(None, 0)
        check_out(out, expect, torch.float16)
        check_weights(weights, expect, [length])
        # and their compaction to other pages there
        kept, _ = jkv.select_entries(weights, lengths, 100)
        moved = torch.tensor([[pages - 3, pages - 4]], dtype=torch.int32, device=device)
        jkv.compact_pages(*pools, tables, kept, moved)
        stay = kept[0, 5].long().cpu()
        got = pools[1][moved[0].long()][:, 5].reshape(-1, dim)[:100].cpu()
        assert torch.equal(got, batch.values[0][stay, 5])


def test_weights_where_heads_times_entries_pass_31_bits(device):
    """2.2 million entries (the same four pages over and over) and 1,024 heads:
    most entries lie far before the window of the new token."""

    length, page, qh, dim, seen = 2_200_000, 4096, 1024, 64, 64
    gen = torch.Generator().manual_seed(41)
    pools = [torch.randn(4, 1, page, dim, generator=gen).to(torch.float16) for _ in range(2)]
    query = torch.randn(1, qh, dim, generator=gen).to(torch.float16)
    width = -(-length // page)
    tables = (torch.arange(width, dtype=torch.int32) % 4)[None]
    at = torch.arange(length - seen, length)
    k, v = (p[at // page % 4, 0, at % page][:, None].double().numpy() for p in pools)
    expect = [ref.attend(query.double().numpy(), k, v, 0, window=seen, sinks=0, theta=None)]
    weights = torch.full((1, 1, length + 3), 7.0, device=device)
    print(f"{length} entries, {qh} heads", flush=True)
    out = jkv.paged_attention(query.to(device), *(p.to(device) for p in pools), tables.to(device),
                              torch.tensor([length], dtype=torch.int32, device=device), window=seen, rope_theta=None,
                              max_length=length, weights=weights)
    check_out(out, expect, torch.float16)
    check_weights(weights[:, :, length - seen :], expect, [seen])
    assert (weights[:, :, : length - seen] == 0).all() and (weights[:, :, length:] == 7.0).all()


def test_two_calls_at_once(device):
    """Two streams with calls in flight over the same pages: each has its own
    workspace."""

    one = Batch(41, [900, 300], [1, 1], qh=8, kvh=2, dim=128)
    two = Batch(42, [500, 90], [60, 9], qh=8, kvh=2, dim=64)
    args = [one.on(device), two.on(device)]
    args[0]["starts"] = None
    queries = [one.query.to(device), two.query.to(device)]
    widths = [torch.zeros(2, 2, 1024, device=device), torch.zeros(2, 2, 1024, device=device)]
    alone = [jkv.paged_attention(q, **a, weights=w).clone() for q, a, w in zip(queries, args, widths)]
    kept = [w.clone() for w in widths]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = [[], []]
    for _ in range(5):
        for i, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                outs[i].append(jkv.paged_attention(queries[i], **args[i], weights=widths[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, alone[i]) for o in outs[i])
        assert torch.equal(widths[i], kept[i])


def test_an_output_may_be_the_query(device):
    for lengths, new in (([900, 300], [1, 1]), ([700, 90], [200, 60])):
        batch = Batch(43, lengths, new, qh=8, kvh=2, dim=128)
        args = batch.on(device)
        query = batch.query.to(device)
        want = jkv.paged_attention(query, **args)
        jkv.paged_attention(query, **args, out=query)
        assert torch.equal(query, want)


def test_bounds_are_kept_where_lengths_are_not(device):
    """Lengths past the table's room or the caller's bound count as that."""

    batch = Batch(44, [96], [1], qh=4, kvh=2, dim=64)
    args = batch.on(device)
    args["starts"] = None
    query = batch.query.to(device)
    want = jkv.paged_attention(query, **args)
    for length in (97, 10 ** 9, 2 ** 31 - 1):
        args["lengths"] = torch.tensor([length], dtype=torch.int32, device=device)
        weights = torch.zeros(1, 2, 96, device=device)
        assert torch.equal(jkv.paged_attention(query, **args, weights=weights), want)
    args["lengths"] = torch.tensor([-5], dtype=torch.int32, device=device)
    assert bool((jkv.paged_attention(query, **args) == 0).all())
    # starts that run past the rows, or backwards, stay inside them
    for starts in ([0, 99], [-7, 1], [1, 0]):
        args["starts"] = torch.tensor(starts, dtype=torch.int32, device=device)
        out = torch.full_like(query, 5.0)
        jkv.paged_attention(query, **args, out=out)
        key = torch.ones(1, 2, 64, dtype=torch.float16, device=device)
        before = args["key_pages"].clone()
        jkv.paged_append(key, key, args["key_pages"], args["value_pages"], args["block_tables"], args["lengths"],
                         starts=args["starts"])
        assert torch.equal(before.view(torch.int16), args["key_pages"].view(torch.int16))


def test_refusals(device):
    batch = Batch(2, [20, 30], [1, 1], qh=4, kvh=2, dim=64)
    args = batch.on(device)
    args["starts"] = None
    query = batch.query.to(device)

    def refused(match, q=query, **change):
        with pytest.raises(ValueError, match=match):
            jkv.paged_attention(q, **{**args, **change})

    refused("type and dims", query.float())
    refused("type and dims", query[:, :, :32])
    refused("multiple of kv heads", query[:, :3])
    refused("one new token a sequence", query[:1])
    refused("starts must be", starts=torch.zeros(2, dtype=torch.int32, device=device))
    refused("starts must be", starts=torch.zeros(3, dtype=torch.int64, device=device))
    refused("lengths must be", lengths=args["lengths"].long())
    refused("positions must be", positions=args["positions"][:1])
    refused("block tables", block_tables=args["block_tables"].long())
    refused("block tables", block_tables=args["block_tables"].t().contiguous().t())
    refused("fp16 or bf16", key_pages=args["key_pages"].float(), value_pages=args["value_pages"].float())
    refused("one shape", value_pages=args["value_pages"][:-1])
    refused("window must be positive", window=0)
    refused("must not be negative", sinks=-1)
    refused("rotary base", rope_theta=-1.0)
    refused("rotary base", rope_theta=float("nan"))
    refused("scale must be finite", scale=float("inf"))
    refused("fewer entries", weights=torch.zeros(2, 2, 20, device=device), max_length=30)
    refused("weights must be fp32", weights=torch.zeros(2, 2, 32, device=device).half())
    refused("must not overlap", weights=torch.zeros(1, 1, 32, device=device).expand(2, 2, 32))
    refused("lse must be", lse=torch.zeros(2, 2, device=device))
    refused("out must match", out=torch.zeros(2, 4, 64, device=device))
    refused("must not overlap", out=torch.zeros(1, 4, 64, dtype=torch.float16, device=device).expand(2, 4, 64))
    page8 = torch.zeros(4, 2, 8, 64, dtype=torch.float16, device=device)
    refused("power of two", key_pages=page8, value_pages=page8.clone())
    page24 = torch.zeros(4, 2, 24, 64, dtype=torch.float16, device=device)
    refused("power of two", key_pages=page24, value_pages=page24.clone())
    dim96 = torch.zeros(4, 2, 16, 96, dtype=torch.float16, device=device)
    refused("head_dim 64 and 128", torch.zeros(2, 4, 96, dtype=torch.float16, device=device), key_pages=dim96,
            value_pages=dim96.clone())
    key = torch.zeros(2, 2, 64, dtype=torch.float16, device=device)
    pools = {k: args[k] for k in ("key_pages", "value_pages", "block_tables", "lengths")}
    with pytest.raises(ValueError, match="pages' type"):
        jkv.paged_append(key.bfloat16(), key.bfloat16(), **pools)
    with pytest.raises(ValueError, match="heads and dims"):
        jkv.paged_append(key[:, :1], key[:, :1], **pools)
    over = torch.zeros(1, 2, 16, 64, dtype=torch.float16, device=device).expand(9, 2, 16, 64)
    with pytest.raises(ValueError, match="must not overlap"):
        jkv.paged_append(key, key, **{**pools, "key_pages": over, "value_pages": over})
    weights = torch.zeros(2, 2, 32, device=device)
    for budget, sinks, recent in ((0, 0, 0), (4, 3, 2), (4, -1, 0)):
        with pytest.raises(ValueError, match="budget"):
            jkv.select_entries(weights, args["lengths"], budget, sinks=sinks, recent=recent)
    with pytest.raises(ValueError, match="kept entries"):
        jkv.compact_pages(args["key_pages"], args["value_pages"], args["block_tables"],
                          torch.zeros(2, 1, 4, dtype=torch.int32, device=device), args["block_tables"])


def test_pools_without_heads_are_refused(device):
    pages = torch.zeros(4, 0, 16, 64, dtype=torch.float16, device=device)
    with pytest.raises(ValueError, match="multiple of kv heads"):
        jkv.paged_attention(torch.zeros(2, 4, 64, dtype=torch.float16, device=device), pages, pages.clone(),
                            torch.zeros(2, 4, dtype=torch.int32, device=device),
                            torch.ones(2, dtype=torch.int32, device=device))


def test_weights_of_scores_that_pass_32_bits(device):
    """Finite keys whose scaled scores pass the largest fp32 number: a row of
    only such scores sees nothing, and its entries' tracked weights stay."""

    for new, length in ((1, 1), (1, 70), (90, 90)):
        batch = Batch(7, [length], [new], qh=4, kvh=2, dim=64, dtype=torch.bfloat16, theta=None)
        batch.query.copy_(batch.query.abs() + 1e5)
        batch.keys[0] = -batch.keys[0].abs() - 1e5
        batch.write(0, batch.keys[0], batch.values[0])
        args = batch.on(device)
        weights = torch.full((1, 2, batch.width * 16), 3.0, device=device)
        out = jkv.paged_attention(batch.query.to(device), **args, window=None, rope_theta=None, scale=1e29,
                                  weights=weights, accumulate=True)
        assert bool((out == 0).all()) and bool((weights == 3.0).all())


def test_a_step_without_new_tokens_stores_zero_weights(device):
    """Entries below the lengths receive nothing: 0 is stored, or added."""

    batch = Batch(6, [40, 0, 17], [0, 0, 0], qh=4, kvh=2, dim=64)
    args = batch.on(device)
    query = torch.zeros(0, 4, 64, dtype=torch.float16, device=device)
    weights = torch.full((3, 2, 48), 7.0, device=device)
    out = jkv.paged_attention(query, **args, weights=weights, accumulate=True)
    assert out.shape == (0, 4, 64) and bool((weights == 7.0).all())
    jkv.paged_attention(query, **args, weights=weights)
    for b, length in enumerate(batch.lengths):
        assert bool((weights[b, :, :length] == 0).all()) and bool((weights[b, :, length:] == 7.0).all())


# ---- infinite and NaN keys and values that rows do see ----

REACHED = [
    # length, new tokens, heads, dims: which kernel and division of the entries
    pytest.param(100, 1, 8, 2, 128, id="one-wave"),
    pytest.param(200, 1, 8, 2, 64, id="waves"),
    pytest.param(200, 5, 8, 2, 128, id="waves-two-groups"),
    pytest.param(900, 1, 4, 2, 128, id="splits"),
    pytest.param(900, 6, 8, 2, 64, id="splits-two-groups"),
    pytest.param(400, 90, 4, 2, 128, id="chunk"),
    pytest.param(5000, 64, 4, 1, 64, id="chunk-splits"),
]


def odd_call(batch, device, exact, **more):
    """Output and weights (where ``exact`` asks for them) of ``batch``, all entries visible."""

    args = batch.on(device)
    weights = torch.zeros(len(batch.lengths), batch.kvh, batch.width * batch.page, device=device) if exact else None
    out = jkv.paged_attention(batch.query.to(device), **args, window=None, rope_theta=batch.theta, weights=weights,
                              max_new=max(batch.new), max_length=max(batch.lengths), **more)
    return out, weights


@pytest.mark.parametrize("exact", [False, True], ids=["out", "weights"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("length,new,qh,kvh,dim", REACHED)
def test_keys_whose_scores_are_minus_infinity_weigh_nothing(device, length, new, qh, kvh, dim, dtype, exact):
    """An entry whose key makes a score of -infinity gets weight 0 and leaves
    the row finite; one that makes +infinity makes it NaN."""

    batch = Batch(length + dim + 1, [length], [new], qh=qh, kvh=kvh, dim=dim, dtype=dtype, theta=None)
    batch.query[:, :, 6] = batch.query[:, :, 6].abs() + 0.25
    batch.query[:, :, 21] = -batch.query[:, :, 21].abs() - 0.25
    batch.queries = [batch.query]
    hidden = [1, 33, 39, 64]  # (all before the new tokens)
    kept = [j for j in range(length) if j not in hidden]
    expect = [ref.attend(batch.query.double().numpy(), batch.keys[0][kept].double().numpy(),
                         batch.values[0][kept].double().numpy(), batch.positions[0], window=None, sinks=0, theta=None)]
    keys = batch.keys[0]
    keys[hidden[:2], :, 6] = float("-inf")
    keys[hidden[2:], :, 21] = float("inf")
    batch.write(0, keys, batch.values[0])
    out, weights = odd_call(batch, device, exact)
    check_out(out, expect, dtype)
    if exact:
        assert bool((weights[0][:, hidden] == 0).all())
        check_weights(weights[:, :, kept], expect, [len(kept)])
    keys[37, kvh - 1, 6] = float("inf")
    batch.write(0, keys, batch.values[0])
    again, _weights = odd_call(batch, device, exact)
    per = qh // kvh
    assert bool(again[:, qh - per :].isnan().all())
    if kvh > 1:
        assert torch.equal(again[:, : qh - per], out[:, : qh - per])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("length,new,dim", [(1, 1, 64), (50, 1, 128), (200, 1, 128), (900, 1, 64), (40, 5, 128),
                                            (80, 80, 64), (400, 90, 128)])
def test_rows_whose_scores_are_all_minus_infinity(device, length, new, dim, dtype):
    """They give 0, a log-sum-exp of -infinity, and no weight to any entry,
    whether the keys or the queries are infinite."""

    for infinite in ("keys", "queries"):
        batch = Batch(length, [length], [new], qh=8, kvh=2, dim=dim, dtype=dtype, theta=None)
        batch.query[:, :, 6] = batch.query[:, :, 6].abs() + 0.25
        batch.keys[0][:, :, 6] = -batch.keys[0][:, :, 6].abs() - 0.25
        (batch.keys[0] if infinite == "keys" else batch.query)[:, :, 6] *= float("inf")
        batch.write(0, batch.keys[0], batch.values[0])
        lse = torch.full((new, 8), 9.0, device=device)
        out, weights = odd_call(batch, device, True, lse=lse)
        assert bool((out == 0).all()) and bool((lse == float("-inf")).all()) and bool((weights == 0).all())
        out, _weights = odd_call(batch, device, False)
        assert bool((out == 0).all())


@pytest.mark.parametrize("exact", [False, True], ids=["out", "weights"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("length,new,qh,kvh,dim", REACHED)
def test_non_finite_values_in_tiles_that_every_row_sees(device, length, new, qh, kvh, dim, dtype, exact):
    """An infinite value that a row sees makes that dim infinite, two of unlike
    sign or a NaN make it NaN, wherever in its tile the entry lies; the other
    dims keep their results."""

    batch = Batch(length + dim, [length], [new], qh=qh, kvh=kvh, dim=dim, dtype=dtype)
    expect = batch.expect(None, 0)
    values = batch.values[0]
    for j in (3, 37, 38, 66):  # (all before the new tokens)
        values[j, 0, 5] = float("inf")
        values[j + 1, 0, 7] = float("-inf")
    values[40, 0, 9] = float("nan")
    values[2, 0, 11], values[70, 0, 11] = float("inf"), float("-inf")
    batch.write(0, batch.keys[0], values)
    out, weights = odd_call(batch, device, exact)
    per, odd = qh // kvh, out[:, : qh // kvh]
    assert bool((odd[:, :, 5] == float("inf")).all()) and bool((odd[:, :, 7] == float("-inf")).all())
    assert bool(odd[:, :, (9, 11)].isnan().all())
    plain = out.clone()
    for d in (5, 7, 9, 11):
        want = torch.from_numpy(expect[0]["out"][:, :per, d])
        plain[:, :per, d] = want.to(device=device, dtype=dtype)
    check_out(plain, expect, dtype)
    if exact:
        check_weights(weights, expect, [length])


@pytest.mark.parametrize("length,new", [(90, 1), (250, 1), (3000, 1), (400, 60), (3000, 60)])
def test_infinite_values_of_entries_that_hardly_count(device, length, new):
    """A weight below what 32 bits hold is still no zero: the infinite value
    that it weighs makes the sum infinite, in one tile as over many."""

    for dtype in (torch.float16, torch.bfloat16):
        batch = Batch(length, [length], [new], qh=2, kvh=1, dim=128, dtype=dtype, theta=None)
        batch.query[:, :, 6] = 8.0
        # scores of the first entries (a whole split, where there are some) lie about 300 below the others'
        batch.keys[0][:, :, 6] = 0.0
        batch.keys[0][: 300 if length > 2000 else 40, :, 6] = -425.0
        batch.values[0][20, 0, 5] = float("inf")
        batch.values[0][21, 0, 7] = float("-inf")
        batch.write(0, batch.keys[0], batch.values[0])
        out, _weights = odd_call(batch, device, False)
        assert bool((out[:, :, 5] == float("inf")).all()) and bool((out[:, :, 7] == float("-inf")).all())
        rest = [d for d in range(128) if d not in (5, 7)]
        assert bool(out[:, :, rest].isfinite().all())


def test_eviction_of_an_almost_full_pool_goes_round_by_round(device):
    """Pages for one sequence's budget are free: three sequences follow one
    another into them, with the same results as in a pool that takes all."""

    kvh, qh, dim = 2, 4, 64
    gen = torch.Generator().manual_seed(44)
    caches = [jkv.PagedKVCache(2, 4, pages, kvh, max_length=128, page_size=16, head_dim=dim, track_weights=True,
                               device=device) for pages in (7 + 4 + 5 + 1 + 2, 40)]
    lengths = [100, 60, 70, 9]
    prompt = [[torch.randn(sum(lengths), heads, dim, generator=gen).half().to(device) for heads in (kvh, kvh, qh)]
              for _ in range(2)]
    single = [[torch.randn(4, heads, dim, generator=gen).half().to(device) for heads in (kvh, kvh, qh)]
              for _ in range(2)]
    outs = []
    for cache in caches:
        step = cache.begin(lengths)
        for layer, (k, v, q) in enumerate(prompt):
            cache.append(layer, step, k, v)
            cache.attention(layer, step, q)
        cache.evict(32, sinks=2, recent=8)
        assert cache.lengths == (32, 32, 32, 9) and cache.positions == (100, 60, 70, 9)
        assert cache.free_pages == cache.key.shape[1] - 7
        cache.release(0)  # (the next entries need pages)
        step = cache.begin([1, 1, 1, 1])
        for layer, (k, v, q) in enumerate(single):
            cache.append(layer, step, k, v)
            outs.append(cache.attention(layer, step, q))
    assert torch.equal(torch.stack(outs[:2]), torch.stack(outs[2:]))
    for few, many in zip(*(c.weights for c in caches)):
        assert torch.equal(few, many)


# ---- how exact the few-row and the weighing kernels are, and the kernels of larger calls ----


def check_parts(out, expect, dtype, p_parts):
    """As :func:`check_out` for a q in two 16-bit parts, and a p in ``p_parts``
    of them.  Two parts hold a number to h^2 of itself: 2^-16 in bf16; in fp16
    2^-22, or 2^-25 for parts that are subnormal, which the rotation's sine and
    cosine (2^-20) and these queries' sizes keep under 2^-18.  The outputs' own
    rounding is off by h / sqrt(3) of a number's power of two, 0.39 h of its size
    where mantissas spread evenly over their logarithm; a p of one part would
    bring as much again, 0.55 h in all."""

    h, slack = half_step(dtype), 2.0 ** -20
    part = 2.0 ** -16 if dtype == torch.bfloat16 else 2.0 ** -18
    got = out.detach().double().cpu().numpy()
    want = np.concatenate([e["out"] for e in expect])
    spread = np.concatenate([e["spread"] for e in expect])
    reach = np.concatenate([e["reach"] for e in expect])[..., None]
    p_error = h if p_parts == 1 else part
    tol = h * np.abs(want) + spread * (p_error + np.expm1(2 * (part + slack) * reach) + slack) * (1 + h)
    err = np.abs(got - want)
    worst = np.unravel_index(np.argmax(err - tol), err.shape)
    assert (err <= tol + float(torch.finfo(dtype).tiny)).all(), f"error {err[worst]} over {tol[worst]} at {worst}"
    rel = np.linalg.norm(err) / np.linalg.norm(want)
    assert rel <= (0.45 if p_parts == 2 else 0.65) * h, f"relative error {rel / h} h"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("length,new,qh,window,sinks", [
    (100, 1, 32, None, 0), (200, 1, 32, None, 0), (900, 1, 32, None, 0), (9000, 1, 32, None, 0), (900, 1, 32, 300, 40),
    (100, 5, 8, None, 0), (200, 5, 8, None, 0), (900, 5, 8, None, 0), (9000, 8, 8, 5000, 3)])
def test_few_rows_keep_queries_and_weights_in_two_parts(device, length, new, qh, dim, window, sinks, dtype):
    """In one wave, in waves that join, in splits, in one and two groups of rows:
    what is left is the output's rounding."""

    batch = Batch(length + new, [length], [new], qh=qh, kvh=2, dim=dim, page=64, dtype=dtype)
    out = jkv.paged_attention(batch.query.to(device), **batch.on(device), window=window, sinks=sinks, max_new=new,
                              max_length=length)
    check_parts(out, batch.expect(window, sinks), dtype, 2)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("length,new,dim", [(400, 90, 128), (300, 300, 64), (5000, 64, 64)])
def test_chunks_that_weigh_keep_queries_in_two_parts(device, length, new, dim, dtype):
    batch = Batch(length + new, [length], [new], qh=4, kvh=2, dim=dim, page=64, dtype=dtype)
    expect = batch.expect(None, 0)
    query, args = batch.query.to(device), batch.on(device)
    lse = torch.empty(new, 4, device=device)
    weights = torch.empty(1, 2, length, device=device)
    for more in (dict(lse=lse), dict(weights=weights)):
        out = jkv.paged_attention(query, **args, window=None, max_new=new, max_length=length, **more)
        check_parts(out, expect, dtype, 1)


def check_some_heads(device, batch, groups, window, sinks):
    """Output, weights and log-sum-exps of a larger call, with weights and
    without, for the kv heads ``groups`` (the oracle takes a row at a time)."""

    per, length = batch.qh // batch.kvh, max(batch.lengths)
    query, args = batch.query.to(device), batch.on(device)
    weights = torch.full((len(batch.lengths), batch.kvh, length), 7.0, device=device)
    lse = torch.empty(len(query), batch.qh, device=device)
    bounds = dict(window=window, sinks=sinks, max_new=max(batch.new), max_length=length)
    plain = jkv.paged_attention(query, **args, **bounds)
    exact = jkv.paged_attention(query, **args, **bounds, weights=weights, lse=lse)
    for g in groups:
        heads = slice(per * g, per * g + per)
        expect = [ref.attend(q[:, heads].double().numpy(), k[:, g : g + 1].double().numpy(),
                             v[:, g : g + 1].double().numpy(), p, window=window, sinks=sinks, theta=batch.theta)
                  for q, k, v, p in zip(batch.queries, batch.keys, batch.values, batch.positions)]
        check_out(plain[:, heads], expect, batch.dtype)
        check_parts(exact[:, heads], expect, batch.dtype, 1)
        check_weights(weights[:, g : g + 1], expect, batch.lengths)
        want = np.concatenate([e["lse"] for e in expect])
        reach = np.concatenate([e["reach"] for e in expect])
        got = lse[:, heads].double().cpu().numpy()
        assert (np.abs(got - want) <= 2.0 ** -17 * reach + 2.0 ** -19 * (1 + np.abs(want))).all()
    for b, n in enumerate(batch.lengths):
        assert bool((weights[b, :, n:] == 7.0).all()), "weights behind the last entry were written"


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("window,sinks", [(None, 0), (700, 20)])
def test_blocks_of_eight_waves(device, window, sinks, dtype):
    """Two ragged chunks of 32 groups of two heads: 256 blocks of 256 rows, one
    a CU, whose last ones hold 232 and 132 rows; weights of 128 entries a
    workgroup, whose last ones hold 76 and 4."""

    batch = Batch(61, [1100, 900], [500, 450], qh=64, kvh=32, dim=128, page=64, dtype=dtype)
    check_some_heads(device, batch, (0, 13, 31), window, sinks)


@pytest.mark.parametrize("dim", [64, 128])
def test_blocks_that_are_resident_at_once_run_in_folded_order(device, dim):
    """Prompts of unlike lengths, one of them idle, in blocks of 128 rows: between
    one and two workgroups a CU, and more row blocks than the order keeps from
    the front."""

    batch = Batch(62, [300, 17, 9, 257], [300, 17, 0, 257], qh=64, kvh=64, dim=dim, page=16)
    check_some_heads(device, batch, (0, 40, 63), None, 0)


def test_the_second_walk_of_eight_waves_changes_only_what_is_infinite(device):
    """An infinite value in blocks of 256 rows: the dim that holds it becomes
    infinite, the others keep every bit."""

    batch = Batch(61, [1100, 900], [500, 450], qh=64, kvh=32, dim=128, page=64)
    query = batch.query.to(device)
    weights = [torch.zeros(2, 32, 1100, device=device) for _ in range(2)]
    bounds = dict(window=None, max_new=500, max_length=1100)
    clean = [jkv.paged_attention(query, **batch.on(device), **bounds, weights=w) for w in (None, weights[0])]
    batch.values[0][100, 4, 77] = float("-inf")
    batch.write(0, batch.keys[0][:101], batch.values[0][:101])
    odd = [jkv.paged_attention(query, **batch.on(device), **bounds, weights=w) for w in (None, weights[1])]
    for was, now in zip(clean, odd):
        assert bool((now[:500, 8:10, 77] == float("-inf")).all())
        now[:500, 8:10, 77] = was[:500, 8:10, 77]
        assert torch.equal(was, now)
    assert torch.equal(*weights)


@pytest.mark.parametrize("length", [250, 3000])
def test_parts_that_hardly_count_add_nothing(device, length):
    """Huge finite values in splits whose weights 32 bits do not hold."""

    batch = Batch(length, [length], [1], qh=2, kvh=1, dim=128, dtype=torch.bfloat16, theta=None)
    batch.query[:, :, 6] = 8.0
    batch.queries = [batch.query]
    low = 300 if length > 2000 else 40
    batch.keys[0][:, :, 6] = 0.0
    batch.keys[0][:low, :, 6] = -425.0
    # (a split's sums hold up to 2^14 weights' worth of them)
    batch.values[0][:low, :, 9] = 2.0 ** 100
    batch.write(0, batch.keys[0], batch.values[0])
    expect = batch.expect(None, 0)
    for e in expect:  # what is left of them in 64 bits is below 1e-90
        assert np.abs(e["out"]).max() < 10
    out, _weights = odd_call(batch, device, False)
    check_out(out, expect, torch.bfloat16)

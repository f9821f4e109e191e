"""Attention of packed sequences on the MI355X against 64-bit definitions."""

from __future__ import annotations

import pytest
import torch

import jointkv_amd as jkv
from oracle import shaped_oracle as ref
from tests.test_gpu_paged import half_step
from tests.test_gpu_paged_shaped import score_slack, slopes_of

pytestmark = pytest.mark.gpu


class Texts:
    """Packed random sequences; rows outside them hold NaN."""

    def __init__(self, seed, sizes, qh, kvh, dim, dtype, *, lead=0, tail=0, gain=1.0, grad_gain=1.0):
        gen = torch.Generator().manual_seed(seed)
        rows = lead + sum(sizes) + tail
        self.sizes, self.dtype, self.dim = sizes, dtype, dim
        self.q = (torch.randn(rows, qh, dim, generator=gen) * gain).to(dtype)
        self.k = (torch.randn(rows, kvh, dim, generator=gen) * gain).to(dtype)
        self.v = torch.randn(rows, kvh, dim, generator=gen).to(dtype)
        self.d = (torch.randn(rows, qh, dim, generator=gen) * grad_gain).to(dtype)
        starts = [lead]
        for n in sizes:
            starts.append(starts[-1] + n)
        self.spans = list(zip(starts, starts[1:]))
        self.starts = torch.tensor(starts, dtype=torch.int32)
        self.owned = torch.zeros(rows, dtype=torch.bool)
        self.owned[lead : starts[-1]] = True
        for x in (self.q, self.k, self.v, self.d):
            x[~self.owned] = float("nan")

    def expect(self, *, prefixes=None, grads=False, **form):
        prefixes = prefixes or [0] * len(self.sizes)
        return [ref.attend(self.q[a:b], self.k[a:b], self.v[a:b], prefix=p, d_out=self.d[a:b] if grads else None, **form)
                for (a, b), p in zip(self.spans, prefixes)]


def check_out(texts, out, results, cap=None, slopes=None, lse=None):
    h = half_step(texts.dtype)
    out = out.detach().cpu().double()
    assert (out[~texts.owned] == 0).all()
    if lse is not None:
        assert (lse[~texts.owned.to(lse.device)] == float("-inf")).all()
    for (a, b), r in zip(texts.spans, results):
        off = score_slack(r, texts.dim, cap, slopes, b - a) * 2
        bound = h * r["out"].abs() + (h + off[..., None]) * r["spread"] * 1.01 + 1e-6 * r["spread"] + 2.0**-24
        assert ((out[a:b] - r["out"]).abs() <= bound).all()
        if lse is not None:
            assert ((lse[a:b].cpu().double() - r["lse"]).abs() <= off + 2.0**-21 * (1 + r["lse"].abs())).all()


SHAPES = [
    ([1], 4, 4, 128, None, 0),
    ([1, 1, 2, 1], 4, 2, 64, None, 0),
    ([31, 1, 64, 0, 33, 128], 8, 2, 128, None, 0),
    ([200, 77], 7, 1, 64, 50, 0),
    ([300, 129], 5, 5, 128, 64, 3),
    ([700], 2, 1, 64, 100, 130),
    ([257, 255, 256], 12, 4, 128, None, 0),
]
FORMS = [dict(), dict(cap=15.0), dict(bias=True), dict(prefix=True), dict(cap=50.0, bias=True, prefix=True)]
NAMES = ["plain", "cap", "bias", "prefix", "all"]


def form_of(texts, form, qh, device):
    slopes = slopes_of(qh) if form.get("bias") else None
    prefixes = [n * 2 // 3 if i % 2 == 0 else n + 5 for i, n in enumerate(texts.sizes)] if form.get("prefix") else None
    want = dict(cap=form.get("cap"), slopes=slopes, prefixes=prefixes)
    call = dict(softcap=form.get("cap"), slopes=None if slopes is None else slopes.to(device),
                prefixes=None if prefixes is None else torch.tensor(prefixes, dtype=torch.int32, device=device))
    return want, call


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,qh,kvh,dim,window,sinks", SHAPES)
def test_forward(device, form, dtype, sizes, qh, kvh, dim, window, sinks):
    texts = Texts(sum(sizes), sizes, qh, kvh, dim, dtype, lead=3, tail=40, gain=2.0)
    want, call = form_of(texts, form, qh, device)
    lse = torch.zeros(texts.q.shape[:2], device=device)
    args = [x.to(device) for x in (texts.q, texts.k, texts.v, texts.starts)]
    out = jkv.packed_attention(*args, window=window, sinks=sinks, lse=lse, **call)
    check_out(texts, out, texts.expect(window=window, sinks=sinks, **want), want["cap"], want["slopes"], lse)
    assert torch.equal(jkv.packed_attention(*args, window=window, sinks=sinks, **call), out)


def test_masked_rows_may_hold_anything(device):
    """What lies behind a row, in its own sequence too, does not reach it."""

    texts = Texts(4, [150, 90], 4, 2, 64, torch.float16)
    args = [x.to(device) for x in (texts.q, texts.k, texts.v, texts.starts)]
    clean = jkv.packed_attention(*args, window=40)
    for bad in (float("inf"), float("-inf"), float("nan")):
        k, v = args[1].clone(), args[2].clone()
        k[100], v[100] = bad, bad
        out = jkv.packed_attention(args[0], k, v, args[3], window=40)
        assert torch.equal(out[:100], clean[:100]) and torch.equal(out[140:], clean[140:])
        v2 = args[2].clone()
        v2[100, 0, 3] = bad  # one dim of the values that rows 100 to 139 see
        out = jkv.packed_attention(args[0], args[1], v2, args[3], window=40)
        assert not torch.isfinite(out[100:140, :2, 3]).any()
        out[100:140, :2, 3] = clean[100:140, :2, 3]
        assert torch.equal(out, clean)


def test_strides_and_given_outputs(device):
    texts = Texts(5, [60, 70], 4, 2, 128, torch.bfloat16)
    q, k, v, starts = (x.to(device) for x in (texts.q, texts.k, texts.v, texts.starts))
    want = jkv.packed_attention(q, k, v, starts)
    qkv = torch.cat((q, k, v), 1)  # one projection's output
    assert torch.equal(jkv.packed_attention(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], starts), want)
    heads_first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    assert torch.equal(jkv.packed_attention(*heads_first, starts), want)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=device)[1:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(jkv.packed_attention(odd, k, v, starts), want)
    out = torch.zeros(130, 6, 128, dtype=q.dtype, device=device)
    given = jkv.packed_attention(q, k, v, starts, out=out[:, 1:5])
    assert torch.equal(given, want) and (out[:, 0] == 0).all() and (out[:, 5] == 0).all()
    one = jkv.packed_attention(q, k[:, :1].expand(130, 2, 128), v, starts)
    assert torch.equal(one, jkv.packed_attention(q, k[:, :1].repeat(1, 2, 1), v, starts))
    assert jkv.packed_attention(q[:0], k[:0], v[:0], torch.zeros(3, dtype=torch.int32, device=device)).shape == (0, 4, 128)
    nobody = jkv.packed_attention(q, k, v, torch.zeros(1, dtype=torch.int32, device=device))
    assert (nobody == 0).all()


def test_agrees_with_the_paged_form(device):
    """The same rows through pages: one definition, both within its bounds."""

    texts = Texts(6, [90], 4, 2, 64, torch.float16)
    q, k, v, starts = (x.to(device) for x in (texts.q, texts.k, texts.v, texts.starts))
    out = jkv.packed_attention(q, k, v, starts, softcap=20.0, window=30, sinks=2)
    cache = jkv.PagedKVCache(1, 1, 8, 2, max_length=100, page_size=16, head_dim=64, device=device)
    step = cache.begin([90])
    cache.append(0, step, k, v, rope_theta=None)
    paged = cache.attention(0, step, q, window=30, sinks=2, rope_theta=None, softcap=20.0)
    assert torch.equal(out, paged)


def check_grads(texts, grads, results, cap=None, slopes=None):
    """Each gradient's own rounding h; p and ds rounded to h each (``slack`` holds
    sum p |do|, and of ds p (|delta| + 2 |dp - delta|): its rounding, p's own
    error in it and delta's, whose o is rounded); scores off as in the forward, which
    p takes on twice; 32-bit sums of the products, D + rows of them, 2^-23 of a
    term's size each.  fp16 holds p to 2^-34 of the largest and ds to 2^-24 of 2^15
    over 2^10 and what inputs of their sizes could give."""

    h = half_step(texts.dtype)
    for name, got, size in zip(("dq", "dk", "dv"), grads, ("dq_size", "dk_size", "dv_size")):
        got = got.detach().cpu().double()
        assert (got[~texts.owned] == 0).all()
        for (a, b), r in zip(texts.spans, results):
            if a == b:
                continue
            off = float(score_slack(r, texts.dim, cap, slopes, b - a).max()) * 2 + (texts.dim + b - a) * 2.0**-23
            if cap:
                off += 2.0**-21  # of the cap's slope
            bound = h * r[name].abs() + (h + 2.0**-22) * r[name + "_slack"] + off * r[size] + 1e-7 * r[size].max() + 2.0**-24
            assert ((got[a:b] - r[name]).abs() <= bound).all(), (name, ((got[a:b] - r[name]).abs() / bound).max())


def run_grads(texts, device, **call):
    q, k, v = (x.to(device).requires_grad_() for x in (texts.q, texts.k, texts.v))
    out = jkv.packed_attention(q, k, v, texts.starts.to(device), **call)
    return out, torch.autograd.grad(out, (q, k, v), texts.d.to(device))


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,qh,kvh,dim,window,sinks", SHAPES)
def test_gradients(device, form, dtype, sizes, qh, kvh, dim, window, sinks):
    texts = Texts(sum(sizes) + 1, sizes, qh, kvh, dim, dtype, lead=5, tail=9, gain=1.5)
    want, call = form_of(texts, form, qh, device)
    out, grads = run_grads(texts, device, window=window, sinks=sinks, **call)
    results = texts.expect(window=window, sinks=sinks, grads=True, **want)
    check_out(texts, out, results, want["cap"], want["slopes"])
    check_grads(texts, grads, results, want["cap"], want["slopes"])
    again = run_grads(texts, device, window=window, sinks=sinks, **call)[1]
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("bad", [float("inf"), float("-inf"), float("nan")])
def test_gradients_beside_odd_rows(device, dtype, dim, bad):
    """An infinite or NaN row reaches what sees it or is seen by it, and in its own
    sequence nothing else: in tiles with masked places too."""

    texts = Texts(9, [150, 200], 4, 2, dim, dtype)
    args = dict(window=20, softcap=30.0)
    _, clean = run_grads(texts, device, **args)
    at = 150 + 90  # row 90 of the second sequence
    near = slice(at - 19, at + 20)  # rows and places within its window, both ways
    far = torch.ones(350, dtype=torch.bool, device=device)
    far[near] = False
    for name in ("q", "k", "v", "d"):
        odd = Texts(9, [150, 200], 4, 2, dim, dtype)
        getattr(odd, name)[at] = bad
        _, grads = run_grads(odd, device, **args)
        # a query or gradient row changes itself and the 20 places it sees; those that
        # share a row with a changed one take it over: a key or value changes the 20
        # rows that see it, and so what these see
        reach = {"q": (at - 19, at + 1), "d": (at - 19, at + 1), "k": (at - 19, at + 20), "v": (at - 19, at + 20)}[name]
        same = torch.ones(350, dtype=torch.bool, device=device)
        same[reach[0] : reach[1]] = False
        for got, want in zip(grads, clean):
            assert torch.equal(got[same], want[same]), name
        if name == "d" and bad != bad:
            assert not torch.isfinite(grads[2][at].float()).any()


@pytest.mark.parametrize("dtype,form", [(torch.float16, 4), (torch.bfloat16, 1), (torch.bfloat16, 2)])
@pytest.mark.parametrize("sizes,qh,kvh,dim,window,sinks", [
    ([600], 16, 2, 128, None, 0),             # heads in splits, whose sums are joined
    ([350, 90], 40, 2, 64, None, 0),
    ([400], 6, 1, 128, 100, 4),
    ([270, 150] * 8, 12, 12, 128, None, 0),   # 128 keys a workgroup, all heads
    ([290, 220] * 16, 24, 24, 64, 120, 0),
])
def test_gradients_of_every_division(device, dtype, form, sizes, qh, kvh, dim, window, sinks):
    texts = Texts(len(sizes), sizes, qh, kvh, dim, dtype, lead=1, tail=3, gain=1.5)
    want, call = form_of(texts, FORMS[form], qh, device)
    out, grads = run_grads(texts, device, window=window, sinks=sinks, **call)
    results = texts.expect(window=window, sinks=sinks, grads=True, **want)
    check_out(texts, out, results, want["cap"], want["slopes"])
    check_grads(texts, grads, results, want["cap"], want["slopes"])
    again = run_grads(texts, device, window=window, sinks=sinks, **call)[1]
    assert all(torch.equal(x, y) for x, y in zip(grads, again))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-6, 1e4])
def test_gradients_of_small_and_large_losses(device, dtype, size):
    """fp16 gradients of a loss that was divided, or multiplied, by much: ds keeps
    its digits (its scale follows the largest of do and v)."""

    texts = Texts(12, [100, 60], 4, 2, 64, dtype)
    texts.d = (texts.d.float() * (size if dtype == torch.bfloat16 or size > 1 else 1e-3)).to(dtype)
    out, grads = run_grads(texts, device, softcap=20.0)
    results = texts.expect(grads=True, cap=20.0)
    h = half_step(dtype)
    for name, got in zip(("dq", "dk", "dv"), grads):
        want = torch.cat([r[name] for r in results])
        size_of = torch.cat([r[name + "_size"] for r in results])
        slack = torch.cat([r[name + "_slack"] for r in results])
        # as in check_grads; fp16 results below 2^-14 are 2^-25 off
        off = h * want.abs() + (h + 2.0**-22) * slack + 2.0**-12 * size_of + (2.0**-25 if dtype == torch.float16 else 1e-30)
        got = got.cpu().double()
        right = (got - want).abs() <= off
        # (65,504 and half a step of 2^5 on, fp16 rounds to infinity)
        right |= torch.isinf(got) & (got.sign() == want.sign()) & (want.abs() + off >= torch.finfo(dtype).max * (1 + h / 2))
        assert int((~right).sum()) == 0, name


def test_which_gradients_are_asked_for(device):
    texts = Texts(13, [90, 40], 4, 2, 64, torch.bfloat16, tail=5)
    _, all_of = run_grads(texts, device)
    names = ("q", "k", "v")
    for wanted in (("q",), ("k",), ("v",), ("q", "v")):
        x = {n: getattr(texts, n).to(device).requires_grad_(n in wanted) for n in names}
        out = jkv.packed_attention(x["q"], x["k"], x["v"], texts.starts.to(device))
        grads = torch.autograd.grad(out, [x[n] for n in wanted], texts.d.to(device))
        for n, g in zip(wanted, grads):
            assert torch.equal(g, all_of[names.index(n)]), n
    # leaves, strided inputs and a broadcast gradient
    qkv = torch.cat((texts.q, texts.k, texts.v), 1).to(device).requires_grad_()
    out = jkv.packed_attention(qkv[:, :4], qkv[:, 4:6], qkv[:, 6:], texts.starts.to(device))
    out.sum().backward()
    x = [getattr(texts, n).to(device).requires_grad_() for n in names]
    whole = jkv.packed_attention(*x, texts.starts.to(device))
    grads = torch.autograd.grad(whole, x, torch.ones_like(whole))
    assert torch.equal(qkv.grad, torch.cat(grads, 1))
    # one kv head seen as two: its gradient is their sum, rounded as they are
    k1 = texts.k[:, :1].to(device).requires_grad_()
    out = jkv.packed_attention(x[0].detach(), k1.expand(135, 2, 64), x[2].detach(), texts.starts.to(device))
    g1 = torch.autograd.grad(out, k1, texts.d.to(device))[0]
    k2 = texts.k[:, :1].repeat(1, 2, 1).to(device).requires_grad_()
    out = jkv.packed_attention(x[0].detach(), k2, x[2].detach(), texts.starts.to(device))
    g2 = torch.autograd.grad(out, k2, texts.d.to(device))[0]
    assert torch.equal(g1, g2.sum(1, keepdim=True))


def test_a_second_derivative_is_refused(device):
    texts = Texts(14, [30], 2, 2, 64, torch.float16)
    q = texts.q.to(device).requires_grad_()
    out = jkv.packed_attention(q, texts.k.to(device), texts.v.to(device), texts.starts.to(device))
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(out.float().pow(2).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="second derivative"):
        torch.autograd.grad(jkv.rotary(q).float().pow(2).sum(), q, create_graph=True)


def test_two_streams_and_graph_replays(device):
    """Two calls at once on streams of their own, and a captured training step
    replayed beside eager calls."""

    texts = [Texts(s, [100, 50], 4, 2, 64, torch.float16) for s in (15, 16)]
    want = [run_grads(t, device, softcap=30.0) for t in texts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in texts]
    got = []
    for s, t in zip(streams, texts):
        with torch.cuda.stream(s):
            got.append(run_grads(t, device, softcap=30.0))
    torch.cuda.synchronize()
    for (o, g), (wo, wg) in zip(got, want):
        assert torch.equal(o, wo) and all(torch.equal(x, y) for x, y in zip(g, wg))
    held = [x.to(device) for x in (texts[0].q, texts[0].k, texts[0].v, texts[0].d)]
    leaves = [x.clone().requires_grad_() for x in held[:3]]
    starts = texts[0].starts.to(device)

    def step():
        out = jkv.packed_attention(*leaves, starts, softcap=30.0)
        return out.detach(), torch.autograd.grad(out, leaves, held[3])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, grads = step()
    for n in (1, 0, 1):
        with torch.no_grad():
            for x, source in zip((*leaves, held[3]), (texts[n].q, texts[n].k, texts[n].v, texts[n].d)):
                x.copy_(source)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[n][0]) and all(torch.equal(x, y) for x, y in zip(grads, want[n][1]))
        run_grads(texts[n], device, softcap=30.0)


def test_a_step_from_turned_queries_to_gradients(device):
    """Rotary, attention and their gradients together, against differences of the
    64-bit definition along random directions."""

    texts = Texts(17, [40, 25], 4, 2, 64, torch.bfloat16)
    rule = jkv.RotaryRule(layout="interleaved", dims=32, scaling="linear", factor=2.0)
    q, k, v = (x.to(device).requires_grad_() for x in (texts.q, texts.k, texts.v))
    starts = texts.starts.to(device)
    tq, tk = jkv.rotary(q, k, rule, starts=starts)
    out = jkv.packed_attention(tq, tk, v, starts, softcap=10.0, window=30)
    grads = torch.autograd.grad(out, (q, k, v), texts.d.to(device))
    rates = ref.rates(32, 10000.0, "linear", 2.0)
    at = list(range(40)) + list(range(25))

    def loss(q, k, v):
        total = 0.0
        q, k = (ref.turn(x, at, rates, layout="interleaved") for x in (q, k))
        for a, b in texts.spans:
            total += (ref.attend(q[a:b], k[a:b], v[a:b], window=30, cap=10.0)["out"] * texts.d[a:b].double()).sum()
        return float(total)

    gen = torch.Generator().manual_seed(1)
    x = [t.double() for t in (texts.q, texts.k, texts.v)]
    for i, g in enumerate(grads):
        way = torch.randn(x[i].shape, generator=gen, dtype=torch.float64)
        step = 1e-4
        moved = [[t + (s * step * way if j == i else 0) for j, t in enumerate(x)] for s in (1, -1)]
        slope = (loss(*moved[0]) - loss(*moved[1])) / (2 * step)
        # bf16 inputs to the products and results: four roundings of 2^-9 in the mean square over
        # all elements' sum, here at eight times its size
        size = float((g.cpu().double() * way).pow(2).sum().sqrt())
        assert abs(float((g.cpu().double() * way).sum()) - slope) <= 8 * 2.0**-8 * size + 1e-3 * abs(slope)


@pytest.mark.parametrize("form", FORMS, ids=NAMES)
@pytest.mark.parametrize("scale", [0.0, -0.2, 1.5])
def test_scales(device, form, scale):
    """Any scale, a negative one and none at all."""

    texts = Texts(18, [100, 70], 4, 2, 64, torch.float16, gain=0.7)
    want, call = form_of(texts, form, 4, device)
    out, grads = run_grads(texts, device, scale=scale, window=60, **call)
    results = texts.expect(scale=scale, window=60, grads=True, **want)
    check_out(texts, out, results, want["cap"], want["slopes"])
    check_grads(texts, grads, results, want["cap"], want["slopes"])
    if not form:
        return  # (a paged call of plain scores rounds the scaled queries: tested with the others)
    pages = jkv.PagedKVCache(1, 2, 20, 2, max_length=100, page_size=16, head_dim=64, device=device)
    step = pages.begin([100, 70])
    pages.append(0, step, texts.k.to(device), texts.v.to(device), rope_theta=None)
    paged = pages.attention(0, step, texts.q.to(device), rope_theta=None, scale=scale, window=60, **call)
    check_out(texts, paged, results, want["cap"], want["slopes"])


@pytest.mark.parametrize("cap,bias", [(None, False), (7.0, False), (None, True), (20.0, True)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128])
def test_a_row_that_sees_one_entry(device, dtype, dim, cap, bias):
    """Its output is the value itself, its score has no gradient.

    The rounded weight divides itself out, and the quotient's 2^-22 is far below half a
    step.  do v and do out are sums of dim products in 32 bits, the second one of two
    parts whose second is rounded (2^-8 of 2^-22): they differ by at most (3 dim + 8)
    2^-24 of the products' magnitudes; ds may round to twice its value, and dq and dk
    add half a step of the smallest numbers.
    """
    texts = Texts(31, [150, 1, 64], 6, 2, dim, dtype, gain=2.0)
    slopes = slopes_of(6).to(device) if bias else None
    q, k, v = (x.to(device).requires_grad_() for x in (texts.q, texts.k, texts.v))
    scale = dim**-0.5
    for training in (False, True):
        with torch.set_grad_enabled(training):
            out = jkv.packed_attention(q, k, v, texts.starts.to(device), softcap=cap, slopes=slopes, window=1)
        torch.testing.assert_close(out.detach().cpu(), texts.v.repeat_interleave(3, dim=1), rtol=0, atol=0)
    out.backward(texts.d.to(device))
    d, key, query = texts.d.double(), texts.k.double().repeat_interleave(3, dim=1), texts.q.double()
    ds = 2 * (3 * dim + 8) * 2.0**-24 * (d * texts.v.double().repeat_interleave(3, dim=1)).abs().sum(-1, keepdim=True)
    least = 2.0**-25 if dtype == torch.float16 else 0.0
    assert (q.grad.cpu().double().abs() <= ds * scale * key.abs() + least).all()
    grouped = (ds * scale * query.abs()).reshape(-1, 2, 3, dim).sum(2)
    assert (k.grad.cpu().double().abs() <= grouped + least).all()
    # p is within 2^-18 of 1 (its score's fraction in 32 bits) and rounds to 1 or beside
    # it; three heads' sum, then half a step
    h = half_step(dtype)
    sums, sizes = d.reshape(-1, 2, 3, dim).sum(2), d.abs().reshape(-1, 2, 3, dim).sum(2)
    assert ((v.grad.cpu().double() - sums).abs() <= h * sums.abs() + (h + 2.0**-18) * 1.01 * sizes + least).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_rows_without_sequences(device, dtype):
    texts = Texts(32, [], 4, 2, 64, dtype, lead=70)
    x = [t.to(device).requires_grad_() for t in (texts.q, texts.k, texts.v)]
    lse = torch.zeros(70, 4, device=device)
    out = jkv.packed_attention(*x, texts.starts.to(device), lse=lse)
    assert (out == 0).all() and (lse == float("-inf")).all()
    out.backward(texts.d.to(device))
    assert all((t.grad == 0).all() for t in x)
    none = [t.detach()[:0].requires_grad_() for t in x]
    out = jkv.packed_attention(*none, torch.zeros(3, dtype=torch.int32, device=device))
    out.sum().backward()
    assert out.shape == (0, 4, 64) and all(t.grad.shape == t.shape for t in none)


def test_rows_past_32_bits(device):
    """Rows 2^22 bytes apart give what rows one behind another give."""
    texts = Texts(33, [600, 440], 4, 2, 64, torch.float16)
    far = torch.zeros(1040, 1 << 21, dtype=torch.float16, device=device)
    starts = texts.starts.to(device)
    near = [t.to(device) for t in (texts.q, texts.k, texts.v, texts.d)]
    apart, at = [], 0
    for t in near:
        place = far[:, at : at + t[0].numel()].view(t.shape)
        place.copy_(t)
        apart.append(place)
        at += t[0].numel()
    results = []
    for q, k, v, d in (near, apart):
        q, k, v = (t.detach().requires_grad_() for t in (q, k, v))
        assert q.stride(0) in (256, 1 << 21)
        out = jkv.packed_attention(q, k, v, starts, softcap=20.0)
        results.append((out.detach(), *torch.autograd.grad(out, (q, k, v), d)))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    target = far[:, at : at + 256].view(1040, 4, 64)
    jkv.packed_attention(*(t.detach() for t in apart[:3]), starts, softcap=20.0, out=target)
    assert torch.equal(target, results[0][0])
    turned = [jkv.rotary(t, starts=starts) for t in (near[0], apart[0])]
    assert torch.equal(*turned)
    jkv.rotary(apart[0], starts=starts, out=target)
    assert torch.equal(target, turned[0])


@pytest.mark.parametrize("form", [FORMS[0], FORMS[4]], ids=["plain", "all"])
@pytest.mark.parametrize("sizes,qh,kvh,dim", [
    ([17, 0, 40, 1, 33] * 15, 2, 1, 64),  # more than 64 sequences
    ([5, 2200, 130], 1, 1, 64),  # one of more than 64 blocks of keys
    ([300, 700, 0, 500], 24, 8, 64),  # few, in an order of lengths, two workgroups a CU
])
def test_orders_of_the_blocks(device, form, sizes, qh, kvh, dim):
    texts = Texts(34, sizes, qh, kvh, dim, torch.bfloat16, lead=2, tail=3)
    want, call = form_of(texts, form, qh, device)
    out, grads = run_grads(texts, device, **call)
    results = texts.expect(grads=True, **want)
    check_out(texts, out, results, want["cap"], want["slopes"])
    check_grads(texts, grads, results, want["cap"], want["slopes"])


def test_buffers_given_beside_autograd(device):
    """An lse buffer may serve two calls before the first's backward; what a kernel
    writes over a saved tensor makes the backward refuse."""
    texts = Texts(35, [40, 90], 4, 2, 64, torch.float16)
    starts, d = texts.starts.to(device), texts.d.to(device)
    x = [t.to(device).requires_grad_() for t in (texts.q, texts.k, texts.v)]
    want = torch.autograd.grad(jkv.packed_attention(*x, starts), x, d)
    lse = torch.empty(130, 4, device=device)
    first = jkv.packed_attention(*x, starts, lse=lse)
    held = lse.clone()
    jkv.packed_attention(*x, starts, softcap=5.0, lse=lse)
    assert not torch.equal(held, lse)
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(first, x, d), want))

    out = jkv.packed_attention(*x, starts)
    with torch.no_grad():
        jkv.packed_attention(*x, starts, softcap=5.0, out=out)
    with pytest.raises(RuntimeError, match="inplace"):
        out.backward(d)
    y = x[0].sigmoid()  # (its backward takes its output)
    with torch.no_grad():
        jkv.rotary(y, starts=starts, out=y)
    with pytest.raises(RuntimeError, match="inplace"):
        y.sum().backward()
    with torch.inference_mode():
        z = x[0].clone()
        assert jkv.rotary(z, starts=starts, out=z) is z
        assert jkv.packed_attention(z, x[1], x[2], starts, out=torch.empty_like(z)).shape == z.shape


def _sum_seen(weights, seen, rows):
    """``sum_i weights[i,j] rows[i]`` over the i that j counts for, infinities and NaN
    among them as they come."""

    weights = torch.where(seen, weights, 0.0)
    odd = ~torch.isfinite(rows).all(-1)
    total = weights[~odd].T @ rows[~odd]
    for i in odd.nonzero()[:, 0].tolist():
        total = total + torch.where(seen[i][:, None], weights[i][:, None] * rows[i], 0.0)
    return total


def defined_gradients(q, k, v, d, *, cap, window, prefix, h):
    """The gradients of one kv head's sequence from their formulas in 64 bits, also
    where rows are not finite, and by how much roundings of h may change what is."""

    q, k, v, d = (x.double() for x in (q, k, v, d))
    rows, heads, dim = q.shape
    seen = ref.visible(rows, rows, window, 0, prefix)
    grads = [torch.zeros_like(x) for x in (q, k, v)]
    bounds = [torch.zeros_like(x) for x in (q, k, v)]
    tame = lambda x: torch.nan_to_num(x.abs(), 0.0, 0.0, 0.0)
    for g in range(heads):
        x, steep = ref.scores(q[:, g], k, scale=dim**-0.5, cap=cap, slope=None, first=0)
        x = torch.where(seen, x, -torch.inf)
        e = torch.exp(x - x.amax(-1, keepdim=True))
        p = e / e.sum(-1, keepdim=True)
        out = _sum_seen(p.T, seen.T, v)
        dp, delta = d[:, g] @ v.T, (d[:, g] * out).sum(-1, keepdim=True)
        slant = steep * dim**-0.5
        ds = p * (dp - delta) * slant
        grads[0][:, g] = _sum_seen(ds.T, seen.T, k)
        grads[1] += _sum_seen(ds, seen, q[:, g])
        grads[2] += _sum_seen(p, seen, d[:, g])
        # p and ds rounded to h each, delta's own rounding, scores off as elsewhere here
        size = float((tame(q[:, g]) @ tame(k).T).max()) * dim**-0.5
        off = 2 * (size * (dim + 2) * 2.0**-23 + 8 * (cap or 0.0) * 2.0**-23 + 2.0**-20) + (dim + rows) * 2.0**-23
        reach = tame(d[:, g]) @ tame(v).T + (tame(d[:, g]) * tame(out)).sum(-1, keepdim=True)
        much = tame(p) * tame(slant) * (h * (2 * tame(dp - delta) + tame(delta)) + (h * h + off) * reach)
        bounds[0][:, g] = _sum_seen(much.T, seen.T, tame(k))
        bounds[1] += _sum_seen(much, seen, tame(q[:, g]))
        bounds[2] += _sum_seen(tame(p) * (h + off) * 1.01, seen, tame(d[:, g]))
    for g, b in zip(grads, bounds):
        b += h * tame(g) + 1e-7 * b.max() + 2.0**-24
    return grads, bounds


@pytest.mark.parametrize("cap", [30.0, None])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,qh,kvh,dim,window,prefix", [
    ([330], 4, 2, 64, None, 0),              # 32 keys a workgroup
    ([100, 330], 4, 2, 128, 150, 40),
    ([600], 16, 2, 128, None, 0),            # heads in splits
    ([330, 250] * 6, 12, 12, 128, None, 0),  # 128 keys a workgroup, all heads
])
def test_what_odd_elements_reach(device, cap, dtype, sizes, qh, kvh, dim, window, prefix):
    """One infinite or NaN element: every gradient is finite where its formula is, in
    tiles with and without masked places, has its value there, and is the same as
    without the element where that takes no part."""

    per = qh // kvh
    at = sum(sizes[: len(sizes) - 1 - len(sizes) // 2]) + 170
    prefixes = torch.full((len(sizes),), prefix, dtype=torch.int32, device=device)
    args = dict(window=window, softcap=cap, prefixes=prefixes)
    base = Texts(41, sizes, qh, kvh, dim, dtype, gain=1.5)
    span = next(slice(a, b) for a, b in base.spans if a <= at < b)
    _, clean = run_grads(base, device, **args)
    for name in ("q", "k", "v", "d"):
        for bad in (float("inf"), float("-inf"), float("nan")):
            odd = Texts(41, sizes, qh, kvh, dim, dtype, gain=1.5)
            getattr(odd, name)[at, 1 if name in "kv" else per, 3] = bad
            _, grads = run_grads(odd, device, **args)
            heads = slice(per, 2 * per)
            want, bounds = defined_gradients(odd.q[span, heads], odd.k[span, 1], odd.v[span, 1], odd.d[span, heads], cap=cap,
                                             window=window, prefix=prefix, h=half_step(dtype))
            # beside the sequence and the group nothing changes
            for got, same, of in zip(grads, clean, (heads, 1, 1)):
                got, same = got.clone(), same.clone()
                got[span, of] = 0
                same[span, of] = 0
                assert torch.equal(got, same), (name, bad)
            if name == "v":  # p does not depend on values
                assert torch.equal(grads[2], clean[2]), bad
            for part, got, w, bound in zip(("dq", "dk", "dv"), (grads[0][span, heads], grads[1][span, 1], grads[2][span, 1]), want, bounds):
                got = got.cpu().double()
                finite = torch.isfinite(w)
                assert torch.equal(torch.isfinite(got), finite), (name, bad, part)
                assert ((got - w).abs() <= bound)[finite].all(), (name, bad, part)
                if (name, part) == ("d", "dv"):
                    assert torch.equal(torch.isnan(got), torch.isnan(w)) and torch.equal(got[~finite & ~torch.isnan(w)], w[~finite & ~torch.isnan(w)])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,qh,kvh,dim", [
    ([150, 90], 4, 2, 64),
    ([200, 290], 4, 2, 128),
    ([600, 40], 16, 2, 128),            # heads in splits
    ([330, 250] * 6, 12, 12, 128),      # 128 keys a workgroup
])
@pytest.mark.parametrize("size", [2.0**-12, 1000.0])
def test_gradients_beside_small_and_large_ones(device, dtype, sizes, qh, kvh, dim, size):
    """A neighbour's sizes, a head's, or those of rows that are not seen change no bit."""

    texts = Texts(51, sizes, qh, kvh, dim, dtype)
    args = dict(window=100, softcap=25.0)
    _, want = run_grads(texts, device, **args)

    def moved(change):
        other = Texts(51, sizes, qh, kvh, dim, dtype)
        change(other)
        return run_grads(other, device, **args)[1]

    def neighbour(t):
        for a, b in t.spans[1::2]:
            t.d[a:b] *= size
            t.v[a:b] *= min(size, 100.0)

    got = moved(neighbour)
    for x, y in zip(got, want):
        for a, b in texts.spans[::2]:
            assert torch.equal(x[a:b], y[a:b])
    # heads of the other kv head
    got = moved(lambda t: (t.d[:, qh // kvh :].mul_(size), t.v[:, 1:].mul_(min(size, 100.0))))
    assert torch.equal(got[0][:, : qh // kvh], want[0][:, : qh // kvh])
    assert torch.equal(got[1][:, 0], want[1][:, 0]) and torch.equal(got[2][:, 0], want[2][:, 0])
    # do of the last rows of the first sequence: of the others' dq, and of keys out of their window
    a, b = texts.spans[0]
    cut = b - 25

    def late(t):
        t.d[cut:b] *= size

    got = moved(late)
    assert torch.equal(got[0][a:cut], want[0][a:cut])
    for x, y in zip(got[1:], want[1:]):
        assert torch.equal(x[a : cut - 99], y[a : cut - 99])

    def late_values(t):
        t.v[cut:b] *= min(size, 100.0)

    got = moved(late_values)
    assert torch.equal(got[0][a:cut], want[0][a:cut]) and torch.equal(got[1][a : cut - 99], want[1][a : cut - 99])


@pytest.mark.parametrize("cap", [None, 25.0])
@pytest.mark.parametrize("qh,kvh,dim,rows", [(4, 2, 64, 400), (16, 2, 128, 600)])
def test_gradients_keep_their_digits_beside_outliers(device, cap, qh, kvh, dim, rows):
    """fp16: one row of do at the end of its type's range, one of values far above the
    others; what neither reaches is as exact as without them (the largest of a row's or
    key's own ds is the measure: 2^-32 of it, and half a step of a result below 2^-14)."""

    texts = Texts(52, [rows], qh, kvh, dim, torch.float16)
    texts.d *= 2.0**-4
    texts.d[200] = 60000.0 * torch.sign(texts.d[200].float()).half()
    texts.v[50] *= 2000.0
    out, grads = run_grads(texts, device, window=60, softcap=cap)
    r = texts.expect(grads=True, cap=cap, window=60)[0]
    far = torch.ones(rows, dtype=torch.bool)
    far[50:110] = False   # rows that see the values
    far[200] = False
    keys = torch.ones(rows, dtype=torch.bool)
    keys[0:110] = False   # keys that those rows see
    keys[141:201] = False
    h = half_step(torch.float16)
    for name, got, kept in zip(("dq", "dk", "dv"), grads, (far, keys, keys)):
        off = float(score_slack(r, dim, cap, None, rows)[far].max()) * 2 + (dim + rows) * 2.0**-23 + (2.0**-21 if cap else 0.0)
        size = r[name + "_size"][kept]
        bound = h * r[name][kept].abs() + (h + 2.0**-22) * r[name + "_slack"][kept] + (off + 1e-7) * size + 2.0**-25 + (
            (2.0**-32 * 60 * size.amax() if name != "dv" else 2.0**-34 * size.amax()))
        assert ((got.cpu().double()[kept] - r[name][kept]).abs() <= bound).all(), name
        # and in the mean a rounding or two of 2^-11
        assert float((got.cpu().double()[kept] - r[name][kept]).norm() / r[name][kept].norm()) < 2.0**-11


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("sizes,qh,kvh,dim,form,gain", [
    ([129], 32, 8, 128, 1, 4.0), ([700], 8, 2, 128, 0, 8.0), ([700, 200], 7, 1, 64, 4, 6.0), ([60] * 10, 4, 4, 64, 2, 4.0)])
def test_gradients_in_the_mean(device, dtype, sizes, qh, kvh, dim, form, gain):
    """The error's norm against that of the exact results' own rounding.  For sharp heads
    too, dq and dk add no rounding of that size (ds has two parts; delta takes the
    forward's weights, whose roundings meet in one sum a row), out and dv one, of p:
    the root of 2 where, as here, terms have signs at random."""

    texts = Texts(61, sizes, qh, kvh, dim, dtype, gain=1.0)
    texts.q = (texts.q.float() * gain).to(dtype)
    texts.d = (texts.d.float() * 0.05).to(dtype)
    want, call = form_of(texts, FORMS[form], qh, device)
    out, grads = run_grads(texts, device, **call)
    results = texts.expect(grads=True, **want)
    for name, got, most in zip(("out", "dq", "dk", "dv"), (out.detach(), *grads), (1.5, 1.45, 1.3, 1.5)):
        exact = torch.cat([r[name] for r in results])
        own = (exact.to(dtype).double() - exact).norm()
        assert (got.cpu().double() - exact).norm() <= most * own, (name, float((got.cpu().double() - exact).norm() / own))

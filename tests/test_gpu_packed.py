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

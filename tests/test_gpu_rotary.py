"""Rotary rules on the MI355X against 64-bit definitions."""

from __future__ import annotations

import pytest
import torch

import jointkv_amd as jkv
from oracle import shaped_oracle as ref

pytestmark = pytest.mark.gpu

RULES = {
    "plain": dict(),
    "linear": dict(scaling="linear", factor=4.0),
    "base": dict(scaling="base", factor=8.0),
    "parts": dict(scaling="parts", factor=8.0, original_length=8192, low=1.0, high=4.0, magnitude=1.25),
}


def expect(x, positions, rule, sign=1):
    dims = rule.dims or x.shape[-1]
    rates = ref.rates(dims, rule.theta, rule.scaling, rule.factor, rule.original_length or 0, rule.low, rule.high)
    return ref.turn(x.cpu(), positions, rates, layout=rule.layout, magnitude=rule.magnitude, sign=sign)


def check(got, want, x, rule):
    """The result's own rounding h, and the 32-bit cosine, sine, two products
    and sum: sine and cosine are within 2^-23 of theirs (2^-24 of rounding, and
    the quarter's rest rounded to 2^-25 of pi/2), times the magnitude rounded once
    and the products' and sum's roundings: under 2^-21 (|x| + |y|) m.  A 64-bit
    product of a position below 2^31 and a rate is off by 2^31 2^-53 turns at most."""

    h = torch.finfo(x.dtype).eps / 2
    pair = 2 * x.detach().double().abs().amax().item() * abs(rule.magnitude)
    off = (got.detach().cpu().double() - want).abs()
    assert (off <= h * want.abs() + 2.0**-21 * pair + (torch.finfo(x.dtype).tiny if x.dtype != torch.float32 else 0)).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("dim,dims", [(128, None), (128, 64), (64, 32), (128, 20), (80, 40), (96, 22), (2, 2), (256, 256), (6, 4)])
def test_layouts_and_parts_of_heads(device, dtype, layout, dim, dims):
    gen = torch.Generator().manual_seed(dim + (dims or 0))
    q = torch.randn(37, 5, dim, generator=gen).to(dtype).to(device)
    k = torch.randn(37, 2, dim, generator=gen).to(dtype).to(device)
    starts = torch.tensor([0, 1, 1, 30, 37], dtype=torch.int32, device=device)
    first = [5, 900, 70001, 0]
    rule = jkv.RotaryRule(layout=layout, dims=dims)
    got = jkv.rotary(q, k, rule, starts=starts, positions=torch.tensor(first, dtype=torch.int32, device=device))
    at = [5] + [70001 + t for t in range(29)] + list(range(7))
    for g, x in zip(got, (q, k)):
        assert g.shape == x.shape and g.dtype == dtype and g.is_contiguous()
        check(g, expect(x, at, rule), x, rule)


@pytest.mark.parametrize("name", RULES)
def test_scalings_at_far_positions(device, name):
    rule = jkv.RotaryRule(theta=500000.0 if name == "parts" else 10000.0, **RULES[name])
    at = [0, 1, 8191, 131071, 1_000_003, 2**31 - 1, -3]
    x = torch.randn(len(at), 3, 128, generator=torch.Generator().manual_seed(3)).to(device)
    got = jkv.rotary(x, rule=rule, positions=torch.tensor(at, dtype=torch.int32, device=device))
    check(got, expect(x, at, rule), x, rule)


def test_agrees_with_the_turn_of_the_paged_append(device):
    """Plain whole heads: the paged cache's own rotation, within both bounds."""

    gen = torch.Generator().manual_seed(9)
    k = torch.randn(50, 2, 128, generator=gen).half().to(device)
    pool = torch.zeros(4, 2, 16, 128, dtype=torch.float16, device=device)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    tables = ints(0, 1, 2, 3).view(1, 4)
    jkv.paged_append(k, k, pool, torch.zeros_like(pool), tables, ints(50), starts=ints(0, 50), positions=ints(1000))
    stored = pool.permute(0, 2, 1, 3).reshape(64, 2, 128)[:50]
    turned = jkv.rotary(k, starts=ints(0, 50), positions=ints(1000))
    # one rounding each, and hardware sine and cosine of 2^-18 there
    assert ((stored.float() - turned.float()).abs() <= 2.0**-10 * turned.float().abs() + 2.0**-15 * k.float().abs().max()).all()


def test_rows_of_no_sequence_and_defaults(device):
    x = torch.randn(12, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(device)
    ints = lambda *v: torch.tensor(v, dtype=torch.int32, device=device)
    got = jkv.rotary(x, starts=ints(3, 6, 10))
    rule = jkv.RotaryRule()
    assert torch.equal(got[:3], x[:3]) and torch.equal(got[10:], x[10:])
    check(got[3:10], expect(x[3:10], [0, 1, 2, 0, 1, 2, 3], rule), x, rule)
    check(jkv.rotary(x), expect(x, range(12), rule), x, rule)
    assert jkv.rotary(x[:0]).shape == (0, 2, 64)
    empty = jkv.rotary(x, starts=ints(0))
    assert torch.equal(empty, x)


def test_many_sequences(device):
    counts = torch.randint(0, 4, (300,), generator=torch.Generator().manual_seed(4)).tolist()
    starts = [0]
    for n in counts:
        starts.append(starts[-1] + n)
    first = torch.randint(0, 10000, (300,), generator=torch.Generator().manual_seed(5)).tolist()
    x = torch.randn(starts[-1], 1, 64, generator=torch.Generator().manual_seed(6)).half().to(device)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=device)
    got = jkv.rotary(x, starts=ints(starts), positions=ints(first))
    at = [f + t for f, n in zip(first, counts) for t in range(n)]
    check(got, expect(x, at, jkv.RotaryRule()), x, jkv.RotaryRule())


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_strides_and_given_outputs(device, layout):
    gen = torch.Generator().manual_seed(2)
    rule = jkv.RotaryRule(layout=layout, dims=64)
    wide = torch.randn(4, 20, 131, generator=gen).half().to(device)
    whole = jkv.rotary(wide[..., :128].transpose(0, 1).contiguous(), rule=rule)
    for view in (wide[..., :128].transpose(0, 1), wide[..., :128].contiguous().transpose(0, 1)):
        assert torch.equal(jkv.rotary(view, rule=rule), whole)
    odd = torch.empty(20 * 4 * 128 + 1, dtype=torch.float16, device=device)[1:].view(20, 4, 128)
    odd.copy_(wide[..., :128].transpose(0, 1))
    assert torch.equal(jkv.rotary(odd, rule=rule), whole)
    assert torch.equal(jkv.rotary(odd, rule=rule, out=odd), whole)  # in place
    assert torch.equal(odd, whole)
    mixed = wide[..., :128].permute(1, 0, 2).transpose(1, 2).contiguous().transpose(1, 2)  # rows not contiguous
    assert torch.equal(jkv.rotary(mixed, rule=rule), whole)
    key = torch.randn(20, 1, 128, generator=gen).half().to(device)
    out, key_out = torch.zeros_like(whole), torch.zeros_like(key)
    got = jkv.rotary(mixed, key, rule, out=out, key_out=key_out)
    assert got[0] is out and got[1] is key_out and torch.equal(out, whole)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("layout,dims", [("half", None), ("interleaved", 32)])
def test_gradients(device, dtype, layout, dims):
    gen = torch.Generator().manual_seed(8)
    rule = jkv.RotaryRule(layout=layout, dims=dims, magnitude=1.1)
    q = torch.randn(33, 4, 64, generator=gen).to(dtype).to(device).requires_grad_()
    k = torch.randn(33, 1, 64, generator=gen).to(dtype).to(device).requires_grad_()
    shared = k.expand(33, 3, 64)  # one kv head seen as three
    starts = torch.tensor([2, 20, 31], dtype=torch.int32, device=device)
    out = jkv.rotary(q, shared, rule, starts=starts)
    gq, gk = torch.randn(33, 4, 64, generator=gen).to(dtype), torch.randn(33, 3, 64, generator=gen).to(dtype)
    dq, dk = torch.autograd.grad(out, (q, k), (gq.to(device), gk.to(device)))
    at = list(range(18)) + list(range(11))

    def back(g):
        want = g.double()
        want[2:31] = expect(g[2:31], at, rule, -1)
        return want

    check(dq, back(gq), gq, rule)
    # three heads' gradients, each rounded, are summed in the tensors' type
    h = torch.finfo(dtype).eps / 2
    want = back(gk)
    assert ((dk.cpu().double() - want.sum(1, keepdim=True)).abs() <= 4 * h * want.abs().sum(1, keepdim=True) + 2.0**-18).all()
    # one of two outputs used, one input needing a gradient
    only = torch.autograd.grad(jkv.rotary(q, shared.detach(), rule, starts=starts)[0], q, gq.to(device))[0]
    assert torch.equal(only, dq)
    # a linear map's gradient against differences: <g, R(x + d) - R(x)> = <R^T g, d>, in 64 bits of 32-bit results
    if dtype == torch.float32:
        d = torch.randn(33, 4, 64, generator=gen).to(device)
        with torch.no_grad():
            change = (jkv.rotary(q + d, rule=rule, starts=starts).double() - jkv.rotary(q, rule=rule, starts=starts).double())
        left, right = (gq.to(device).double() * change).sum(), (dq.double() * d.double()).sum()
        assert abs(left - right) <= 33 * 4 * 64 * 2.0**-20 * 4


def test_two_streams_and_graph_replays(device):
    x = torch.randn(64, 4, 128, generator=torch.Generator().manual_seed(5)).half().to(device)
    at = torch.arange(64, dtype=torch.int32, device=device)
    want = jkv.rotary(x, positions=at)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = jkv.rotary(x, positions=at)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = jkv.rotary(x, positions=at)
    for n in range(3):
        at.copy_(torch.arange(64, dtype=torch.int32, device=device) + 1000 * n)
        graph.replay()
        assert torch.equal(held, jkv.rotary(x, positions=at))

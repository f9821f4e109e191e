"""Operators around attention that differs from one model to the next, as a
training or serving program calls them.

* ``rotary``: queries and keys turned at their positions in one call, either
  layout, part of a head, frequencies scaled for long contexts; with the
  gradients in training.
* ``packed``: attention inside documents packed one behind another, scores
  capped by a tanh or biased by distance, a sliding window, prefixes seen from
  both sides; forward (prompts) or with all gradients (training).
* ``paged``: the same scores over the paged cache, single tokens and chunks.
* ``copy``: pages copied in all layers, what a forked sequence needs before it
  writes to a page that it shares.

Head counts and dims are the framework's own (32 query and 8 kv heads of 128
dims, a 4,096-token window) beside other groupings.

``run`` computes the plain form in 32 bits (rotary angles in 64), or with
``own`` calls the framework.  ``exact`` restates every operator in 64 bits.
"""

from __future__ import annotations

import functools
import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

THETA = 10000.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
# trained on 8,192 positions, stretched eightfold
SCALINGS = {"none": {}, "linear": {"scaling": "linear", "factor": 8.0}, "base": {"scaling": "base", "factor": 8.0},
            "parts": {"scaling": "parts", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 4.0,
                      "magnitude": 1.2}}


def _rotary(seqs, tokens, *, dtype="fp16", qh=32, kvh=8, dim=128, layout="half", turned=0, scaling="none", far=0,
            train=False):
    return {"op": "rotary", "seqs": seqs, "tokens": tokens, "dtype": dtype, "qh": qh, "kvh": kvh, "dim": dim,
            "layout": layout, "turned": turned or dim, "scaling": scaling, "far": far, "train": train}


def _packed(docs, tokens, *, dtype="fp16", qh=32, kvh=8, dim=128, window=0, sinks=0, cap=0.0, bias=False,
            prefix=False, train=True):
    return {"op": "packed", "seqs": docs, "tokens": tokens, "dtype": dtype, "qh": qh, "kvh": kvh, "dim": dim,
            "window": window, "sinks": sinks, "cap": cap, "bias": bias, "prefix": prefix, "train": train}


def _paged(seqs, length, new, *, dtype="fp16", qh=32, kvh=8, dim=128, page=64, window=0, sinks=0, cap=0.0,
           bias=False, prefix=False, ragged=True):
    return {"op": "paged", "seqs": seqs, "length": length, "tokens": new, "dtype": dtype, "qh": qh, "kvh": kvh,
            "dim": dim, "page": page, "window": window, "sinks": sinks, "cap": cap, "bias": bias, "prefix": prefix,
            "ragged": ragged}


def _copy(pairs, layers, *, dtype="fp16", kvh=8, dim=128, page=64, partial=True):
    return {"op": "copy", "pairs": pairs, "layers": layers, "dtype": dtype, "kvh": kvh, "dim": dim, "page": page,
            "partial": partial}


def listed():
    return [
        # a decode step of 16 sequences, scaled frequencies, far positions: a launch's latency
        {"name": "rotary_step", **_rotary(16, 1, scaling="parts", far=60000)},
        # a training step's 12,000 or so packed tokens, half of each head turned, pairs side by side, with gradients
        {"name": "rotary_train", **_rotary(6, 2500, dtype="bf16", layout="interleaved", turned=64, train=True)},
        # one short text in training: latency
        {"name": "packed_one", **_packed(1, 129, cap=30.0)},
        # many short texts of unequal length packed for training; 64-dim heads, 7 to a kv head
        {"name": "packed_texts", **_packed(48, 511, qh=28, kvh=4, dim=64, cap=50.0)},
        # prompts whose first part sees itself from both sides, scores biased by distance
        {"name": "packed_prompts", **_packed(4, 2047, dtype="bf16", bias=True, prefix=True, train=False)},
        # long documents in training, the framework's window: the matrix products count
        {"name": "packed_long", **_packed(3, 8192, dtype="bf16", window=4096, cap=50.0)},
        # one user's chat, small pages: latency
        {"name": "decode_cap_one", **_paged(1, 1501, 1, page=16, cap=50.0, ragged=False)},
        # the framework's own decode configuration with capped scores
        {"name": "decode_cap_b16", **_paged(16, 4096, 1, window=4096, cap=50.0, ragged=False)},
        # long documents of unequal length, scores biased by distance
        {"name": "decode_bias_long", **_paged(4, 65536, 1, dtype="bf16", page=128, bias=True)},
        # prompt chunks over a long cache, capped scores, prefixes
        {"name": "chunk_cap", **_paged(2, 8192, 2048, dtype="bf16", cap=30.0, prefix=True)},
        # the last, half-written pages of eight forked sequences
        {"name": "copy_fork", **_copy(8, 32)},
        # whole pages: a prompt's cache made private
        {"name": "copy_prompt", **_copy(48, 32, dtype="bf16", partial=False)},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["rotary", "rotary", "packed", "packed", "packed", "packed", "paged", "paged", "paged", "copy"])
    kvh = rng.choice([1, 2, 4, 8, 8])
    per = rng.choice([1, 2, 3, 4, 4, 5, 7, 8]) if kvh < 8 else rng.choice([1, 4, 4, 5])
    dtype, dim = rng.choice(["fp16", "bf16"]), rng.choice([64, 128, 128])
    if op == "rotary":
        dim = rng.choice([64, 80, 96, 128, 128, 256])
        seqs = _log_int(rng, 1, 32)
        tokens = rng.choice([1, _log_int(rng, 1, max(1, 15000 // seqs))])
        return _rotary(seqs, tokens, dtype=rng.choice(["fp16", "bf16", "bf16", "fp32"]), qh=kvh * per, kvh=kvh, dim=dim,
                       layout=rng.choice(["half", "interleaved"]), turned=rng.choice([0, dim // 2, dim // 4, 20]),
                       scaling=rng.choice(list(SCALINGS)), far=rng.choice([0, _log_int(rng, 1, 200000)]),
                       train=rng.random() < 0.5)
    if op == "copy":
        page = rng.choice([16, 32, 64, 128, 256])
        return _copy(_log_int(rng, 1, 48 * 64 // page if page > 64 else 48), rng.choice([1, 2, 16, 24, 32]), dtype=dtype,
                     kvh=kvh, dim=dim, page=page, partial=rng.random() < 0.6)
    more = {"dtype": dtype, "qh": kvh * per, "kvh": kvh, "dim": dim,
            "cap": rng.choice([0.0, 20.0, 30.0, 50.0, 50.0]), "bias": rng.random() < 0.3, "prefix": rng.random() < 0.3}
    if rng.random() < 0.4:
        more.update(window=_log_int(rng, 16, 6000), sinks=rng.choice([0, 0, 1, 4, 100]))
    if op == "packed":
        tokens = _log_int(rng, 1, 6000)
        docs = rng.randint(1, max(1, min(64, 16000 // tokens)))
        return _packed(docs, tokens, train=rng.random() < 0.7, **more)
    more["page"] = rng.choice([16, 32, 64, 64, 128, 256])
    more["ragged"] = rng.random() < 0.7
    if rng.random() < 0.5:  # single tokens
        length = _log_int(rng, 1, 60000)
        return _paged(rng.randint(1, max(1, min(64, 65536 // length))), length, 1, **more)
    length = _log_int(rng, 2, 12000)
    new = min(length, _log_int(rng, 2, 2048))
    return _paged(rng.randint(1, max(1, min(16, 80000 // length, (1 << 25) // (length * new)))), length, new, **more)


# what a case's sequences are: known to the program on the host


def _sizes(case):
    """Per sequence: entries and how many of them are new (packed: all); the
    first is the longest."""

    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    paged = case["op"] == "paged"
    entries, new = [case["length"] if paged else case["tokens"]], [case["tokens"]]
    for _ in range(case["seqs"] - 1):
        if not paged:
            entries.append(rng.randint(max(1, case["tokens"] // 4), case["tokens"]))
            new.append(entries[-1])
        elif case["ragged"]:
            entries.append(rng.randint(max(1, case["length"] // 8), case["length"]))
            most = min(entries[-1], case["tokens"])
            new.append(rng.choice([1, rng.randint(1, most)]) if most > 1 else most)
        else:
            entries.append(case["length"])
            new.append(case["tokens"])
    return entries, new


def _prefixes(case):
    """Per sequence, how many first entries all of its tokens see."""

    if not case["prefix"]:
        return [0] * case["seqs"]
    rng = random.Random(case["tokens"] * 1009 + case["seqs"])
    return [rng.randint(0, x) for x in _sizes(case)[0]]


def _pairs_and_entries(case):
    """Visible (token, entry) pairs and distinct visible entries, over all sequences."""

    pairs = entries = 0
    window = case["window"] or 1 << 60
    for length, new, prefix in zip(*_sizes(case), _prefixes(case)):
        i = np.arange(length - new, length, dtype=np.int64)
        low, high = np.maximum(i - window + 1, 0), np.maximum(i, prefix - 1)
        pairs += int((high - low + 1 + np.minimum(case["sinks"], low)).sum())
        entries += int(high.max() - low.min() + 1 + min(case["sinks"], low.min()))
    return pairs, entries


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "copy":
        rows = sum(_copied(case)) * case["layers"] * case["kvh"]
        return {"bytes": 4 * rows * case["dim"] * size, "flops": 0}
    tokens = sum(_sizes(case)[1])
    if case["op"] == "rotary":
        passes = 2 if case["train"] else 1
        heads = tokens * (case["qh"] + case["kvh"])
        return {"bytes": passes * 2 * heads * case["dim"] * size, "flops": passes * 3 * heads * case["turned"]}
    pairs, entries = _pairs_and_entries(case)
    query, kv = tokens * case["qh"] * case["dim"] * size, entries * case["kvh"] * case["dim"] * size
    moved, flops = 2 * query + 2 * kv, 4 * pairs * case["qh"] * case["dim"]
    if case.get("train"):  # the output's gradient in, three gradients out
        return {"bytes": moved + 2 * query + 2 * kv, "flops": 14 * pairs * case["qh"] * case["dim"]}
    return {"bytes": moved, "flops": flops}


def _copied(case):
    """Entries of each copied page."""

    rng = random.Random(case["pairs"] * 31 + case["page"])
    return [rng.randint(1, case["page"]) if case["partial"] else case["page"] for _ in range(case["pairs"])]


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    kvh, dim = case["kvh"], case["dim"]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=device, dtype=torch.float32)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device=device)

    state = {"case": case}
    if case["op"] == "copy":
        pairs = case["pairs"]
        order = torch.randperm(2 * pairs + 3, generator=gen, device=device).to(torch.int32)
        state.update(sources=order[:pairs].clone(), targets=order[pairs : 2 * pairs].clone(),
                     entries=ints(_copied(case)) if case["partial"] else None)
        for name in ("key_pages", "value_pages"):
            state[name] = torch.empty(case["layers"], 2 * pairs + 3, kvh, case["page"], dim, dtype=dtype, device=device)
            for layer in state[name]:
                layer.copy_(randn(*layer.shape))
        return state
    qh, (lengths, new) = case["qh"], _sizes(case)
    tokens = sum(new)
    state["spans"] = [0] + np.cumsum(new).tolist()
    state["starts"] = ints(state["spans"])
    # a few channels of each head are large, as queries and keys show
    gain = torch.ones(dim, device=device)
    gain[: dim // 32] = 3.0
    # sharp heads, whose scores a cap acts on
    sharp = 2.0 if case.get("cap") else 1.0
    if case["op"] == "rotary":
        state["positions_host"] = [case["far"] + 97 * b for b in range(case["seqs"])]
        state["positions"] = ints(state["positions_host"])
    else:
        state["prefixes"] = ints(_prefixes(case)) if case["prefix"] else None
        # the usual slopes: a geometric series over the heads, from a half to 2^-8
        state["slopes"] = (2.0 ** (-8.0 * torch.arange(1, qh + 1, device=device, dtype=torch.float64) / qh)).float() if (
            case["bias"]) else None
    state["query"] = (randn(tokens, qh, dim) * gain * sharp).to(dtype)
    if case["op"] == "paged":
        page = case["page"]
        pages_of = [-(-x // page) for x in lengths]
        total = sum(pages_of) + 3
        # pages lie in the pool in no order
        order = torch.randperm(total, generator=gen, device=device).to(torch.int32)
        tables = torch.full((case["seqs"], max(pages_of)), -1, dtype=torch.int32, device=device)
        at = 0
        for b, n in enumerate(pages_of):
            tables[b, :n] = order[at : at + n]
            at += n
        state.update(tables=tables, lengths=ints(lengths), lengths_host=lengths, new_host=new,
                     single=all(n == 1 for n in new))
        for name in ("key_pages", "value_pages"):
            state[name] = torch.empty(total, kvh, page, dim, dtype=dtype, device=device)
            for i in range(0, total, 4096):
                part = state[name][i : i + 4096]
                part.copy_(randn(*part.shape) * gain if name == "key_pages" else randn(*part.shape))
        return state
    state["key"] = (randn(tokens, kvh, dim) * gain).to(dtype)
    names = ["query", "key"]
    if case["op"] == "packed":
        state["value"] = randn(tokens, kvh, dim).to(dtype)
        names.append("value")
        state["d_out"] = (randn(tokens, qh, dim) * 0.01).to(dtype) if case["train"] else None
    elif case["train"]:
        state["d_out"] = [(randn(tokens, h, dim) * 0.01).to(dtype) for h in (qh, kvh)]
    if case["train"]:
        for name in names:
            state[name].requires_grad_()
    return state


# the plain forms


def _rates(case):
    """64-bit radians a position of each turned pair, and the magnitude."""

    turned, rule = case["turned"], SCALINGS[case["scaling"]]
    theta, factor, kind = THETA, rule.get("factor", 1.0), rule.get("scaling")
    if kind == "base":
        theta = theta * factor ** (turned / (turned - 2))
    rate = theta ** (-torch.arange(0, turned, 2, dtype=torch.float64) / turned)
    if kind == "linear":
        rate = rate / factor
    if kind == "parts":  # fast pairs stay, slow ones are stretched, a ramp between
        turns = rule["original_length"] * rate / (2 * math.pi)
        keep = ((turns - rule["low"]) / (rule["high"] - rule["low"])).clamp(0, 1)
        rate = rate * (keep + (1 - keep) / factor)
    return rate, rule.get("magnitude", 1.0)


def _row_positions(state):
    starts, positions = state["starts"].long(), state["positions"].long()
    n = torch.arange(state["spans"][-1], device=starts.device)
    seq = torch.searchsorted(starts[1:], n, right=True)
    return positions[seq] + n - starts[seq]


def _turn(x, position, case, back):
    """fp32 rotary of ``x[tokens, heads, dim]``: angles in 64 bits."""

    rate, magnitude = _rates(case)
    angle = position.double()[:, None, None] * rate.to(position.device)
    cos, sin = (torch.cos(angle) * magnitude).float(), (torch.sin(angle) * (-magnitude if back else magnitude)).float()
    out = x.float().clone()
    turned = case["turned"]
    if case["layout"] == "half":
        first, second = slice(0, turned // 2), slice(turned // 2, turned)
    else:
        first, second = slice(0, turned, 2), slice(1, turned, 2)
    a, b = out[..., first].clone(), out[..., second].clone()
    out[..., first] = a * cos - b * sin
    out[..., second] = b * cos + a * sin
    return out.to(x.dtype)


def _plain_rotary(state):
    case, position = state["case"], _row_positions(state)
    outs = [_turn(state[name].detach(), position, case, False) for name in ("query", "key")]
    if case["train"]:
        outs += [_turn(g, position, case, True) for g in state["d_out"]]
    return outs


def _seen(i, j, case, prefix):
    seen = (j <= i) | (j < prefix)
    if case["window"]:
        seen &= (j > i - case["window"]) | (j < case["sinks"])
    return seen


def _plain_sequence(case, query, key, value, first, prefix, slopes, d_out):
    """One sequence and kv head in 32 bits: ``query[T,per,D]`` from entry
    ``first`` on, ``key``/``value`` ``[L,D]``; the output, and with ``d_out``
    the three gradients."""

    tokens, per, dim = query.shape
    length, scale, cap = key.shape[0], dim ** -0.5, case["cap"]
    query, key, value = query.float().transpose(0, 1), key.float(), value.float()
    scores = torch.matmul(query, key.t().contiguous()) * scale
    slant = None
    if cap:
        bent = torch.tanh(scores / cap)
        slant = 1 - bent * bent if d_out is not None else None
        scores = bent * cap
    i = torch.arange(first, first + tokens, device=key.device)[:, None]
    j = torch.arange(length, device=key.device)[None]
    if slopes is not None:
        scores = scores - slopes[:, None, None] * (i - j).abs()
    scores = scores.masked_fill(~_seen(i, j, case, prefix), float("-inf"))
    p = torch.exp(scores - scores.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    out = torch.matmul(p, value)
    if d_out is None:
        return out.transpose(0, 1), None
    d_out = d_out.float().transpose(0, 1)
    d_value = torch.matmul(p.reshape(per * tokens, length).t().contiguous(), d_out.reshape(per * tokens, dim))
    ds = torch.matmul(d_out, value.t().contiguous())
    ds = p * (ds - (d_out * out).sum(-1, keepdim=True)) * scale
    if cap:
        ds = ds * slant
    d_query = torch.matmul(ds, key)
    d_key = torch.matmul(ds.reshape(per * tokens, length).t().contiguous(), query.reshape(per * tokens, dim))
    return out.transpose(0, 1), (d_query.transpose(0, 1), d_key, d_value)


def _entries(state, b):
    """Pool rows (page, slot) of sequence b's entries."""

    j = torch.arange(state["lengths_host"][b], device=state["tables"].device)
    page = state["case"]["page"]
    return state["tables"][b].long()[j // page], j % page


def _plain_attention(state):
    case, spans = state["case"], state["spans"]
    per, prefixes = case["qh"] // case["kvh"], _prefixes(case)
    paged, train = case["op"] == "paged", case.get("train", False)
    out = torch.empty_like(state["query"])
    grads = [torch.empty_like(state[x]) for x in ("query", "key", "value")] if train else []
    for b in range(case["seqs"]):
        rows = slice(spans[b], spans[b + 1])
        if paged:
            pages, slots = _entries(state, b)
        for h in range(case["kvh"]):
            heads = slice(h * per, h * per + per)
            if paged:
                key, value = state["key_pages"][pages, h, slots], state["value_pages"][pages, h, slots]
                first = state["lengths_host"][b] - state["new_host"][b]
            else:
                key, value, first = state["key"].detach()[rows, h], state["value"].detach()[rows, h], 0
            o, d = _plain_sequence(case, state["query"].detach()[rows, heads], key, value, first, prefixes[b],
                                   state["slopes"][heads] if case["bias"] else None,
                                   state["d_out"][rows, heads] if train else None)
            out[rows, heads] = o.to(out.dtype)
            if train:
                grads[0][rows, heads] = d[0].to(out.dtype)
                grads[1][rows, h] = d[1].to(out.dtype)
                grads[2][rows, h] = d[2].to(out.dtype)
    return [out.detach(), *(g.detach() for g in grads)]


def _plain_copy(state):
    case = state["case"]
    src, dst = state["sources"].long(), state["targets"].long()
    slot = torch.arange(case["page"], device=src.device)
    for name in ("key_pages", "value_pages"):
        for layer in state[name]:
            taken, there = layer[src], layer[dst]
            if case["partial"]:
                taken = torch.where((slot < state["entries"][:, None])[:, None, :, None], taken, there)
            layer[dst] = taken
    return [state["key_pages"], state["value_pages"]]


@functools.lru_cache(maxsize=1)
def _framework():
    path = str(Path(__file__).resolve().parent.parent / "tac-vq-kv-cache_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import jointkv_amd

    return jointkv_amd


def _own(state):
    jkv, case = _framework(), state["case"]
    if case["op"] == "rotary":
        rule = jkv.RotaryRule(theta=THETA, layout=case["layout"], dims=case["turned"], **SCALINGS[case["scaling"]])
        outs = jkv.rotary(state["query"], state["key"], rule, starts=state["starts"], positions=state["positions"])
        if not case["train"]:
            return list(outs)
        return [*outs, *torch.autograd.grad(outs, (state["query"], state["key"]), state["d_out"])]
    if case["op"] == "copy":
        jkv.copy_pages(state["key_pages"], state["value_pages"], state["sources"], state["targets"],
                       entries=state["entries"])
        return [state["key_pages"], state["value_pages"]]
    form = {"window": case["window"] or None, "sinks": case["sinks"], "softcap": case["cap"] or None,
            "slopes": state["slopes"], "prefixes": state["prefixes"]}
    if case["op"] == "packed":
        out = jkv.packed_attention(state["query"], state["key"], state["value"], state["starts"], **form)
        if not case["train"]:
            return [out]
        return [out, *torch.autograd.grad(out, (state["query"], state["key"], state["value"]), state["d_out"])]
    return [jkv.paged_attention(state["query"], state["key_pages"], state["value_pages"], state["tables"],
                                state["lengths"], starts=None if state["single"] else state["starts"], rope_theta=None,
                                max_new=max(state["new_host"]), max_length=max(state["lengths_host"]), **form)]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "rotary":
        return _plain_rotary(state)
    return _plain_copy(state) if op == "copy" else _plain_attention(state)


# the definitions in 64 bits


def _turned(x, positions, case, sign):
    """Rotary as a product of complex numbers."""

    rule, turned = SCALINGS[case["scaling"]], case["turned"]
    rates = []
    for i in range(turned // 2):
        base = THETA
        if rule.get("scaling") == "base":
            base = THETA * math.exp(math.log(rule["factor"]) * turned / (turned - 2))
        rate = math.exp(-2 * i / turned * math.log(base))
        if rule.get("scaling") == "linear":
            rate /= rule["factor"]
        if rule.get("scaling") == "parts":
            turns = rule["original_length"] / (2 * math.pi / rate)
            if turns < rule["low"]:
                rate /= rule["factor"]
            elif turns <= rule["high"]:
                share = (turns - rule["low"]) / (rule["high"] - rule["low"])
                rate = share * rate + (1 - share) * rate / rule["factor"]
        rates.append(rate)
    angle = torch.as_tensor(positions, dtype=torch.float64, device=x.device)[:, None] * torch.tensor(
        rates, dtype=torch.float64, device=x.device)
    turn = torch.polar(torch.full_like(angle, rule.get("magnitude", 1.0)), sign * angle)[:, None]
    x = x.detach().double()
    part, rest = x[..., :turned], x[..., turned:]
    if case["layout"] == "half":
        z = torch.complex(part[..., : turned // 2].contiguous(), part[..., turned // 2 :].contiguous()) * turn
        return torch.cat((z.real, z.imag, rest), -1)
    z = torch.view_as_complex(part.contiguous().unflatten(-1, (-1, 2))) * turn
    return torch.cat((torch.view_as_real(z).flatten(-2), rest), -1)


def _exact_head(query, key, value, first, case, prefix, slope):
    """Output of one query head: softmax in 64 bits."""

    i = torch.arange(query.shape[0], device=key.device)[:, None] + first
    j = torch.arange(key.shape[0], device=key.device)[None]
    logits = query @ key.t().contiguous() / math.sqrt(query.shape[1])
    if case["cap"]:
        logits = case["cap"] * torch.tanh(logits / case["cap"])
    if slope is not None:
        logits = logits - slope * torch.abs(j - i).double()
    hidden = (j > i) & (j >= prefix)
    if case["window"]:
        hidden |= (i - j >= case["window"]) & (j >= case["sinks"])
    return torch.softmax(logits.masked_fill(hidden, float("-inf")), -1) @ value


def exact(case, seed):
    if case["op"] in ("packed", "paged") and _pairs_and_entries(case)[0] * case["qh"] * (
            3 if case.get("train") else 1) > 1 << 33:
        return None
    s = prepare(case, seed)
    if case["op"] == "copy":
        outs = [s["key_pages"].clone(), s["value_pages"].clone()]
        for src, dst, count in zip(s["sources"].tolist(), s["targets"].tolist(), _copied(case)):
            for pool in outs:
                pool[:, dst, :, :count] = pool[:, src, :, :count]
        return outs
    spans = s["spans"]
    if case["op"] == "rotary":
        at = np.concatenate([p + np.arange(hi - lo) for p, lo, hi in zip(s["positions_host"], spans, spans[1:])])
        outs = [_turned(s[name], at, case, 1) for name in ("query", "key")]
        if case["train"]:
            outs += [_turned(g, at, case, -1) for g in s["d_out"]]
        return outs
    per, prefixes, train = case["qh"] // case["kvh"], _prefixes(case), case.get("train", False)
    results = [torch.zeros(s["query"].shape, dtype=torch.float64, device="cuda")]
    if train:
        results += [torch.zeros(s[x].shape, dtype=torch.float64, device="cuda") for x in ("query", "key", "value")]
    for b in range(case["seqs"]):
        rows = slice(spans[b], spans[b + 1])
        if case["op"] == "paged":
            where = _entries(s, b)
        for h in range(case["qh"]):
            kv = h // per
            if case["op"] == "paged":
                key, value = (s[x][where[0], kv, where[1]].double() for x in ("key_pages", "value_pages"))
                first = s["lengths_host"][b] - s["new_host"][b]
            else:
                key, value, first = s["key"].detach()[rows, kv].double(), s["value"].detach()[rows, kv].double(), 0
            query = s["query"].detach()[rows, h].double()
            leaves = [x.requires_grad_(train) for x in (query, key, value)]
            out = _exact_head(*leaves, first, case, prefixes[b], s["slopes"][h].double() if case["bias"] else None)
            results[0][rows, h] = out.detach()
            if train:
                dq, dk, dv = torch.autograd.grad(out, leaves, s["d_out"][rows, h].double())
                results[1][rows, h] = dq
                results[2][rows, kv] += dk
                results[3][rows, kv] += dv
    return results

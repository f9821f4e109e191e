"""The operators of a paged K/V cache, as a serving program calls them.

A pool of pages holds the (codec's) keys, rotated when they are written, and
values of many sequences; a block table lists each sequence's pages.  Four
operators work on it: the append of new tokens, the attention of new tokens
(one a sequence, or chunks of many) over the cached ones with a sliding window
and first entries that stay visible, the same attention with the weight that
every cached entry received, and eviction by that weight.

Head counts and dims are the framework's own (32 query and 8 kv heads of 128
dims, a 4,096-token window) beside other groupings; new tokens are packed
``[tokens, heads, dim]`` with ``starts`` between the sequences.

``run`` computes the plain form in 32 bits (rotary angles in 64), or with
``own`` calls the framework.  ``exact`` restates every operator in 64 bits,
sequence by sequence.
"""

from __future__ import annotations

import math
import random
import sys
from pathlib import Path

import numpy as np
import torch

own = False

THETA = 10000.0
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _case(op, batch, length, new, *, dtype="fp16", qh=32, kvh=8, dim=128, page=64, window=0, sinks=0,
          ragged=True, budget=0, recent=0):
    return {"op": op, "batch": batch, "length": length, "new": new, "dtype": dtype, "qh": qh, "kvh": kvh,
            "dim": dim, "page": page, "window": window, "sinks": sinks, "ragged": ragged, "budget": budget,
            "recent": recent}


def listed():
    return [
        # one decode step's keys and values of a batch into their pages: a launch's latency
        {"name": "append_step_b16", **_case("append", 16, 4096, 1)},
        # the prompts of four users, of unequal length, into their pages
        {"name": "append_prompts", **_case("append", 4, 8192, 6000, dtype="bf16")},
        # one user's chat, small pages: latency
        {"name": "decode_one", **_case("attend", 1, 1501, 1, page=16, ragged=False)},
        # the framework's own decode configuration: 16 sequences, a full window of 4,096
        {"name": "decode_b16", **_case("attend", 16, 4096, 1, window=4096, ragged=False)},
        # long documents of unequal length in bf16
        {"name": "decode_long", **_case("attend", 4, 65536, 1, dtype="bf16", page=128)},
        # endless chats: 8 sequences that see their first 4 entries and the last 4,096; 64-dim heads, 7 to a kv head
        {"name": "decode_sinks", **_case("attend", 24, 20000, 1, qh=28, kvh=4, dim=64, page=32, window=4096, sinks=4)},
        # a step that mixes prompt chunks with single tokens, sizes odd
        {"name": "chunk_mixed", **_case("attend", 12, 6007, 777, qh=28, kvh=4, dim=64, page=16, window=2048, sinks=64)},
        # chunks of two long prompts: the matrix products count
        {"name": "chunk_long", **_case("attend", 2, 16384, 2048, dtype="bf16", ragged=False)},
        # a decode step of a cache that evicts: its attention and what each entry received
        {"name": "weigh_b16", **_case("weigh", 16, 4096, 1, ragged=False)},
        # a prompt's chunk with the weights that its eviction goes by
        {"name": "weigh_chunk", **_case("weigh", 2, 4096, 1024, dtype="bf16")},
        # one sequence down to its budget
        {"name": "evict_one", **_case("evict", 1, 3001, 0, page=16, ragged=False, budget=1024, sinks=4, recent=256)},
        # a batch down to its budget
        {"name": "evict_b8", **_case("evict", 8, 16384, 0, dtype="bf16", budget=4096, sinks=4, recent=1024)},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "weigh", "weigh", "evict", "evict"])
    kvh = rng.choice([1, 2, 4, 8, 8])
    per = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 16]) if kvh < 8 else rng.choice([1, 4, 4, 5, 8])
    page, dim = rng.choice([16, 32, 64, 64, 128, 256]), rng.choice([64, 128, 128])
    more = {"dtype": rng.choice(["fp16", "bf16"]), "qh": kvh * per, "kvh": kvh, "dim": dim, "page": page,
            "ragged": rng.random() < 0.7}
    if op == "append":
        batch = _log_int(rng, 1, 64)
        new = rng.choice([1, _log_int(rng, 1, max(1, 24000 // batch))])
        return _case(op, batch, new + _log_int(rng, 1, 500), new, **more)
    if op == "evict":
        length = _log_int(rng, 20, 30000)
        batch = rng.randint(1, max(1, min(16, 60000 // length)))
        budget = rng.randint(max(2, length // 16), max(2, int(length * 0.75)))
        return _case(op, batch, length, 0, budget=budget, sinks=rng.choice([0, 1, 4]) if budget >= 8 else 0,
                     recent=rng.randint(0, budget // 2), **more)
    if rng.random() < 0.4:
        more.update(window=_log_int(rng, 16, 6000), sinks=rng.choice([0, 1, 4, 64, 100]))
    if rng.random() < 0.5:  # single tokens
        length = _log_int(rng, 1, 60000)
        batch = rng.randint(1, max(1, min(64, 65536 // length)))
        return _case(op, batch, length, 1, **more)
    length = _log_int(rng, 2, 16000)
    new = min(length, _log_int(rng, 2, 2048))
    batch = rng.randint(1, max(1, min(16, 100000 // length, (1 << 25) // (length * new))))
    return _case(op, batch, length, new, **more)


# what a case's sequences are: known to the program on the host


def _sizes(case):
    """(lengths, new tokens) of a case's sequences; the first is the longest."""

    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    lengths, new = [case["length"]], [case["new"]]
    for _ in range(case["batch"] - 1):
        if case["ragged"]:
            lengths.append(rng.randint(max(1, case["length"] // 8), case["length"]))
            # a step mixes chunks with single tokens
            new.append(min(lengths[-1], rng.choice([1, rng.randint(1, case["new"])]) if case["new"] > 1 else case["new"]))
        else:
            lengths.append(case["length"])
            new.append(case["new"])
    return lengths, new


def _spans(case):
    """Per sequence, the first and last entry index that a new token sits at."""

    return [(length - new, length) for length, new in zip(*_sizes(case))]


def _pairs_and_entries(case):
    """Visible (token, entry) pairs and distinct visible entries, over all sequences."""

    pairs = entries = 0
    window, sinks = case["window"] or 1 << 60, case["sinks"]
    for first, last in _spans(case):
        at = np.arange(first, last, dtype=np.int64)
        low = np.maximum(at - window + 1, 0)
        pairs += int((at - low + 1 + np.minimum(sinks, low)).sum())
        low0 = max(first - window + 1, 0)
        entries += last - low0 + min(sinks, low0) if last > first else 0
    return pairs, entries


def work(case):
    lengths, new = _sizes(case)
    row = case["dim"] * 2
    tokens = sum(new)
    if case["op"] == "append":  # keys and values in, keys and values out
        return {"bytes": 4 * tokens * case["kvh"] * row, "flops": 3 * tokens * case["kvh"] * case["dim"]}
    if case["op"] == "evict":
        kept = sum(min(x, case["budget"]) for x in lengths)
        return {"bytes": case["kvh"] * (sum(lengths) * 4 + kept * (4 * row + 4 + 4)), "flops": case["kvh"] * sum(lengths)}
    pairs, entries = _pairs_and_entries(case)
    moved = 2 * tokens * case["qh"] * row + 2 * entries * case["kvh"] * row
    if case["op"] == "weigh":
        moved += 4 * sum(lengths) * case["kvh"]
    return {"bytes": moved, "flops": 4 * pairs * case["qh"] * case["dim"]}


def prepare(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    batch, kvh, qh, dim, page = case["batch"], case["kvh"], case["qh"], case["dim"], case["page"]
    lengths, new = _sizes(case)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=device, dtype=torch.float32)

    pages_of = [-(-x // page) for x in lengths]
    wide = max(pages_of)
    out_of = [-(-min(x, case["budget"]) // page) for x in lengths]
    total = sum(pages_of) + (sum(out_of) if case["op"] == "evict" else 0) + 3
    # pages lie in the pool in no order
    order = torch.randperm(total, generator=gen, device=device).to(torch.int32)

    def table(counts, at):
        rows = torch.full((batch, max(max(counts), 1)), -1, dtype=torch.int32, device=device)
        for b, n in enumerate(counts):
            rows[b, :n] = order[at : at + n]
            at += n
        return rows, at

    tables, at = table(pages_of, 0)
    # a few channels of each head are large, as K/V caches show
    gain = torch.ones(kvh, 1, dim, device=device)
    gain[:, :, :4] = 3.0
    state = {
        "key_pages": torch.empty(total, kvh, page, dim, dtype=dtype, device=device),
        "value_pages": torch.empty(total, kvh, page, dim, dtype=dtype, device=device),
        "tables": tables,
        "lengths": torch.tensor(lengths, dtype=torch.int32, device=device),
        "case": case, "lengths_host": lengths, "new_host": new,
    }
    for name in ("key_pages", "value_pages"):
        pool = state[name]
        for i in range(0, total, 4096):
            part = pool[i : i + 4096]
            part.copy_(randn(*part.shape) * gain if name == "key_pages" else randn(*part.shape))
    if case["op"] == "evict":
        # most entries received little, some much, and some exactly the same
        weights = torch.exp(2.0 * randn(batch, kvh, max(lengths)))
        weights = torch.where(randn(batch, kvh, max(lengths)) > 1.5, weights.new_zeros(()), weights)
        state["weights"] = weights
        state["new_tables"], _ = table(out_of, at)
        return state
    tokens = sum(new)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    # sequences that had entries evicted before: their positions run ahead of their lengths
    ahead = [97 * b if case["op"] != "append" else 0 for b in range(batch)]
    state["starts"] = torch.tensor(starts, dtype=torch.int32, device=device)
    state["positions_host"] = [x - n + a for x, n, a in zip(lengths, new, ahead)]
    state["positions"] = torch.tensor(state["positions_host"], dtype=torch.int32, device=device)
    state["single"] = all(n == 1 for n in new)
    if case["op"] == "append":
        state["key"] = (randn(tokens, kvh, dim) * gain.squeeze(1)).to(dtype)
        state["value"] = randn(tokens, kvh, dim).to(dtype)
    else:
        state["query"] = randn(tokens, qh, dim).to(dtype)
        state["weights"] = torch.zeros(batch, kvh, max(lengths), dtype=torch.float32, device=device)
    return state


# the plain forms


def _rotated(x, positions):
    """fp32 rotary of ``x[tokens, heads, dim]`` (fp32): angles in 64 bits."""

    half = x.shape[-1] // 2
    rate = THETA ** (-torch.arange(half, dtype=torch.float64, device=x.device) / half)
    angle = positions.double()[:, None, None] * rate
    cos, sin = torch.cos(angle).float(), torch.sin(angle).float()
    a, b = x[..., :half], x[..., half:]
    return torch.cat((a * cos - b * sin, b * cos + a * sin), -1)


def _token_rows(state):
    """Per packed token: its sequence, its entry index and its position."""

    starts, lengths, positions = (state[k].long() for k in ("starts", "lengths", "positions"))
    tokens = sum(state["new_host"])
    n = torch.arange(tokens, device=starts.device)
    seq = torch.searchsorted(starts[1:], n, right=True)
    at = n - starts[seq]
    entry = lengths[seq] - (starts[seq + 1] - starts[seq]) + at
    return seq, at, entry, positions[seq] + at


def _plain_append(state):
    seq, _at, entry, position = _token_rows(state)
    page = state["case"]["page"]
    where, slot = state["tables"][seq, entry // page].long(), entry % page
    dtype = state["key_pages"].dtype
    state["key_pages"][where, :, slot] = _rotated(state["key"].float(), position).to(dtype)
    state["value_pages"][where, :, slot] = state["value"]
    return [state["key_pages"], state["value_pages"]]


def _plain_attention(state, weigh):
    case = state["case"]
    batch, kvh, qh, dim, page = case["batch"], case["kvh"], case["qh"], case["dim"], case["page"]
    seq, at, _entry, position = _token_rows(state)
    most, longest, per = max(state["new_host"]), max(state["lengths_host"]), qh // kvh
    device = seq.device
    # one row of the batch a sequence, padded
    query = torch.zeros(batch, most, kvh, per, dim, device=device)
    query[seq, at] = _rotated(state["query"].float(), position).view(-1, kvh, per, dim)
    query = query.permute(0, 2, 3, 1, 4).reshape(batch, kvh, per * most, dim)

    def rows(pool):  # a sequence's entries, in their order
        whole = pool[state["tables"].clamp_min(0).long()]
        return whole.permute(0, 2, 1, 3, 4).reshape(batch, kvh, -1, dim)[:, :, :longest].float()

    scores = torch.matmul(query, rows(state["key_pages"]).transpose(2, 3).contiguous())
    scores = scores.view(batch, kvh, per, most, longest) / math.sqrt(dim)
    lengths, new = state["lengths"].long(), (state["starts"][1:] - state["starts"][:-1]).long()
    own_entry = (lengths - new)[:, None] + torch.arange(most, device=device)
    entry = torch.arange(longest, device=device)
    seen = entry <= own_entry[..., None]
    if case["window"]:
        seen &= (entry > own_entry[..., None] - case["window"]) | (entry < case["sinks"])
    # padding rows behind a sequence's tokens take part in nothing
    seen &= (torch.arange(most, device=device) < new[:, None])[..., None]
    seen = seen[:, None, None]
    scores = scores.masked_fill(~seen, float("-inf"))
    top = scores.amax(-1, keepdim=True)
    scores = torch.exp(scores - torch.where(torch.isfinite(top), top, torch.zeros_like(top)))
    total = scores.sum(-1, keepdim=True)
    scores = scores / torch.where(total > 0, total, torch.ones_like(total))
    value = rows(state["value_pages"])
    value = torch.where((entry < lengths[:, None])[:, None, :, None], value, value.new_zeros(()))
    out = torch.matmul(scores.view(batch, kvh, per * most, longest), value)
    out = out.view(batch, kvh, per, most, dim).permute(0, 3, 1, 2, 4)[seq, at]
    out = out.reshape(-1, qh, dim).to(state["query"].dtype)
    if not weigh:
        return [out]
    weights = state["weights"]
    here = scores.sum((2, 3))
    weights.copy_(torch.where((entry < lengths[:, None])[:, None], here, weights))
    return [out, weights]


def _plain_evict(state):
    case = state["case"]
    budget, sinks, recent, page = case["budget"], case["sinks"], case["recent"], case["page"]
    weights, lengths = state["weights"], state["lengths"].long()
    batch, kvh, longest = weights.shape
    entry = torch.arange(longest, device=weights.device)
    always = (entry < sinks) | (entry >= (lengths - recent)[:, None])
    rank = weights.masked_fill(always[:, None], float("inf"))
    rank = rank.masked_fill((entry >= lengths[:, None])[:, None], -1.0)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    chosen = torch.arange(longest, device=weights.device) < torch.minimum(lengths, torch.full_like(lengths, budget))[:, None]
    none = longest
    kept = torch.where(chosen[:, None], order, torch.full_like(order, none)).sort(-1).values[..., :budget]
    if kept.shape[-1] < budget:
        kept = torch.nn.functional.pad(kept, (0, budget - kept.shape[-1]), value=none)
    valid = kept < none
    new_lengths = torch.minimum(lengths, torch.full_like(lengths, budget))
    b, h, j = torch.nonzero(valid, as_tuple=True)
    src, dst = state["tables"].long(), state["new_tables"].long()
    e = kept[b, h, j]
    for name in ("key_pages", "value_pages"):
        pool = state[name]
        pool[dst[b, j // page], h, j % page] = pool[src[b, e // page], h, e % page]
    moved = torch.zeros_like(weights)
    moved[b, h, j] = weights[b, h, e]
    kept = kept.masked_fill(~valid, -1).to(torch.int32)
    return [kept, new_lengths.to(torch.int32), state["key_pages"], state["value_pages"], moved]


def _framework():
    path = str(Path(__file__).resolve().parent.parent / "tac-vq-kv-cache_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import jointkv_amd

    return jointkv_amd


def _own(state):
    jkv = _framework()
    case = state["case"]
    if case["op"] == "append":
        starts = None if state["single"] else state["starts"]
        jkv.paged_append(state["key"], state["value"], state["key_pages"], state["value_pages"], state["tables"],
                         state["lengths"], starts=starts, positions=state["positions"], rope_theta=THETA)
        return [state["key_pages"], state["value_pages"]]
    if case["op"] == "evict":
        kept, lengths = jkv.select_entries(state["weights"], state["lengths"], case["budget"], sinks=case["sinks"],
                                           recent=case["recent"])
        moved = jkv.compact_pages(state["key_pages"], state["value_pages"], state["tables"], kept,
                                  state["new_tables"], weights=state["weights"])
        return [kept, lengths, state["key_pages"], state["value_pages"], moved]
    weights = state["weights"] if case["op"] == "weigh" else None
    out = jkv.paged_attention(
        state["query"], state["key_pages"], state["value_pages"], state["tables"], state["lengths"],
        starts=None if state["single"] else state["starts"], positions=state["positions"],
        window=case["window"] or None, sinks=case["sinks"], rope_theta=THETA, max_new=max(state["new_host"]),
        max_length=max(state["lengths_host"]), weights=weights)
    return [out] if weights is None else [out, weights]


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "append":
        return _plain_append(state)
    if op == "evict":
        return _plain_evict(state)
    return _plain_attention(state, op == "weigh")


# the definitions in 64 bits


def _turned(x, positions):
    """Rotary as a product of complex numbers."""

    half = x.shape[-1] // 2
    rate = torch.exp(torch.arange(half, dtype=torch.float64, device=x.device) * (-math.log(THETA) / half))
    turn = torch.polar(torch.ones_like(rate), rate)  # a turn by one position
    turn = torch.polar(torch.ones(len(positions), half, dtype=torch.float64, device=x.device),
                       torch.as_tensor(positions, dtype=torch.float64, device=x.device)[:, None] * turn.angle())
    z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn[:, None]
    return torch.cat((z.real, z.imag), -1)


def exact(case, seed):
    if case["op"] in ("attend", "weigh") and _pairs_and_entries(case)[0] * case["qh"] > 1 << 33:
        return None
    s = prepare(case, seed)
    page, kvh, dim, batch = case["page"], case["kvh"], case["dim"], case["batch"]
    tables = s["tables"].tolist()

    def where(b, entries):
        """Pool rows (page, slot) of entries of sequence b."""
        entries = np.asarray(entries, dtype=np.int64)
        pages = np.asarray(tables[b], dtype=np.int64)[entries // page]
        return (torch.from_numpy(pages).cuda(), torch.from_numpy(entries % page).cuda())

    if case["op"] == "append":
        keys, values = s["key_pages"].double(), s["value_pages"].double()
        at = 0
        for b, (first, last) in enumerate(_spans(case)):
            n = last - first
            pages, slots = where(b, np.arange(first, last))
            position = np.arange(n) + s["positions_host"][b]
            keys[pages, :, slots] = _turned(s["key"][at : at + n], position)
            values[pages, :, slots] = s["value"][at : at + n].double()
            at += n
        return [keys, values]
    if case["op"] == "evict":
        keys, values = s["key_pages"].double(), s["value_pages"].double()
        new_tables, weights = s["new_tables"].tolist(), s["weights"].double().cpu().numpy()
        kept_all = np.full((batch, kvh, case["budget"]), -1, dtype=np.int32)
        moved = np.zeros_like(weights)
        for b, length in enumerate(s["lengths_host"]):
            count = min(length, case["budget"])
            for h in range(kvh):
                w = weights[b, h, :length]
                middle = np.arange(length)
                if length > count:
                    inner = np.arange(case["sinks"], length - case["recent"])
                    best = inner[np.lexsort((inner, -w[inner]))][: count - case["sinks"] - case["recent"]]
                    middle = np.sort(np.concatenate((np.arange(case["sinks"]), best,
                                                     np.arange(length - case["recent"], length))))
                kept_all[b, h, :count] = middle
                moved[b, h, :count] = w[middle]
                pages, slots = where(b, middle)
                to = torch.tensor([new_tables[b][j // page] for j in range(count)], device="cuda")
                to_slot = torch.arange(count, device="cuda") % page
                keys[to, h, to_slot] = keys[pages, h, slots]
                values[to, h, to_slot] = values[pages, h, slots]
        lengths = np.minimum(s["lengths_host"], case["budget"]).astype(np.int32)
        return [kept_all, lengths, keys, values, moved]
    out, weights, at = [], s["weights"].double(), 0
    per = case["qh"] // kvh
    for b, (first, last) in enumerate(_spans(case)):
        n = last - first
        query = _turned(s["query"][at : at + n], np.arange(n) + s["positions_host"][b])
        at += n
        pages, slots = where(b, np.arange(last))
        keys, values = s["key_pages"][pages, :, slots].double(), s["value_pages"][pages, :, slots].double()
        i = torch.arange(first, last, device="cuda")[:, None]
        j = torch.arange(last, device="cuda")[None]
        hidden = j > i
        if case["window"]:
            hidden |= (j <= i - case["window"]) & (j >= case["sinks"])
        of_heads = []
        for h in range(kvh):
            received = torch.zeros(last, dtype=torch.float64, device="cuda")
            for g in range(per):
                logits = query[:, h * per + g] @ keys[:, h].T.contiguous() * dim ** -0.5
                p = torch.softmax(logits.masked_fill(hidden, float("-inf")), -1)
                of_heads.append(p @ values[:, h].contiguous())
                received += p.sum(0)
            weights[b, h, :last] = received
        out.append(torch.stack(of_heads, 1))
    out = torch.cat(out)
    return [out] if case["op"] == "attend" else [out, weights]

"""Attention over a paged 8-bit key/value cache: the cases that are measured.

Three operators of the serving path work on one cache, whose pages hold ``page`` tokens of
every key/value head in 8 bits with one scale for each page and head:

* ``write``   quantises new keys and values into the pages of their sequences (a page that
              already holds tokens is rescaled when a larger value arrives) and returns the
              touched pages as the values they now stand for,
* ``read``    gives back a range of every sequence in a floating type,
* ``attend``  attention of new query tokens over the cached sequences, causal, with grouped
              heads, ragged lengths and an optional sliding window.

``run`` computes them with elementary torch operations in 32 bits, or, with ``own`` set,
through the backend of this repository.
"""
import math
import random

import torch

own = False

_FLOAT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = torch.finfo(torch.float32).eps
_LARGEST = {"int8": 127.0, "e4m3": 448.0}


# --------------------------------------------------------------------------------------
# cases
# --------------------------------------------------------------------------------------
def _case(kind, name=None, **values):
    case = {"kind": kind, "batch": 1, "new_min": 1, "new_max": 1, "past_min": 0, "past_max": 0, "heads": 12,
            "kv_heads": 12, "dim": 64, "page": 64, "cache": "int8", "dtype": "fp16", "window": 0, "idle": 0,
            "fused": False, "lse": False}
    case.update(values)
    if name is not None:
        case["name"] = name
    return case


def listed():
    return [
        # one decode step of a small decoder (12 heads of 64): 8 sequences append a token each,
        # most of them into a page that already holds tokens
        _case("write", "write_8x1_12h64", batch=8, past_min=512, past_max=639, fused=True),
        # a prompt of 4096 tokens of a 32-head model arrives, its k and v column blocks of one
        # fused projection
        _case("write", "write_4096_32h128", new_min=4096, new_max=4096, heads=32, kv_heads=32, dim=128,
              fused=True),
        # mixed batch of a server: prompts of odd lengths behind cached prefixes
        _case("write", "write_mixed_24_8h128_e4m3", batch=24, new_min=1, new_max=1531, past_min=0, past_max=2000, heads=32,
              kv_heads=8, dim=128, page=32, cache="e4m3", dtype="bf16"),
        # cached prefixes handed to a consumer of floating keys and values: a short batch, a long sequence
        _case("read", "read_8x640_12h64", batch=8, past_min=513, past_max=640),
        _case("read", "read_65537_8h128", past_min=65537, past_max=65537, heads=32, kv_heads=8, dim=128,
              dtype="bf16"),
        # decode of the small decoder: the smallest call, latency counts
        _case("attend", "decode_8x640_12h64", batch=8, past_min=512, past_max=639, fused=True),
        # decode of a ragged server batch with grouped heads; two slots of the batch are idle
        _case("attend", "decode_64x8k_32over8h128", batch=64, past_min=0, past_max=8191, heads=32, kv_heads=8,
              dim=128, dtype="bf16", idle=2),
        # one long conversation: few rows, so the long axis has to be split
        _case("attend", "decode_1x131072_32over8h128_e4m3", past_min=131071, past_max=131071, heads=32, kv_heads=8,
              dim=128, cache="e4m3", dtype="bf16", lse=True),
        # several drafted tokens verified at once, heads of 80, small pages, sliding window
        _case("attend", "verify_16x5_16over4h80_window", batch=16, new_min=3, new_max=5, past_min=100,
              past_max=5000, heads=16, kv_heads=4, dim=80, page=16, window=1024),
        # prefill of the small decoder: 8 prompts of 512 tokens
        _case("attend", "prompt_8x512_12h64", batch=8, new_min=512, new_max=512, fused=True),
        # prefill of a 32-head model: one prompt of 4096 tokens
        _case("attend", "prompt_4096_32h128", new_min=4096, new_max=4096, heads=32, kv_heads=32, dim=128),
        # a chunk of a long prompt behind what is cached of it, grouped heads
        _case("attend", "chunk_509_past_32768_32over8h128", new_min=509, new_max=509, past_min=32768,
              past_max=32768, heads=32, kv_heads=8, dim=128, page=128, dtype="bf16", lse=True),
    ]


def _log_int(rng, low, high):
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """One more case of the ranges above."""
    while True:
        kind = rng.choice(("write", "read", "attend", "attend", "attend"))
        kv_heads = rng.choice((1, 2, 4, 8, 12, 32))
        heads = kv_heads * (1 if kv_heads > 8 else rng.choice((1, 1, 3, 4, 7, 8)))
        case = _case(kind, kv_heads=kv_heads, heads=heads, dim=rng.choice((64, 64, 80, 96, 128, 128, 256)),
                     page=rng.choice((16, 32, 64, 128)), cache=rng.choice(("int8", "int8", "e4m3")),
                     dtype=rng.choice(("fp16", "bf16")), batch=_log_int(rng, 1, 64))
        if kind == "read":
            case["past_max"] = _log_int(rng, 17, 65536)
            case["past_min"] = rng.randint(1, case["past_max"])
        else:
            case["fused"] = heads == kv_heads and rng.random() < 0.5
            if rng.random() < 0.5:                               # decode and verification
                case["new_max"] = rng.choice((1, 1, 1, 2, 5, 8))
                case["past_max"] = _log_int(rng, 16, 131072)
                case["past_min"] = rng.randint(0, case["past_max"])
            else:                                                # prompts and chunks of them
                case["new_max"] = _log_int(rng, 17, 4096)
                case["past_max"] = rng.choice((0, 0, _log_int(rng, 16, 32768)))
                case["past_min"] = rng.randint(0, case["past_max"])
                case["batch"] = min(case["batch"], 16)
            case["new_min"] = rng.randint(1, case["new_max"])
            if kind == "attend":
                case["window"] = rng.choice((0, 0, 0, _log_int(rng, 16, 4096)))
                case["idle"] = rng.choice((0, 0, 1)) if case["batch"] > 1 else 0
                case["lse"] = case["idle"] == 0 and rng.random() < 0.5
        if _within(case):
            return case


def _within(case):
    """No more work than the largest listed cases, and plain intermediates of a few GB."""
    need = work(case)
    padded = case["batch"] * (case["past_max"] + case["new_max"])
    scores = padded * case["heads"] * case["new_max"] if case["kind"] == "attend" else 0
    return (need["bytes"] <= 5.3e8 and need["flops"] <= 2.7e11 and scores <= 6e8
            and padded * case["kv_heads"] * case["dim"] <= 6e8)


# --------------------------------------------------------------------------------------
# shapes that follow from a case alone
# --------------------------------------------------------------------------------------
def _lengths(case):
    """(cached tokens before the call, new tokens) of every sequence."""
    pairs = []
    for b in range(case["batch"]):
        at = b / max(1, case["batch"] - 1)
        other = (b * 7 % case["batch"]) / max(1, case["batch"] - 1)
        past = round(case["past_max"] + (case["past_min"] - case["past_max"]) * at)
        new = round(case["new_max"] + (case["new_min"] - case["new_max"]) * other)
        pairs.append((past, 0 if case["kind"] == "read" else new))
    return pairs


def _visible(case, past, new):
    """(pairs of query and key that meet, tokens of the cache that any query meets)."""
    window, total = case["window"], past + new
    pairs = sum(min(p + 1, window) if window else p + 1 for p in range(past, total))
    first = max(0, past + 1 - window) if window else 0
    return pairs, total - first


def work(case):
    wide = case["kv_heads"] * case["dim"]
    size = 4 if case["dtype"] == "fp32" else 2
    pairs = _lengths(case)
    if case["kind"] == "read":
        rows = sum(past for past, _ in pairs)
        return {"bytes": rows * 2 * wide * (1 + size), "flops": rows * 2 * wide}
    if case["kind"] == "write":
        new = sum(n for _, n in pairs)
        rows = sum(past + n - past // case["page"] * case["page"] for past, n in pairs)
        return {"bytes": new * 2 * wide * (size + 1) + rows * 2 * wide * size, "flops": rows * 2 * wide * 4}
    met = keys = 0
    for i, (past, new) in enumerate(pairs):
        if i >= case["batch"] - case["idle"]:
            continue
        a, b = _visible(case, past, new)
        met, keys = met + a, keys + b
    tokens = sum(n for _, n in pairs)
    return {"bytes": keys * 2 * wide + tokens * case["heads"] * case["dim"] * 2 * size,
            "flops": 4 * met * case["heads"] * case["dim"]}


# --------------------------------------------------------------------------------------
# inputs
# --------------------------------------------------------------------------------------
def _to_cache(x, cache):
    if cache == "int8":
        return x.round().clamp(-127, 127).to(torch.int8)
    return x.to(torch.float8_e4m3fn).view(torch.int8)


def _from_cache(q, cache, dtype=torch.float32):
    if cache == "int8":
        return q.to(dtype)
    return q.view(torch.float8_e4m3fn).to(dtype)


def _filled(pages, case, gen, spread):
    """Random pages in 8 bits with their scales: channels of different size, pages too."""
    heads, page, dim, device = case["kv_heads"], case["page"], case["dim"], "cuda"
    data = torch.empty((pages, heads, page, dim), dtype=torch.int8, device=device)
    scale = torch.empty((pages, heads), dtype=torch.float32, device=device)
    channel = 0.5 + 1.5 * torch.rand((heads, 1, dim), generator=gen, device=device) ** 4 * spread
    step = max(1, (1 << 26) // (heads * page * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn((n, heads, page, dim), generator=gen, device=device) * channel
        x *= 0.5 + torch.rand((n, heads, 1, 1), generator=gen, device=device)
        s = x.abs().amax(dim=(2, 3)).clamp_min(_EPS) / _LARGEST[case["cache"]]
        scale[at:at + n] = s
        data[at:at + n] = _to_cache(x / s[:, :, None, None], case["cache"])
    return data, scale


def prepare(case, seed):
    rng = random.Random(seed * 7919 + 17)
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed * 1000003 + 11)
    page, kv_heads, dim, heads = case["page"], case["kv_heads"], case["dim"], case["heads"]
    dtype = _FLOAT[case["dtype"]]
    pairs = _lengths(case)
    live, idle = pairs[:len(pairs) - case["idle"]], pairs[len(pairs) - case["idle"]:]
    rng.shuffle(live)
    pairs = live + [(0, n) for _, n in idle]
    # an idle slot of a fixed batch still has its query tokens, but nothing cached
    totals = [0 if i >= len(live) else past + new for i, (past, new) in enumerate(pairs)]
    counts = [-(-t // page) for t in totals]
    width = max(counts) + 1
    pages = sum(counts) + 3
    order = list(range(pages))
    rng.shuffle(order)
    table = [[0] * width for _ in pairs]
    at = 0
    for b, count in enumerate(counts):
        table[b][:count] = order[at:at + count]
        at += count
    k_data, k_scale = _filled(pages, case, gen, 2.0)
    v_data, v_scale = _filled(pages, case, gen, 0.5)
    new = [n for _, n in pairs]
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state = {"case": case, "k": k_data, "v": v_data, "k_scale": k_scale, "v_scale": v_scale,
             "table": torch.tensor(table, dtype=torch.int32, device="cuda"),
             "lens": torch.tensor(totals, dtype=torch.int32, device="cuda"),
             "starts": torch.tensor(starts, dtype=torch.int32, device="cuda"), "max_new": max(new)}
    tokens = starts[-1]
    if case["kind"] == "read":
        rows = [0]
        for t in totals:
            rows.append(rows[-1] + t)
        first = [0] * len(pairs)
    else:
        # rows of the pages that a write touches, from the start of the first of them
        first = [past // page * page for past, _ in pairs]
        rows = [0]
        for (past, n), f in zip(pairs, first):
            rows.append(rows[-1] + past + n - f)
    state["first"] = torch.tensor(first, dtype=torch.int32, device="cuda")
    state["rows"] = torch.tensor(rows, dtype=torch.int32, device="cuda")
    state["n_rows"] = rows[-1]
    state["max_rows"] = max(b - a for a, b in zip(rows, rows[1:]))

    def tensor(n_heads, gain):
        return torch.randn((tokens, n_heads, dim), generator=gen, device="cuda") * gain

    if case["kind"] != "read":
        q = (tensor(heads, 1.5)).to(dtype)
        if case["kind"] == "write":
            k = (tensor(kv_heads, 1.0) * (0.5 + torch.rand((1, kv_heads, dim), generator=gen, device="cuda") ** 4 * 4))
            k = k.to(dtype)
            v = tensor(kv_heads, 0.8).to(dtype)
            if case["fused"]:                       # column blocks of one fused projection
                qkv = torch.cat((q, k, v), dim=1)
                k, v = qkv[:, heads:heads + kv_heads], qkv[:, heads + kv_heads:]
            state["new_k"], state["new_v"] = k, v
            touched = [(b, p) for b, (past, n) in enumerate(pairs) if n
                       for p in range(past // page, -(-(past + n) // page))]
            state["touched"] = torch.tensor(touched, dtype=torch.int64, device="cuda")
        else:
            if case["fused"]:
                wide = torch.empty((tokens, heads + 2 * kv_heads, dim), dtype=dtype, device="cuda")
                wide[:, :heads] = q
                wide[:, heads:] = 0
                q = wide[:, :heads]
            state["q"] = q
    if own:
        from rns_llm_b200.backends import CudaRNSBackend, QuantizedKVCache

        state["backend"] = CudaRNSBackend()
        kind = torch.int8 if case["cache"] == "int8" else torch.float8_e4m3fn
        state["cache"] = QuantizedKVCache(k=k_data.view(kind), v=v_data.view(kind), k_scale=k_scale, v_scale=v_scale)
    return state


# --------------------------------------------------------------------------------------
# the operators
# --------------------------------------------------------------------------------------
def run(state):
    case = state["case"]
    if own:
        return _run_own(state, case)
    if case["kind"] == "write":
        for which in ("k", "v"):
            _plain_write(state, case, which)
    if case["kind"] != "attend":
        k, v = (_plain_read(state, case, which) for which in ("k", "v"))
        if case["kind"] == "read":
            return k, v
        return k, v, state["k_scale"], state["v_scale"]
    return _plain_attend(state, case)


def _run_own(state, case):
    backend, cache, table = state["backend"], state["cache"], state["table"]
    dtype = _FLOAT[case["dtype"]]
    if case["kind"] == "attend":
        return backend.kv_cache_attention(
            state["q"], cache, table, state["lens"], state["starts"], max_query_len=state["max_new"],
            softmax_scale=case["dim"] ** -0.5, causal=True, window=case["window"] or None, return_lse=case["lse"])
    if case["kind"] == "write":
        backend.kv_cache_write(cache, state["new_k"], state["new_v"], table, state["lens"], state["starts"],
                               max_query_len=state["max_new"])
    k, v = backend.kv_cache_read(cache, table, state["first"], state["rows"], rows=state["n_rows"],
                                 max_rows=state["max_rows"], dtype=dtype)
    if case["kind"] == "read":
        return k, v
    return k, v, cache.k_scale, cache.v_scale


def _row_owner(starts, rows):
    """(sequence, index inside it) of every packed row."""
    at = torch.arange(rows, device=starts.device)
    owner = torch.searchsorted(starts[1:].long(), at, right=True)
    return owner, at - starts.long()[owner]


def _plain_write(state, case, which):
    page, largest = case["page"], _LARGEST[case["cache"]]
    data, scale, x = state[which], state[which + "_scale"], state["new_" + which]
    seq, nth = state["touched"][:, 0], state["touched"][:, 1]
    lens, starts = state["lens"].long(), state["starts"].long()
    begin = (lens - (starts[1:] - starts[:-1]))[seq]                      # first new position
    pos = nth[:, None] * page + torch.arange(page, device=x.device)       # [touched, page]
    fresh = (pos >= begin[:, None]) & (pos < lens[seq][:, None])
    kept = pos < begin[:, None]
    token = (starts[:-1][seq][:, None] + pos - begin[:, None]).clamp(0, x.shape[0] - 1)
    values = x[token].float().permute(0, 2, 1, 3)                         # [touched, heads, page, dim]
    values = values * fresh[:, None, :, None]
    ids = state["table"].long()[seq, nth]
    old = data[ids]
    old_scale = torch.where(kept[:, 0][:, None], scale[ids], torch.zeros_like(scale[ids]))
    wanted = values.abs().amax(dim=(2, 3)).clamp_min(_EPS) / torch.full_like(old_scale, largest)
    new_scale = torch.maximum(wanted, old_scale)
    ratio = old_scale / new_scale
    again = _to_cache(_from_cache(old, case["cache"]) * ratio[:, :, None, None], case["cache"])
    put = _to_cache(values / new_scale[:, :, None, None], case["cache"])
    data[ids] = torch.where(fresh[:, None, :, None], put, torch.where(kept[:, None, :, None], again, old))
    scale[ids] = new_scale


def _plain_read(state, case, which):
    owner, at = _row_owner(state["rows"], state["n_rows"])
    pos = state["first"].long()[owner] + at
    ids = state["table"].long()[owner, pos // case["page"]]
    values = _from_cache(state[which][ids, :, pos % case["page"]], case["cache"])
    return (values * state[which + "_scale"][ids][:, :, None]).to(_FLOAT[case["dtype"]])


def _plain_attend(state, case):
    page, dim, heads, kv_heads = case["page"], case["dim"], case["heads"], case["kv_heads"]
    group, batch, most = heads // kv_heads, case["batch"], state["max_new"]
    q, lens, starts, table = state["q"], state["lens"].long(), state["starts"].long(), state["table"].long()
    width = table.shape[1] - 1 or 1
    ids = table[:, :width]

    def padded(which):                                                    # [batch, kv_heads, keys, dim]
        values = _from_cache(state[which][ids], case["cache"])
        values *= state[which + "_scale"][ids][:, :, :, None, None]
        return values.permute(0, 2, 1, 3, 4).reshape(batch, kv_heads, width * page, dim)

    new = starts[1:] - starts[:-1]
    step = torch.arange(most, device=q.device)
    row = (starts[:-1][:, None] + step).clamp_max(q.shape[0] - 1)
    rows = q[row].float().permute(0, 2, 1, 3).reshape(batch, kv_heads, group * most, dim)
    scores = torch.matmul(rows, padded("k").transpose(2, 3)) * dim ** -0.5
    scores = scores.view(batch, kv_heads, group, most, width * page)
    key = torch.arange(width * page, device=q.device)
    last = (lens - new)[:, None] + step                                   # position of each query
    seen = (key <= last[:, :, None]) & (key < lens[:, None, None])
    if case["window"]:
        seen &= key > last[:, :, None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], float("-inf"))
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(top == float("-inf"), torch.zeros_like(top), top)
    scores -= top
    scores.exp_()
    total = scores.sum(dim=-1, keepdim=True)
    out = torch.matmul(scores.view(batch, kv_heads, group * most, width * page), padded("v"))
    out = out.view(batch, kv_heads, group, most, dim) / torch.where(total > 0, total, torch.ones_like(total))
    owner, at = _row_owner(state["starts"], q.shape[0])
    result = out.permute(0, 3, 1, 2, 4).reshape(batch, most, heads, dim)[owner, at].to(q.dtype)
    if not case["lse"]:
        return result
    lse = (top + total.log()).squeeze(-1)
    return result, lse.permute(0, 3, 1, 2).reshape(batch, most, heads)[owner, at]


# --------------------------------------------------------------------------------------
# the definition in 64 bits
# --------------------------------------------------------------------------------------
def exact(case, seed):
    """Each sequence and head by itself, in float64.  The 8-bit grid is part of the definition:
    scales and quotients are 32-bit numbers (a quotient of two of them rounded from 64 bits is
    the correctly rounded one), and what is rounded to the grid is rounded from those."""
    global own
    saved, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = saved
    page = case["page"]
    lens, starts, table = (state[n].tolist() for n in ("lens", "starts", "table"))

    def sequence(which, b, first, end):                                    # [kv_heads, tokens, dim]
        ids = torch.tensor(table[b][first // page:-(-end // page)], dtype=torch.int64, device="cuda")
        wide = _from_cache(state[which][ids], case["cache"]).double() * state[which + "_scale"][ids].double()[..., None, None]
        return wide.transpose(0, 1).flatten(1, 2)[:, first % page:first % page + end - first]

    if case["kind"] == "attend":
        return _exact_attend(case, state, sequence, lens, starts)
    if case["kind"] == "write":
        for which in ("k", "v"):
            _exact_write(case, state, which, lens, starts, table)
    outputs = []
    for which in ("k", "v"):
        parts = [sequence(which, b, first, lens[b]).transpose(0, 1)
                 for b, first in enumerate(state["first"].tolist()) if lens[b] > first]
        outputs.append(torch.cat(parts))
    if case["kind"] == "write":
        outputs += [state["k_scale"].double(), state["v_scale"].double()]
    return tuple(outputs)


def _exact_write(case, state, which, lens, starts, table):
    page, largest = case["page"], _LARGEST[case["cache"]]

    def grid(x):
        x = x.float()
        return x.round().clamp(-127, 127).to(torch.int8) if case["cache"] == "int8" else \
            x.to(torch.float8_e4m3fn).view(torch.int8)

    for b, end in enumerate(lens):
        begin = end - (starts[b + 1] - starts[b])
        for nth in range(begin // page, -(-end // page)):
            at, stop = max(begin, nth * page), min(end, nth * page + page)
            x = state["new_" + which][starts[b] + at - begin:starts[b] + stop - begin].double().transpose(0, 1)
            held = at - nth * page                                         # tokens that stay in the page
            entry, scales = state[which][table[b][nth]], state[which + "_scale"][table[b][nth]]
            scale = (x.abs().amax(dim=(1, 2)).clamp_min(_EPS) / largest).float().double()
            if held:
                scale = torch.maximum(scale, scales.double())
                ratio = (scales.double() / scale).float().double()
                before = _from_cache(entry[:, :held], case["cache"]).double()
                entry[:, :held] = grid(before * ratio[:, None, None])
            entry[:, held:held + stop - at] = grid(x / scale[:, None, None])
            scales.copy_(scale.float())


def _exact_attend(case, state, sequence, lens, starts):
    heads, dim = case["heads"], case["dim"]
    group = heads // case["kv_heads"]
    q = state["q"]
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:2], float("-inf"), dtype=torch.float64, device="cuda")
    for b, end in enumerate(lens):
        if end == 0:
            continue
        keys, values = sequence("k", b, 0, end), sequence("v", b, 0, end)
        position = torch.arange(end - (starts[b + 1] - starts[b]), end, device="cuda")[:, None]
        key = torch.arange(end, device="cuda")[None]
        hidden = key > position
        if case["window"]:
            hidden = hidden | (key <= position - case["window"])
        for h in range(heads):
            s = q[starts[b]:starts[b + 1], h].double() @ keys[h // group].T / dim ** 0.5
            s = s.masked_fill(hidden, float("-inf"))
            lse[starts[b]:starts[b + 1], h] = torch.logsumexp(s, dim=1)
            out[starts[b]:starts[b + 1], h] = torch.softmax(s, dim=1) @ values[h // group]
    return (out, lse) if case["lse"] else out

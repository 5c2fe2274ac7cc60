"""The paged 8-bit KV cache's operators, as cases to be timed and compared.

Four kinds of case, in the order in which a serving step calls them:

* ``plan``: block tables, slot map, positions and lengths of a step, from the requests'
  lengths (``sparknet.ops.plan_pages``);
* ``append``: new keys and values into e4m3 pages with one power-of-two scale for each
  (page, KV head), then the sequences' values read back (``kv_append`` /
  ``rope_kv_append``, then ``kv_read``);
* ``read``: cached keys and values by slot, in a 16-bit type (``kv_read``);
* ``attention``: decode attention over the pages (``paged_decode_attention``).

Without ``own`` a pass computes the same in elementary torch operations in fp32.
"""

import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
E4M3_MAX = 448.0
MIN_EXPONENT = -100


# -- cases -------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small batch: latency of the bookkeeping alone
        {"name": "plan, 8 requests decode", "op": "plan", "requests": 8, "page": 64, "context": 1024, "chunk": 0,
         "finished": False},
        # a busy server's step: most requests decode, some bring a chunk of their prompt, some have ended
        {"name": "plan, 1024 requests mixed", "op": "plan", "requests": 1024, "page": 16, "context": 2000,
         "chunk": 512, "finished": True},
        # one token of each of 8 sequences on a TP8 rank (8 query heads, 1 KV head), RoPE fused
        {"name": "append, 8 tokens rope", "op": "append", "sequences": 8, "tokens": 1, "context": 300, "heads": 8,
         "kv_heads": 1, "dim": 128, "page": 64, "rope": True, "dtype": "bf16"},
        # one token of each of 64 sequences on one GPU (64 query heads, 8 KV heads), RoPE fused
        {"name": "append, 64 tokens rope", "op": "append", "sequences": 64, "tokens": 1, "context": 63, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "rope": True, "dtype": "bf16"},
        # a prompt's chunks, odd length, starting inside a page
        {"name": "append, 4 chunks of 2047", "op": "append", "sequences": 4, "tokens": 2047, "context": 37,
         "heads": 0, "kv_heads": 8, "dim": 128, "page": 32, "rope": False, "dtype": "fp16"},
        # a short cached prefix read back for a prompt's own attention
        {"name": "read, 500 tokens", "op": "read", "sequences": 1, "context": 500, "kv_heads": 8, "dim": 64,
         "page": 16, "dtype": "bf16"},
        # long cached prefixes of several sequences
        {"name": "read, 16 x 8191 tokens", "op": "read", "sequences": 16, "context": 8191, "kv_heads": 8, "dim": 128,
         "page": 64, "dtype": "bf16"},
        # one short chat, one token: latency
        {"name": "attention, 1 x 500", "op": "attention", "sequences": 1, "tokens": 1, "context": 500, "heads": 64,
         "kv_heads": 8, "dim": 128, "page": 64, "ragged": False, "window": 0, "dtype": "bf16"},
        # a TP8 rank's decode step: 8 query heads on 1 KV head
        {"name": "attention, 8 x 1024 TP8", "op": "attention", "sequences": 8, "tokens": 1, "context": 1024,
         "heads": 8, "kv_heads": 1, "dim": 128, "page": 64, "ragged": False, "window": 0, "dtype": "bf16"},
        # a ragged batch with padded (empty) rows, small pages
        {"name": "attention, 64 ragged to 8192", "op": "attention", "sequences": 64, "tokens": 1, "context": 8192,
         "heads": 64, "kv_heads": 8, "dim": 128, "page": 16, "ragged": True, "window": 0, "dtype": "bf16"},
        # checking four drafted tokens at once, head size 64, sliding window
        {"name": "attention, 16 x 4 drafted", "op": "attention", "sequences": 16, "tokens": 4, "context": 5001,
         "heads": 32, "kv_heads": 8, "dim": 64, "page": 32, "ragged": True, "window": 4096, "dtype": "fp16"},
        # few long contexts: the key axis is all the parallelism there is
        {"name": "attention, 2 x 131072", "op": "attention", "sequences": 2, "tokens": 1, "context": 131072,
         "heads": 64, "kv_heads": 8, "dim": 128, "page": 128, "ragged": False, "window": 0, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(("plan", "append", "read", "attention", "attention"))
    page = rng.choice((16, 32, 64, 128))
    dim = rng.choice((64, 128, 128))
    dtype = rng.choice(("bf16", "bf16", "fp16"))
    if op == "plan":
        return {"op": op, "requests": _log_int(rng, 1, 1024), "page": page, "context": _log_int(rng, 1, 4000),
                "chunk": rng.choice((0, 0, _log_int(rng, 2, 512))), "finished": rng.random() < 0.5}
    kv_heads = rng.choice((1, 2, 4, 8))
    group = rng.choice((1, 2, 4, 7, 8, 16))
    if op == "append":
        rope = rng.random() < 0.5
        tokens = rng.choice((1, 1, _log_int(rng, 2, 2047)))
        sequences = _log_int(rng, 1, max(1, min(256, 8188 // tokens)))
        return {"op": op, "sequences": sequences, "tokens": tokens, "context": rng.randint(0, 300),
                "heads": kv_heads * group if rope else 0, "kv_heads": kv_heads, "dim": dim, "page": page,
                "rope": rope, "dtype": "bf16" if rope else dtype}
    if op == "read":
        context = _log_int(rng, 1, 32768)
        return {"op": op, "sequences": _log_int(rng, 1, max(1, min(64, 131072 // context))), "context": context,
                "kv_heads": kv_heads, "dim": dim, "page": page, "dtype": dtype}
    context, tokens = _log_int(rng, 1, 65536), rng.choice((1, 1, 1, rng.randint(2, 8)))
    return {"op": op, "sequences": _log_int(rng, 1, max(1, min(128, 262144 // (tokens * context)))),
            "tokens": tokens, "context": context, "heads": kv_heads * group,
            "kv_heads": kv_heads, "dim": dim, "page": page, "ragged": rng.random() < 0.6,
            "window": rng.choice((0, 0, 0, _log_int(rng, 16, 8192))), "dtype": dtype}


def _plan_lengths(case):
    """Lengths held, new tokens and ended requests of a plan case: its shape, the same for every seed."""
    rng = random.Random("plan %d %d %d" % (case["requests"], case["context"], case["chunk"]))
    n = case["requests"]
    held = [rng.randint(0, case["context"]) for _ in range(n)]
    new = [rng.randint(2, case["chunk"]) if case["chunk"] > 1 and rng.random() < 0.15 else 1 for _ in range(n)]
    ended = [case["finished"] and rng.random() < 0.1 for _ in range(n)]
    new = [0 if e else k for k, e in zip(new, ended)]
    return held, new, ended


def _lengths(case):
    """Keys held by each sequence of a read or attention case: its shape, the same for every seed."""
    n, most = case["sequences"], case["context"]
    if not case.get("ragged"):
        return [most] * n
    rng = random.Random("lengths %d %d" % (n, most))
    got = [0 if rng.random() < 0.08 else rng.randint(1, most) for _ in range(n)]
    got[rng.randrange(n)] = most
    return got


def _pages(length, page):
    return -(-length // page)


def _seen(case):
    """(keys read, (query row, key) pairs per query head) of an attention case."""
    t, window = case["tokens"], case["window"]
    keys = pairs = 0
    for n in _lengths(case):
        first = n
        for i in range(t):
            last = n - t + i + 1
            if last <= 0:
                continue
            low = max(0, last - window) if window else 0
            pairs += last - low
            first = min(first, low)
        keys += n - first
    return keys, pairs


def work(case):
    op = case["op"]
    if op == "plan":
        held, new, ended = _plan_lengths(case)
        page = case["page"]
        moved = sum(_pages(h, page) for h, e in zip(held, ended) if e)
        got = sum(_pages(h + k, page) - _pages(h, page) for h, k, e in zip(held, new, ended) if not e)
        # lengths, new and ended in; lengths, granted, row starts out; pages moved; slot and position of each row
        return {"bytes": 4 * (6 * case["requests"] + 2 * moved + 2 * got + 2 * sum(new)), "flops": 0}
    values = 2 * case["kv_heads"] * case["dim"]  # K and V of one token
    size = 4 if case["dtype"] == "fp32" else 2
    if op == "append":
        n = case["sequences"] * case["tokens"]
        read_back = case["sequences"] * (case["context"] + case["tokens"])
        moved = n * values * (size + 1) + n * case["heads"] * case["dim"] * 2 * size
        return {"bytes": moved + read_back * values * (1 + 2), "flops": 4 * n * values}
    if op == "read":
        return {"bytes": sum(_lengths(case)) * values * (1 + size), "flops": 0}
    keys, pairs = _seen(case)
    q = case["sequences"] * case["tokens"] * case["heads"] * case["dim"]
    scales = keys // case["page"] * 2 * case["kv_heads"] * 4
    return {"bytes": keys * values + scales + 2 * q * size, "flops": 4 * pairs * case["heads"] * case["dim"]}


# -- inputs ------------------------------------------------------------------------------
def _exponent(amax):
    """Smallest e >= MIN_EXPONENT with amax <= 448 * 2^e, as floats; 448 = 0.875 * 2^9."""
    mantissa, exponent = torch.frexp(amax)
    e = exponent - torch.where(mantissa <= 0.875, 9, 8)
    return torch.where(amax > 0, e, MIN_EXPONENT).clamp_min(MIN_EXPONENT)


def _quantise_pages(x):
    """Pages of values [pages, heads, page, dim] -> codes, scales [pages, heads]."""
    scale = torch.ldexp(torch.ones((), device=x.device), _exponent(x.abs().amax((2, 3)).float()))
    return (x.float() / scale[:, :, None, None]).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn), scale


def _values(gen, shape, dim, key):
    """Keys with a few strong channels, as models have; values plain."""
    x = torch.randn(shape, generator=gen, device=gen.device, dtype=torch.float32)
    return x * _strength(dim, gen.device) if key else x


def _strength(dim, device):
    return 1.0 + 4.0 * (torch.arange(dim, device=device) % 29 == 3)


def _cache(gen, case, pages):
    """A filled pool of pages: codes and scales of K and V, made in pieces."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    state = {}
    for name in ("k", "v"):
        codes = torch.empty(shape, dtype=torch.float8_e4m3fn, device=gen.device)
        scale = torch.empty(shape[:2], device=gen.device)
        step = max(1, (1 << 27) // math.prod(shape[1:]))
        for at in range(0, pages, step):
            n = min(step, pages - at)
            codes[at:at + n], scale[at:at + n] = _quantise_pages(_values(gen, (n, *shape[1:]), case["dim"],
                                                                         name == "k"))
        state[name], state[name + "_scale"] = codes, scale
    if own:
        from sparknet.ops import Fp8KVCache

        state["cache"] = Fp8KVCache.from_tensors(state["k"], state["v"], state["k_scale"], state["v_scale"])
    return state


def _tables(gen, lengths, page):
    """Pages in random order for sequences of these lengths: (tables [n, width] int32, pages in the pool)."""
    counts = [_pages(n, page) for n in lengths]
    width, pool = max(1, max(counts)), sum(counts) + 3
    order = torch.randperm(pool, generator=gen, device=gen.device).int()
    counts = torch.tensor(counts, device=gen.device)
    at = torch.arange(width, device=gen.device)
    index = (counts.cumsum(0) - counts)[:, None] + at
    return torch.where(at < counts[:, None], order[index.clamp_max(pool - 1)], 0), pool


def _slots(tables, start, lengths, page, device):
    """Slots of positions start[i] .. lengths[i] of each sequence, packed, int32."""
    at = [torch.arange(a, b, device=device) for a, b in zip(start, lengths)]
    return torch.cat([tables[i][p // page] * page + (p % page) for i, p in enumerate(at)]).int()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    op, page, device = case["op"], case["page"], gen.device
    state = {"case": case}
    if op == "plan":
        held, new, ended = _plan_lengths(case)
        tables, pool = _tables(gen, held, page)
        width = _pages(case["context"] + max(1, case["chunk"]), page)
        tables = torch.nn.functional.pad(tables, (0, width - tables.shape[1])).contiguous()
        spare = sum(_pages(h + k, page) - _pages(h, page) for h, k in zip(held, new)) + 5
        free = torch.randperm(spare, generator=gen, device=device).int() + pool
        state |= {"lengths": torch.tensor(held, dtype=torch.int32, device=device),
                  "new": torch.tensor(new, dtype=torch.int32, device=device), "tables": tables,
                  "free": torch.cat([free, torch.zeros(pool, dtype=torch.int32, device=device)]),
                  "count": torch.tensor([spare], dtype=torch.int32, device=device),
                  "ended": torch.tensor(ended, device=device) if case["finished"] else None,
                  "rows": sum(new) + 7}
        return state
    dtype, dim, heads = DTYPES[case["dtype"]], case["dim"], case["kv_heads"]
    if op == "append":
        n, t = case["sequences"], case["tokens"]
        start, lengths = [case["context"]] * n, [case["context"] + t] * n
        tables, pool = _tables(gen, lengths, page)
        state |= _cache(gen, case, pool)
        state["slots"] = _slots(tables, start, lengths, page, device)
        state["all"] = _slots(tables, [0] * n, lengths, page, device)
        x = torch.cat([_values(gen, (n * t, case["heads"] + heads, dim), dim, True),
                       _values(gen, (n * t, heads, dim), dim, False)], 1)
        if case["rope"]:
            state["qkv"] = x.to(dtype).flatten(1)
            state["positions"] = (torch.arange(t, device=device).repeat(n) + case["context"]).int()
            inverse = 500000.0 ** (-torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
            angle = torch.arange(case["context"] + t, device=device, dtype=torch.float64)[:, None] * inverse
            state["cos"], state["sin"] = angle.cos().float(), angle.sin().float()
        else:
            x = x.to(dtype)
            state["new_k"], state["new_v"] = x[:, :heads], x[:, heads:]
        return state
    lengths = _lengths(case)
    tables, pool = _tables(gen, lengths, page)
    state |= _cache(gen, case, pool)
    if op == "read":
        state["slots"] = _slots(tables, [0] * len(lengths), lengths, page, device)
        return state
    shape = (case["sequences"], case["tokens"], case["heads"], dim)
    state["q"] = (_values(gen, shape, dim, False) * 1.5).to(dtype)
    state["tables"] = tables.int()
    state["lengths"] = torch.tensor(lengths, dtype=torch.int32, device=device)
    return state


# -- plain forms -------------------------------------------------------------------------
def _plain_plan(s):
    page, rows = s["case"]["page"], s["rows"]
    lengths, new, tables, free, count = (s[k] for k in ("lengths", "new", "tables", "free", "count"))
    device, width = tables.device, tables.shape[1]
    at = torch.arange(width, device=device)
    if s["ended"] is not None:  # pages of ended requests go back on the stack, in order
        gone = torch.where(s["ended"], (lengths + page - 1) // page, 0)
        to = (count + gone.cumsum(0) - gone)[:, None] + at
        to = torch.where(at < gone[:, None], to, free.numel())
        free = torch.cat([free, free.new_zeros(1)]).scatter_(0, to.flatten(), tables.flatten())[:-1]
        count = (count + gone.sum()).int()
        lengths = torch.where(s["ended"], 0, lengths)
    ends = new.cumsum(0)
    held = (lengths + page - 1) // page
    after = (lengths + new + page - 1) // page
    fits = (after <= width) & (ends <= rows)
    need = torch.where(fits, after - held, 0)
    taken = need.cumsum(0)
    granted = fits & ((need == 0) | (taken <= count))
    top = torch.where(granted & (need > 0), taken, 0).amax()
    place = count - 1 - (taken - need)[:, None] - (at - held[:, None])
    fresh = granted[:, None] & (at >= held[:, None]) & (at < after[:, None])
    tables = torch.where(fresh, free[place.clamp(0, free.numel() - 1)], tables)
    row = torch.arange(rows, device=device)
    request = torch.searchsorted(ends, row, right=True).clamp_max(len(new) - 1)
    real = row < ends[-1]
    position = torch.where(real, lengths[request] + row - (ends - new)[request], 0)
    slot = tables[request, (position // page).clamp_max(width - 1)] * page + position % page
    return {"tables": tables, "free": free, "count": (count - top).int(),
            "lengths": torch.where(granted, lengths + new, lengths).int(),
            "granted": torch.where(granted, new, 0).int(),
            "starts": torch.cat([ends.new_zeros(1), ends]).int(),
            "slots": torch.where(real & granted[request], slot, -1).int(), "positions": position.int()}


def _plain_append(codes, scale, x, slots):
    """In place: rows x [n, heads, dim] (fp32) into the pool."""
    page = codes.shape[2]
    where, offset = (slots // page).long(), (slots % page).long()
    magnitude = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(2)
    index = where[:, None].expand_as(magnitude)
    amax = torch.zeros_like(scale).scatter_reduce_(0, index, magnitude, "amax")
    need = torch.ldexp(torch.ones_like(scale), _exponent(amax))
    touched = torch.zeros(scale.shape[0], dtype=torch.bool, device=x.device).index_fill_(0, where, True)
    begins = torch.zeros(scale.shape[0], device=x.device).scatter_reduce_(0, where, (offset == 0).float(), "amax") > 0
    grown = torch.where(begins[:, None], need, torch.maximum(need, scale))
    grown = torch.where(touched[:, None], grown, scale)
    shrink = torch.where(begins[:, None], 1.0, scale / grown)
    codes.copy_((codes.float() * shrink[:, :, None, None]).to(codes.dtype))
    scale.copy_(grown)
    new = (x / grown[where][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(codes.dtype)
    codes.view(torch.uint8)[where, :, offset] = new.view(torch.uint8)


def _plain_read(codes, scale, slots, dtype):
    page = codes.shape[2]
    where, offset = (slots // page).long(), (slots % page).long()
    return (codes.view(torch.uint8)[where, :, offset].view(codes.dtype).float() * scale[where][:, :, None]).to(dtype)


def _rotate(x, cos, sin, positions):
    half = x.shape[2] // 2
    c, s = cos[positions.long()][:, None], sin[positions.long()][:, None]
    a, b = x[..., :half], x[..., half:]
    return torch.cat([a * c - b * s, b * c + a * s], 2)


def _plain_append_case(s):
    case = s["case"]
    if case["rope"]:
        heads, kv = case["heads"], case["kv_heads"]
        x = s["qkv"].float().view(-1, heads + 2 * kv, case["dim"])
        turned = _rotate(x[:, :heads + kv], s["cos"], s["sin"], s["positions"])
        q, k, v = turned[:, :heads].to(s["qkv"].dtype), turned[:, heads:], x[:, heads + kv:]
    else:
        q, k, v = None, s["new_k"].float(), s["new_v"].float()
    _plain_append(s["k"], s["k_scale"], k, s["slots"])
    _plain_append(s["v"], s["v_scale"], v, s["slots"])
    out = {"k": _plain_read(s["k"], s["k_scale"], s["all"], torch.bfloat16),
           "v": _plain_read(s["v"], s["v_scale"], s["all"], torch.bfloat16)}
    return out if q is None else out | {"q": q}


def _visible(lengths, tokens, keys, window, device):
    """[sequences, tokens, keys]: which key a new token sees."""
    last = lengths[:, None].long() - tokens + torch.arange(tokens, device=device)
    key = torch.arange(keys, device=device)
    seen = key <= last[..., None]
    return seen & (key > last[..., None] - window) if window else seen


def _plain_attention(s):
    case, q = s["case"], s["q"]
    n, t, heads, dim = q.shape
    kv, group = case["kv_heads"], heads // case["kv_heads"]

    def pages(name):  # [sequences, kv heads, keys, dim]
        at = s["tables"].long()
        x = s[name].view(torch.uint8)[at].view(torch.float8_e4m3fn).float() * s[name + "_scale"][at][..., None, None]
        return x.transpose(1, 2).reshape(n, kv, -1, dim)

    rows = q.float().view(n, t, kv, group, dim).transpose(1, 2).reshape(n, kv, t * group, dim)
    scores = rows @ pages("k").transpose(2, 3) / math.sqrt(dim)
    seen = _visible(s["lengths"], t, scores.shape[3], case["window"], q.device)
    seen = seen[:, None].repeat_interleave(group, 2)
    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(3, keepdim=True)
    p = (scores - torch.where(top == -math.inf, 0.0, top)).exp()
    total = p.sum(3, keepdim=True)
    out = (p @ pages("v")) / torch.where(total == 0, 1.0, total)
    return out.view(n, kv, t, group, dim).transpose(1, 2).reshape(n, t, heads, dim).to(q.dtype)


# -- the framework's own -----------------------------------------------------------------
def _own_run(s):
    from sparknet import ops

    case, op = s["case"], s["case"]["op"]
    if op == "plan":
        plan = ops.plan_pages(s["lengths"], s["new"], s["tables"], s["free"], s["count"], page_size=case["page"],
                              max_tokens=s["rows"], finished=s["ended"])
        return {"tables": s["tables"], "free": s["free"], "count": plan.free_count, "lengths": plan.lengths,
                "granted": plan.granted, "starts": plan.starts, "slots": plan.slots, "positions": plan.positions}
    cache = s["cache"]
    if op == "append":
        q = None
        if case["rope"]:
            q = ops.rope_kv_append(cache, s["qkv"], s["cos"], s["sin"], s["positions"], s["slots"])
        else:
            ops.kv_append(cache, s["new_k"], s["new_v"], s["slots"])
        k, v = ops.kv_read(cache, s["all"])
        return {"k": k, "v": v} if q is None else {"k": k, "v": v, "q": q}
    if op == "read":
        k, v = ops.kv_read(cache, s["slots"], dtype=DTYPES[case["dtype"]])
        return {"k": k, "v": v}
    return ops.paged_decode_attention(s["q"], cache, s["tables"], s["lengths"], window=case["window"])


def run(state):
    if own:
        return _own_run(state)
    op = state["case"]["op"]
    if op == "plan":
        return _plain_plan(state)
    if op == "append":
        return _plain_append_case(state)
    if op == "read":
        dtype = DTYPES[state["case"]["dtype"]]
        return {"k": _plain_read(state["k"], state["k_scale"], state["slots"], dtype),
                "v": _plain_read(state["v"], state["v_scale"], state["slots"], dtype)}
    return _plain_attention(state)


# -- from the definitions, in 64 bits ----------------------------------------------------
def _nearest_e4m3(x):
    """Doubles to the nearest e4m3 value, ties to even, saturating: steps of 2^-3 of the
    value's power of two, at least 2^-9."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(x / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(codes, scale, x, slots):
    """Doubles: (codes, scales) after rows x, page by page as the definition says."""
    page = codes.shape[2]
    codes, scale = codes.double().clone(), scale.double().clone()
    where = slots.long() // page
    order = where.tolist()
    start = 0
    while start < len(order):
        stop = start
        while stop < len(order) and order[stop] == order[start]:
            stop += 1
        p, first = order[start], int(slots[start]) % page
        rows = x[start:stop].transpose(0, 1)  # [heads, rows, dim]
        amax = rows.abs().amax((1, 2))
        need = torch.exp2(torch.ceil(torch.log2(amax / E4M3_MAX)).clamp_min(MIN_EXPONENT))
        if first:
            grown = torch.maximum(scale[p], need)
            codes[p, :, :first] = _nearest_e4m3(codes[p, :, :first] * (scale[p] / grown)[:, None, None])
        else:
            grown = need
        scale[p] = grown
        codes[p, :, first:first + stop - start] = _nearest_e4m3(rows / grown[:, None, None])
        start = stop
    return codes, scale


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    if op == "plan":
        return None  # whole numbers
    if op in ("append", "read"):
        out = {}
        pool = {"k": (s["k"], s["k_scale"]), "v": (s["v"], s["v_scale"])}
        if op == "append":
            if case["rope"]:
                heads, kv, dim = case["heads"], case["kv_heads"], case["dim"]
                x = s["qkv"].double().view(-1, heads + 2 * kv, dim)
                z = torch.complex(x[:, :heads + kv, :dim // 2], x[:, :heads + kv, dim // 2:])
                at = s["positions"].long()
                z = z * torch.complex(s["cos"].double()[at], s["sin"].double()[at])[:, None]
                turned = torch.cat([z.real, z.imag], 2)
                out["q"], k, v = turned[:, :heads], turned[:, heads:], x[:, heads + kv:]
            else:
                k, v = s["new_k"].double(), s["new_v"].double()
            pool = {"k": _exact_append(*pool["k"], k, s["slots"]), "v": _exact_append(*pool["v"], v, s["slots"])}
        slots = (s["all"] if op == "append" else s["slots"]).long()
        for name, (codes, scale) in pool.items():
            at = slots // case["page"]
            code = codes if codes.dtype == torch.float64 else codes.float()
            out[name] = code[at, :, slots % case["page"]].double() * scale.double()[at][:, :, None]
        return out
    n, t, heads, dim = s["q"].shape
    group = heads // case["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for i, length in enumerate(_lengths(case)):
        if not length:
            continue
        at = torch.arange(length, device="cuda")
        slots = s["tables"][i][at // case["page"]].long(), at % case["page"]
        seen = at <= length - t + torch.arange(t, device="cuda")[:, None]
        if case["window"]:
            seen &= at > length - t + torch.arange(t, device="cuda")[:, None] - case["window"]
        some = seen.any(1)
        for h in range(case["kv_heads"]):
            def values(name):
                codes = s[name][:, h].view(torch.uint8)[slots].view(torch.float8_e4m3fn).double()
                return codes * s[name + "_scale"][:, h].double()[slots[0]][:, None]

            q = s["q"][i, :, h * group:(h + 1) * group].double()
            scores = torch.einsum("tgd,jd->tgj", q, values("k")) * dim ** -0.5
            weights = torch.softmax(scores.masked_fill(~seen[:, None], -math.inf), -1)
            got = torch.einsum("tgj,jd->tgd", torch.where(seen[:, None], weights, 0.0), values("v"))
            out[i, :, h * group:(h + 1) * group] = torch.where(some[:, None, None], got, 0.0)
    return out

"""The paged 8-bit KV cache on the GPU: page planning, append, read and decode attention
against plain computations in 64 bits (planning against a sequential loop)."""

import math
import random

import pytest

torch = pytest.importorskip("torch")

from sparknet import ops  # noqa: E402

pytestmark = pytest.mark.gpu

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
E4M3_MAX = 448.0


# -- planning ----------------------------------------------------------------------------
def plan_by_loop(lengths, new, tables, free, count, page, rows, finished):
    """The definition of plan_pages, one request after the other, on lists."""
    width = len(tables[0])
    tables, free = [list(t) for t in tables], list(free)
    count = min(max(count, 0), len(free))
    lengths = [max(n, 0) for n in lengths]
    for r, gone in enumerate(finished or []):
        if gone:
            for i in range(min(-(-lengths[r] // page), width)):
                if count < len(free):
                    free[count] = tables[r][i]
                    count += 1
            lengths[r] = 0
    slots, positions, starts, granted = [-1] * rows, [0] * rows, [], []
    row = asked = taken = 0
    for r, n in enumerate(lengths):
        add = max(new[r], 0)
        starts.append(row)
        held, after = -(-n // page), -(-(n + add) // page)
        fits = after <= width and row + add <= rows
        before, need = asked, after - held if fits else 0
        asked += need
        ok = fits and (need == 0 or asked <= count)
        if ok:
            for i in range(need):
                tables[r][held + i] = free[count - 1 - before - i]
            if need:
                taken = asked
        for i in range(min(add, max(0, rows - row))):
            positions[row + i] = n + i
            if ok:
                slots[row + i] = tables[r][(n + i) // page] * page + (n + i) % page
        granted.append(add if ok else 0)
        lengths[r] = n + add if ok else n
        row += add
    return {"slots": slots, "positions": positions, "starts": starts + [row], "lengths": lengths, "granted": granted,
            "free_count": [count - taken], "tables": tables, "free": free}


def plan_case(seed, requests, page, width, spare, most_new, rows, with_finished):
    """Lengths up to the tables' width, distinct pages, `spare` pages on the stack."""
    rng = random.Random(seed)
    lengths = [rng.choice((0, 1, page - 1, page, page + 1, rng.randint(0, width * page))) for _ in range(requests)]
    lengths = [min(n, width * page) for n in lengths]
    new = [rng.choice((0, 1, 1, rng.randint(0, most_new))) for _ in range(requests)]
    finished = [rng.random() < 0.3 for _ in range(requests)] if with_finished else None
    held = [-(-n // page) for n in lengths]
    pages = list(range(sum(held) + spare))
    rng.shuffle(pages)
    tables = [[-7] * width for _ in range(requests)]
    for t, h in zip(tables, held):
        t[:h] = [pages.pop() for _ in range(h)]
    free = pages + [-9] * (sum(held) + 3)
    return lengths, new, tables, free, spare, page, rows, finished


def ints(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


PLANS = [dict(requests=1, page=64, width=3, spare=2, most_new=1, rows=1, with_finished=False),
         dict(requests=5, page=16, width=4, spare=3, most_new=20, rows=64, with_finished=True),
         dict(requests=33, page=32, width=5, spare=40, most_new=70, rows=1500, with_finished=True),
         dict(requests=33, page=32, width=5, spare=2, most_new=70, rows=300, with_finished=False),
         dict(requests=1024, page=16, width=9, spare=900, most_new=40, rows=12000, with_finished=True),
         dict(requests=1025, page=128, width=3, spare=5000, most_new=300, rows=90000, with_finished=False),
         dict(requests=4096, page=64, width=6, spare=1200, most_new=30, rows=30000, with_finished=True),
         dict(requests=7, page=16, width=2, spare=0, most_new=3, rows=0, with_finished=True)]


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("case", PLANS, ids=lambda c: f"{c['requests']}x{c['width']}of{c['page']}")
def test_plan_pages(device, case, in_place):
    lengths, new, tables, free, count, page, rows, finished = plan_case(11, **case)
    want = plan_by_loop(lengths, new, tables, free, count, page, rows, finished)
    t, f, n, c = ints(tables, device), ints(free, device), ints(lengths, device), ints([count], device)
    out = {"lengths_out": n, "free_count_out": c} if in_place else {}
    plan = ops.plan_pages(n, ints(new, device), t, f, c, page_size=page, max_tokens=rows,
                          finished=None if finished is None else torch.tensor(finished, device=device), **out)
    got = {**plan._asdict(), "tables": t, "free": f}
    for name, value in want.items():
        assert got[name].tolist() == value, name
    if in_place:
        assert plan.lengths.data_ptr() == n.data_ptr() and c.tolist() == want["free_count"]


def test_plan_hostile_numbers(device):
    """Negative lengths and counts, tokens that sum past 2^31, a count above the list, a
    finished length above the width: refused or clamped as the loop says, nothing outside."""
    lengths, new = [-5, 10, 2000, 0, 3], [3, 1 << 30, 1, 1 << 30, -4]
    tables, free = [[-1] * 4 for _ in range(5)], [7, 8, 9]
    tables[1][0], tables[2] = 20, [21, 22, 23, 24]
    args = (lengths, new, tables, free, 50, 16, 12, [False, False, True, False, False])
    want = plan_by_loop(*args)
    t, f = ints(tables, device), ints(free, device)
    plan = ops.plan_pages(ints(lengths, device), ints(new, device), t, f, ints([50], device), page_size=16,
                          max_tokens=12, finished=torch.tensor(args[-1], device=device))
    want["starts"] = [min(s, 2 ** 31 - 1) for s in want["starts"]]
    for name, value in want.items():
        assert {**plan._asdict(), "tables": t, "free": f}[name].tolist() == value, name


def test_page_table_never_shares_a_page(device):
    """Requests come, grow and end at random: held pages are distinct, none is free, none lost."""
    rng = random.Random(3)
    table = ops.PageTable(40, page_size=16, max_requests=6, max_pages=12, device=device)
    for _ in range(60):
        new = [rng.choice((0, 1, 1, rng.randint(1, 60))) for _ in range(6)]
        done = [rng.random() < 0.1 for _ in range(6)]
        plan = table.extend(ints(new, device), 400, torch.tensor(done, device=device))
        held = [-(-n // 16) for n in table.lengths.tolist()]
        used = [p for r, h in enumerate(held) for p in table.block_tables[r, :h].tolist()]
        free = table.free_pages[:int(table.free_count)].tolist()
        assert sorted(used + free) == list(range(40))
        real = [s for s in plan.slots.tolist() if s >= 0]
        assert len(real) == len(set(real)) == sum(plan.granted.tolist())


# -- the cache's format, in 64 bits ------------------------------------------------------
def power_scale(amax):
    """Smallest 2^e, e >= -100, with amax <= 448 * 2^e (Python numbers)."""
    e = -100
    while amax > E4M3_MAX * 2.0 ** e:
        e += 1
    return 2.0 ** e


def nearest_code(x):
    """Doubles to the nearest e4m3 value (ties to even), saturating; NaN stays."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp(2.0 ** -6, 1e30))) - 3)
    return (torch.round(x.clamp(-1e30, 1e30) / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def append_by_definition(codes, scale, x, slots):
    """Doubles on the CPU: codes [pages, heads, page, dim], scale [pages, heads], rows x in order."""
    page = codes.shape[2]
    runs, last = [], None
    for r, s in enumerate(slots):
        if not 0 <= s < codes.shape[0] * page:
            last = None
            continue
        if last is not None and s == last + 1 and s % page:
            runs[-1].append(r)
        else:
            runs.append([r])
        last = s
    for run in runs:
        p, first = divmod(slots[run[0]], page)
        for h in range(codes.shape[1]):
            rows = x[run, h]
            finite = rows[torch.isfinite(rows)].abs()
            new = power_scale(float(finite.max()) if finite.numel() else 0.0)
            if first:
                new = max(new, float(scale[p, h]))
                codes[p, h, :first] = nearest_code(codes[p, h, :first] * (scale[p, h] / new))
            scale[p, h] = new
            codes[p, h, first:first + len(run)] = nearest_code(rows / new)


def filled_cache(gen, pages, heads, page, dim, device):
    """Pages with values at several magnitudes, scales powers of two."""
    c = ops.Fp8KVCache(pages, heads, page_size=page, head_dim=dim, device=device)
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        x = torch.randn(codes.shape, generator=gen, device=device) * 120
        codes.copy_(x.clamp(-E4M3_MAX, E4M3_MAX).to(codes.dtype))
        scale.copy_(torch.exp2(torch.randint(-9, -4, scale.shape, generator=gen, device=device).float()))
    return c


def as_doubles(cache, name):
    return getattr(cache, name).float().double().cpu(), getattr(cache, name + "_scale").double().cpu()


def same_codes(cache, name, codes, scale):
    assert torch.equal(getattr(cache, name + "_scale").double().cpu(), scale)
    got = getattr(cache, name).float().double().cpu()
    assert torch.equal(got.nan_to_num(nan=12345.0), codes.nan_to_num(nan=12345.0))


APPENDS = [  # pages, heads, page, dim, slots
    (3, 1, 64, 128, [64 + 5]),                                        # one token inside a page
    (3, 2, 16, 64, [16, 17, 18]),                                     # a page's beginning
    (9, 3, 16, 128, [*range(5, 16), *range(96, 112), *range(32, 45)]),  # a chunk over three pages
    (6, 8, 32, 64, [31, 64, 33 + 64 * 2, 127]),                       # decode: each its own page
    (6, 2, 128, 128, [*range(130, 256), *range(0, 128), -1, -1, *range(384, 391)]),
    (5, 1, 32, 128, [-1, 40, -3, 160, 161, 1 << 30, 70]),             # skipped rows between
    (40, 4, 16, 128, list(range(3, 600))),                            # enough rows to share blocks
]


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("case", APPENDS, ids=lambda c: f"p{c[2]}d{c[3]}h{c[1]}n{len(c[4])}")
def test_append_is_exact(device, case, dtype):
    """Codes and scales equal the definition bit for bit: old pages that must be rescaled,
    rows that are skipped, everything else untouched."""
    pages, heads, page, dim, slots = case
    gen = torch.Generator(device=device).manual_seed(5)
    c = filled_cache(gen, pages, heads, page, dim, device)
    n = len(slots)
    k, v = (torch.randn(n, heads, dim, generator=gen, device=device) * torch.exp2(
        torch.randint(-3, 7, (n, heads, 1), generator=gen, device=device).float()) for _ in range(2))
    k, v = k.to(DTYPES[dtype]), v.to(DTYPES[dtype])
    want = {name: as_doubles(c, name) for name in ("k", "v")}
    for name, x in (("k", k), ("v", v)):
        append_by_definition(*want[name], x.double().cpu(), slots)
    ops.kv_append(c, k, v, ints(slots, device))
    for name in ("k", "v"):
        same_codes(c, name, *want[name])


def test_append_strided_rows_and_odd_values(device):
    """Rows as slices of a wider tensor; infinities, NaN, zeros, huge and tiny values."""
    gen = torch.Generator(device=device).manual_seed(6)
    heads, dim, n = 3, 64, 10
    wide = torch.randn(n, 2 * heads + 1, dim + 8, generator=gen, device=device).to(torch.bfloat16)
    k, v = wide[:, :heads, 8:], wide[:, heads:2 * heads, :dim]
    k[0, 0, 3], k[1, 1, 5], k[2, 2, 7] = math.inf, -math.inf, math.nan
    k[:, 2, 9] = 3e38
    v[:, 0] = 0.0
    v[:, 1] *= 1e-34
    v[4, 2] = math.nan
    c = filled_cache(gen, 2, heads, 16, dim, device)
    want = {name: as_doubles(c, name) for name in ("k", "v")}
    slots = list(range(16, 26))
    for name, x in (("k", k), ("v", v)):
        append_by_definition(*want[name], x.double().cpu(), slots)
    ops.kv_append(c, k, v, ints(slots, device))
    for name in ("k", "v"):
        same_codes(c, name, *want[name])
    assert float(c.v_scale[1, 0]) == 2.0 ** -100


def test_append_token_by_token_keeps_the_largest_scale(device):
    """A page filled one token at a time has the scale of the page filled at once, and values
    within one more rounding of a subnormal: half a step, 2^-10 of the scale."""
    gen = torch.Generator(device=device).manual_seed(7)
    k, v = (torch.randn(32, 2, 128, generator=gen, device=device).mul(
        torch.exp2(torch.arange(32, device=device) / 4.0)[:, None, None]).to(torch.bfloat16) for _ in range(2))
    whole, steps = (ops.Fp8KVCache(2, 2, page_size=32, head_dim=128, device=device) for _ in range(2))
    slots = torch.arange(32, 64, dtype=torch.int32, device=device)
    ops.kv_append(whole, k, v, slots)
    for i in range(32):
        ops.kv_append(steps, k[i:i + 1], v[i:i + 1], slots[i:i + 1])
    assert torch.equal(whole.k_scale, steps.k_scale) and torch.equal(whole.v_scale, steps.v_scale)
    for a, b, s in ((whole.k, steps.k, whole.k_scale), (whole.v, steps.v, whole.v_scale)):
        diff = (a.float() - b.float()).abs()
        # a rounding to a multiple of 2^-9 is off by up to 2^-10, the growing scale's roundings add up to 2^-9
        assert float(diff.max()) <= 2.0 ** -9


@pytest.mark.parametrize("dtype", sorted(DTYPES))
@pytest.mark.parametrize("hq,hkv,dim,page,slots", [
    (8, 1, 128, 64, [70]), (14, 2, 64, 16, [*range(3, 40)]), (5, 5, 128, 32, [5, -1, 64, 65, 130]),
    (64, 8, 128, 64, [63 + 64 * i for i in range(20)]), (1, 1, 64, 128, [*range(0, 300)])])
def test_rope_append(device, hq, hkv, dim, page, slots, dtype):
    """q within its rounding of the rotation in 64 bits, codes within half a step (and the
    rotation's own rounding) of it, v exact; positions outside the tables are clamped."""
    gen = torch.Generator(device=device).manual_seed(8)
    n, table = len(slots), 90
    qkv = torch.randn(n, (hq + 2 * hkv) * dim, generator=gen, device=device).to(DTYPES[dtype])
    angle = torch.arange(table, device=device, dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    cos, sin = angle.cos().float(), angle.sin().float()
    at = [(7 * i) % table for i in range(n)]
    given = list(at)
    given[0], at[0] = 5000, table - 1
    if n > 1:
        given[1], at[1] = -3, 0
    c = filled_cache(gen, 24, hkv, page, dim, device)
    before = {name: as_doubles(c, name) for name in ("k", "v")}
    q = ops.rope_kv_append(c, qkv, cos, sin, ints(given, device), ints(slots, device))
    x = qkv.double().view(n, hq + 2 * hkv, dim).cpu()
    cs, sn = cos.double().cpu()[at][:, None], sin.double().cpu()[at][:, None]
    a, b = x[:, :hq + hkv, :dim // 2], x[:, :hq + hkv, dim // 2:]
    turned = torch.cat([a * cs - b * sn, b * cs + a * sn], 2)
    size = torch.cat([a.abs() + b.abs()] * 2, 2)  # bounds both products
    off = 3 * 2.0 ** -24 * size                   # two products and a sum, each rounded to fp32
    half = torch.finfo(qkv.dtype).eps / 2
    # the result's rounding, relative, and half the type's smallest step (fp16 2^-25, bf16 below)
    assert bool(((q.double().cpu() - turned[:, :hq]).abs() <= off[:, :hq] * 1.01 +
                 half * turned[:, :hq].abs() + 2.0 ** -25).all())
    append_by_definition(*before["v"], x[:, hq + hkv:], slots)
    same_codes(c, "v", *before["v"])
    append_by_definition(*before["k"], turned[:, hq:], slots)  # same scales, codes to the nearer neighbour
    assert torch.equal(c.k_scale.double().cpu(), before["k"][1])
    kept = [i for i, s in enumerate(slots) if s >= 0]
    got = c.k.float().double().cpu()[[slots[i] // page for i in kept], :, [slots[i] % page for i in kept]]
    scale = before["k"][1][[slots[i] // page for i in kept]][:, :, None]
    k = turned[kept, hq:] / scale
    step = torch.exp2(torch.floor(torch.log2(k.abs().clamp_min(2.0 ** -6))) - 3)
    # a value that the fp32 rotation moves over a power of two is off by half the larger step
    assert bool(((got - k).abs() <= step / 2 * (1 + 2.0 ** -20) + off[kept, hq:] / scale).all())


def test_rope_append_into_a_given_q(device):
    gen = torch.Generator(device=device).manual_seed(9)
    c = filled_cache(gen, 3, 2, 16, 64, device)
    wide = torch.randn(6, 8 * 64 + 16, generator=gen, device=device).to(torch.bfloat16)
    qkv = wide[:, 8:8 + 8 * 64]
    cos, sin = torch.ones(4, 32, device=device), torch.zeros(4, 32, device=device)
    q_out = torch.empty(6, 4, 64, dtype=torch.bfloat16, device=device)
    got = ops.rope_kv_append(c, qkv, cos, sin, ints([0] * 6, device), ints(range(16, 22), device), q_out)
    assert got.data_ptr() == q_out.data_ptr()
    assert torch.equal(q_out, qkv.reshape(6, 8, 64)[:, :4])  # turned by nothing


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("heads,page,dim", [(1, 16, 64), (3, 64, 128), (8, 128, 128)])
def test_read(device, heads, page, dim, dtype):
    """Exactly code * scale; slots in any order, repeated, absent (zeros)."""
    gen = torch.Generator(device=device).manual_seed(10)
    c = filled_cache(gen, 7, heads, page, dim, device)
    slots = torch.randint(0, 7 * page, (501,), generator=gen, device=device).int()
    slots[3], slots[77], slots[78], slots[79] = -1, 7 * page, 2 ** 31 - 1, -(2 ** 31)
    for at in (slots, slots[:1], slots[:0]):
        k, v = ops.kv_read(c, at, dtype=dtype)
        ok = (at >= 0) & (at < 7 * page)
        s = torch.where(ok, at, 0).long()
        for got, codes, scale in ((k, c.k, c.k_scale), (v, c.v, c.v_scale)):
            want = codes.float()[s // page, :, s % page] * scale[s // page][:, :, None]
            assert torch.equal(got, torch.where(ok[:, None, None], want, 0.0).to(dtype))
    k, v = torch.full((2, 3, heads, dim), 7.0, dtype=dtype, device=device)
    out = ops.kv_read(c, slots[:3], dtype=dtype, k_out=k, v_out=v)
    assert out[0].data_ptr() == k.data_ptr() and torch.equal(out[1], ops.kv_read(c, slots[:3], dtype=dtype)[1])


def test_read_back_of_an_append(device):
    """What comes back is within half an e4m3 step of what went in: 2^-4 of the value, or
    2^-10 of the scale for values in the subnormals."""
    gen = torch.Generator(device=device).manual_seed(12)
    c = ops.Fp8KVCache(9, 4, page_size=32, head_dim=128, device=device)
    k, v = (torch.randn(200, 4, 128, generator=gen, device=device).to(torch.bfloat16) for _ in range(2))
    slots = torch.arange(32, 232, dtype=torch.int32, device=device)
    ops.kv_append(c, k, v, slots)
    for x, y, s in zip((k, v), ops.kv_read(c, slots), (c.k_scale, c.v_scale)):
        s = s[slots.long() // 32][:, :, None]
        assert bool(((y.float() - x.float()).abs() <= torch.maximum(x.float().abs() / 16, s * 2.0 ** -10)).all())


# -- attention ---------------------------------------------------------------------------
def attention_inputs(device, lengths, tokens, hq, hkv, dim, page, dtype="bf16", seed=1, pages=None):
    """Random pages in random order; what no sequence holds is NaN (codes and scales)."""
    gen = torch.Generator(device=device).manual_seed(seed)
    held = [-(-n // page) for n in lengths]
    pages = pages or sum(held) + 2
    width = max(1, max(held))
    c = ops.Fp8KVCache(pages, hkv, page_size=page, head_dim=dim, device=device)
    order = torch.randperm(pages, generator=gen, device=device).int().tolist()
    tables = torch.full((len(lengths), width), -1, dtype=torch.int32, device=device)
    for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
        codes.view(torch.uint8).fill_(0x7F)
        scale.fill_(math.nan)
    for b, n in enumerate(lengths):
        mine = [order.pop() for _ in range(held[b])]
        if mine:
            tables[b, :len(mine)] = ints(mine, device)
        for codes, scale in ((c.k, c.k_scale), (c.v, c.v_scale)):
            for i, p in enumerate(mine):
                m = min(page, n - i * page)
                x = torch.randn(hkv, m, dim, generator=gen, device=device) * 100
                codes[p, :, :m] = x.clamp(-E4M3_MAX, E4M3_MAX).to(codes.dtype)
                scale[p] = torch.exp2(torch.randint(-9, -5, (hkv,), generator=gen, device=device).float())
    q = torch.randn(len(lengths), tokens, hq, dim, generator=gen, device=device).to(DTYPES[dtype])
    return q, c, tables, ints(lengths, device)


def attention_by_definition(q, c, tables, lengths, window=0, scale=None):
    """(out, lse, bound) in doubles.  The bound counts, relative to the weighted |v|: a softmax
    weight's rounding to fp16 (2^-11) and its exp2 (2^-21), the scores' fp32 sums over the head
    (each of dim + 4 roundings at most 2^-22 of the largest partial sum, as tensor cores may
    truncate; the difference of two scores enters the exponent), and the sums over n keys."""
    n, tokens, hq, dim = q.shape
    hkv, page = c.kv_heads, c.page_size
    group = hq // hkv
    scale = dim ** -0.5 if scale is None else scale
    out = torch.zeros(q.shape, dtype=torch.float64)
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64)
    bound = torch.zeros(q.shape, dtype=torch.float64)
    pools = {name: (getattr(c, name).float(), getattr(c, name + "_scale")) for name in ("k", "v")}
    for b in range(n):
        total = max(0, min(int(lengths[b]), tables.shape[1] * page))
        at = torch.arange(total, device=q.device)
        where = tables[b][at // page].long()
        real = (where >= 0) & (where < c.num_pages)
        at, where = at[real], where[real]
        kv = {name: (codes[where, :, at % page] * s[where][:, :, None]).double().cpu() for name, (codes, s) in pools.items()}
        for t in range(tokens):
            last = int(total) - tokens + t
            seen = at.cpu() <= last
            if window:
                seen &= at.cpu() > last - window
            if not bool(seen.any()):
                continue
            k, v = kv["k"][seen], kv["v"][seen]
            x = q[b, t].double().cpu().view(hkv, group, dim)
            s = torch.einsum("hgd,jhd->hgj", x, k) * scale
            size = torch.einsum("hgd,jhd->hgj", x.abs(), k.abs()).amax(2) * abs(scale)
            w = torch.softmax(s, 2)
            out[b, t] = torch.einsum("hgj,jhd->hgd", w, v).reshape(hq, dim)
            lse[b, t] = torch.logsumexp(s, 2).reshape(hq)
            keys = k.shape[0]
            rel = 2.0 ** -11 + 2.0 ** -21 + 2 * (dim + 4) * 2.0 ** -22 * size + 2 * (keys + 8) * 2.0 ** -23
            spread = torch.einsum("hgj,jhd->hgd", w, v.abs())
            bound[b, t] = (rel[..., None] * spread).reshape(hq, dim)
    half = torch.finfo(q.dtype).eps / 2
    return out, lse, bound + half * (out.abs() + bound) + 2.0 ** -25


def check_attention(q, c, tables, lengths, window=0, scale=None):
    out, lse = ops.paged_decode_attention(q, c, tables, lengths, window=window, scale=scale, return_lse=True)
    again = ops.paged_decode_attention(q, c, tables, lengths, window=window, scale=scale)
    assert torch.equal(out, again)
    want, want_lse, bound = attention_by_definition(q, c, tables, lengths, window, scale)
    off = (out.double().cpu() - want).abs()
    assert bool((off <= bound).all()), float((off / bound).max())
    empty = torch.isinf(want_lse)
    got = lse.double().cpu()
    assert torch.equal(torch.isinf(got) & (got < 0), empty)
    assert bool((out.cpu()[empty] == 0).all())
    # lse: the score's sums (the bound's second part over |v|) and log2's and the products' roundings
    keys, dim = tables.shape[1] * c.page_size, q.shape[3]
    tol = 1e-4 + want_lse[~empty].abs() * 2.0 ** -20 + keys * 2.0 ** -23 + dim * 2.0 ** -14
    assert bool(((got - want_lse)[~empty].abs() <= tol).all())
    return out


ATTENTIONS = [  # lengths, tokens, hq, hkv, dim, page, dtype
    ([1], 1, 1, 1, 128, 64, "bf16"),
    ([1], 1, 8, 1, 64, 16, "fp16"),
    ([31, 32, 33], 1, 8, 2, 128, 16, "bf16"),
    ([500], 1, 64, 8, 128, 64, "bf16"),
    ([0, 127, 128, 0, 129, 1], 1, 8, 1, 128, 128, "fp16"),
    ([1000, 17, 0, 640], 1, 14, 2, 64, 32, "bf16"),                   # 7 query heads to a KV head
    ([2049, 63], 1, 32, 2, 128, 64, "bf16"),                          # 16 to one
    ([700, 5, 90], 3, 24, 8, 128, 32, "bf16"),                        # drafted tokens
    ([257, 2, 0, 4], 4, 8, 1, 64, 16, "fp16"),                        # 32 rows, sequences shorter than the draft
    ([300, 900], 8, 16, 2, 128, 64, "bf16"),                          # 64 rows
    ([100, 33], 17, 16, 1, 128, 16, "fp16"),                          # 272 rows
    ([45, 8], 5, 3, 3, 64, 32, "bf16"),                               # multi-head, odd counts
    ([20000, 3], 1, 8, 1, 128, 64, "bf16"),                           # few rows, long
    ([5003], 2, 16, 2, 64, 16, "fp16"),
    ([700 + 13 * i for i in range(40)], 1, 16, 4, 128, 64, "bf16"),   # more pairs than one wave takes
]


@pytest.mark.parametrize("case", ATTENTIONS, ids=lambda c: f"b{len(c[0])}t{c[1]}h{c[2]}-{c[3]}d{c[4]}p{c[5]}n{max(c[0])}")
def test_paged_attention(device, case):
    check_attention(*attention_inputs(device, *case))


@pytest.mark.parametrize("window", [1, 2, 31, 33, 64, 200, 5000])
@pytest.mark.parametrize("tokens", [1, 3])
def test_paged_attention_window(device, window, tokens):
    check_attention(*attention_inputs(device, [900, 64, 0, 2, 33], tokens, 8, 2, 128, 32), window=window)


def test_paged_attention_small_inputs_take_a_batch_dim_of_three(device):
    """q [B, heads, D] is T = 1; out keeps the shape; a given out is used."""
    q, c, tables, lengths = attention_inputs(device, [70, 3], 1, 4, 2, 64, 16)
    out = ops.paged_decode_attention(q, c, tables, lengths)
    flat = ops.paged_decode_attention(q[:, 0], c, tables, lengths, out=torch.empty_like(q[:, 0].contiguous()))
    assert flat.shape == (2, 4, 64) and torch.equal(flat, out[:, 0])
    assert ops.paged_decode_attention(q[:0], c, tables[:0], lengths[:0]).shape == (0, 1, 4, 64)


def test_paged_attention_strides(device):
    """q, tables as slices of wider tensors."""
    q, c, tables, lengths = attention_inputs(device, [700, 90, 41], 2, 8, 2, 128, 32)
    wide = torch.randn(3, 3, 11, 136, device=device).to(q.dtype)
    wide[:, 1:, 2:10, :128] = q
    broad = torch.full((3, tables.shape[1] + 5), 10 ** 6, dtype=torch.int32, device=device)
    broad[:, 2:2 + tables.shape[1]] = tables
    got = ops.paged_decode_attention(wide[:, 1:, 2:10, :128], c, broad[:, 2:2 + tables.shape[1]], lengths)
    assert torch.equal(got, ops.paged_decode_attention(q, c, tables, lengths))


def test_paged_attention_scales_and_scores_far_apart(device):
    """Scores of hundreds, pages whose scales differ by 2^40, large and tiny queries."""
    q, c, tables, lengths = attention_inputs(device, [800, 300], 1, 8, 1, 128, 16, seed=4)
    some = torch.isfinite(c.v_scale)
    c.v_scale[some] = torch.exp2(torch.arange(int(some.sum()), device=device) % 9 * 5.0 - 40)
    q[0, 0, :4] *= 60
    q[0, 0, 4:] *= 1e-6
    check_attention(q, c, tables, lengths)
    check_attention(q, c, tables, lengths, scale=-1.5)
    check_attention(q, c, tables, lengths, scale=0.0)


def test_paged_attention_many_weights_below_the_largest(device):
    """One key far above 20000 alike ones whose weights, 2^-16 of the largest, add up to a
    third of its weight: none may vanish."""
    dim, n = 64, 20000
    c = ops.Fp8KVCache(313, 1, page_size=64, head_dim=dim, device=device)
    c.k[0, 0, 0, 0] = 1.0
    c.v.copy_(torch.ones_like(c.v, dtype=torch.float32).to(c.v.dtype))
    c.v[0, 0, 0] = torch.full((dim,), -1.0, device=device).to(c.v.dtype)
    q = torch.zeros(1, 1, 1, dim, dtype=torch.float16, device=device)
    q[..., 0] = 16 * math.log(2.0) * 8  # score 16 ln 2 at dim^-0.5 = 1/8
    tables = torch.arange(313, dtype=torch.int32, device=device)[None]
    check_attention(q, c, tables, ints([n], device))


def test_paged_attention_nan_stays_in_its_rows(device):
    """NaN and infinity in one head's query, in one sequence's keys, and behind the window or
    the causal edge of drafted tokens: other rows are what they were."""
    q, c, tables, lengths = attention_inputs(device, [200, 150], 2, 8, 2, 128, 16)
    clean = ops.paged_decode_attention(q, c, tables, lengths)
    bad = q.clone()
    bad[0, 0, 1, 5] = math.nan
    bad[1, 1, 6, 0] = math.inf
    out = ops.paged_decode_attention(bad, c, tables, lengths)
    hit = torch.zeros(out.shape[:3], dtype=torch.bool, device=device)
    hit[0, 0, 1] = hit[1, 1, 6] = True
    assert torch.equal(out[~hit], clean[~hit]) and bool(out[hit].isnan().all())
    page, place = int(tables[0, 199 // 16]), 199 % 16  # the newest key: only the newest token sees it
    for pool in (c.k, c.v):
        kept = pool.view(torch.uint8)[page, 0, place].clone()
        pool.view(torch.uint8)[page, 0, place, 3] = 0x7F
        out = ops.paged_decode_attention(q, c, tables, lengths)
        assert bool(out[0, 1, :4].isnan().any(-1).all())
        assert torch.equal(out[0, 0], clean[0, 0]) and torch.equal(out[1], clean[1])
        assert torch.equal(out[0, 1, 4:], clean[0, 1, 4:])
        pool.view(torch.uint8)[page, 0, place] = kept
    windowed = ops.paged_decode_attention(q, c, tables, lengths, window=7)
    page, place = int(tables[0, 191 // 16]), 191 % 16  # behind the window of both tokens
    for pool in (c.k, c.v):
        pool.view(torch.uint8)[page, 0, place, 3] = 0x7F
    assert torch.equal(ops.paged_decode_attention(q, c, tables, lengths, window=7), windowed)


def test_paged_attention_bad_pages_hold_no_keys(device):
    """Table entries outside the pool, and lengths above the table's width or below 0."""
    q, c, tables, lengths = attention_inputs(device, [200, 100, 64, 30], 1, 8, 2, 64, 16)
    tables[0, 3], tables[0, 7], tables[1, 0], tables[2, :4] = -1, c.num_pages, 2 ** 31 - 1, -(2 ** 31)
    tables[0, 12] = tables[0, 11]
    lengths = ints([208 + 5000, 100, 64, -9], device)
    last = int(tables[0, 11])
    for pool in (c.k, c.v):  # the page that the clamped length now ends in
        pool[last] = torch.ones(pool[last].shape, device=device).to(pool.dtype)
    check_attention(q, c, tables, lengths)


def test_paged_attention_streams_and_threads_of_calls(device):
    """Calls at once on two streams, and on the default one, do not disturb each other."""
    args = [attention_inputs(device, [3000 + i, 40], 1, 16, 2, 128, 64, seed=i) for i in range(3)]
    want = [ops.paged_decode_attention(*a) for a in args]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(device), torch.cuda.Stream(device), torch.cuda.default_stream(device)]
    got = [[] for _ in args]
    for _ in range(20):
        for s, a, g in zip(streams, args, got):
            with torch.cuda.stream(s):
                g.append(ops.paged_decode_attention(*a))
    torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, x) for x in g)


def test_step_of_the_whole_path_and_its_graphs(device):
    """Plan, append with RoPE, attend: a prompt and decode steps, eager and as two captured
    graphs replayed in turn, equal; against attention over what the cache holds."""
    hq, hkv, dim, page, n = 8, 2, 128, 16, 3
    gen = torch.Generator(device=device).manual_seed(21)
    angle = torch.arange(256, device=device, dtype=torch.float64)[:, None] * 1e4 ** (
        -torch.arange(0, dim, 2, device=device, dtype=torch.float64) / dim)
    cos, sin = angle.cos().float(), angle.sin().float()
    prompt = [40, 16, 1]
    first = torch.randn(64, (hq + 2 * hkv) * dim, generator=gen, device=device).to(torch.bfloat16)
    steps = torch.randn(6, n, (hq + 2 * hkv) * dim, generator=gen, device=device).to(torch.bfloat16)
    ones = torch.ones(n, dtype=torch.int32, device=device)

    def begin():
        table = ops.PageTable(24, page_size=page, max_requests=n, max_pages=6, device=device)
        caches = [ops.Fp8KVCache(24, hkv, page_size=page, head_dim=dim, device=device) for _ in range(2)]
        plan = table.extend(ints(prompt, device), 64)
        for c in caches:
            ops.rope_kv_append(c, first, cos, sin, plan.positions, plan.slots)
        return table, caches

    def step(table, caches, x):
        plan = table.extend(ones, n)
        outs = []
        for c in caches:
            q = ops.rope_kv_append(c, x, cos, sin, plan.positions, plan.slots)
            outs.append(ops.paged_decode_attention(q, c, table.block_tables, table.lengths))
            x = x + 1
        return outs, q

    table, caches = begin()
    eager = []
    for x in steps:
        outs, q = step(table, caches, x)
        eager.append([o.clone() for o in outs])
    check_attention(q[:, None], caches[1], table.block_tables, table.lengths)
    assert table.lengths.tolist() == [p + 6 for p in prompt]

    graphs = []
    for _ in range(2):
        table, caches = begin()
        x = steps[0].clone()
        side = torch.cuda.Stream(device)
        side.wait_stream(torch.cuda.current_stream(device))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            outs, _ = step(table, caches, x)
        graphs.append((graph, x, outs, table, caches))  # a graph's tensors are kept as long as it
    for i, s in enumerate(steps):
        for graph, x, *_ in graphs:
            x.copy_(s)
            graph.replay()
        for _, _, outs, *_ in graphs:
            assert all(torch.equal(a, b) for a, b in zip(outs, eager[i]))
    assert graphs[0][3].lengths.tolist() == [p + 6 for p in prompt]


def test_attention_offsets_past_32_bits(device):
    """A pool of more than 2^32 bytes: its last pages."""
    pages = (1 << 32) // (8 * 128 * 128) + 9
    c = ops.Fp8KVCache(pages, 8, page_size=128, head_dim=128, device=device)
    gen = torch.Generator(device=device).manual_seed(2)
    k, v = (torch.randn(300, 8, 128, generator=gen, device=device).to(torch.bfloat16) for _ in range(2))
    tables = torch.arange(pages - 3, pages, dtype=torch.int32, device=device)[None]
    slots = torch.arange(300, dtype=torch.int32, device=device) + (pages - 3) * 128
    ops.kv_append(c, k, v, slots)
    got = ops.kv_read(c, slots, dtype=torch.float32)
    assert float((got[0] - k.float()).abs().max()) <= float(k.float().abs().max()) / 16
    small = ops.Fp8KVCache.from_tensors(c.k[-3:], c.v[-3:], c.k_scale[-3:], c.v_scale[-3:])
    q = torch.randn(1, 1, 16, 128, generator=gen, device=device).to(torch.bfloat16)
    a = check_attention(q, small, torch.arange(3, dtype=torch.int32, device=device)[None], ints([300], device))
    assert torch.equal(a, ops.paged_decode_attention(q, c, tables, ints([300], device)))


# -- the model that decodes over it ------------------------------------------------------
@pytest.mark.parametrize("gemm", ["sparknet", "cublas"])
def test_tiny_model_over_the_fp8_cache(device, gemm):
    """A decode step's last attention against the definition over what the last layer's cache
    holds; graph replay decodes the eager tokens; pages run over a border (page 16)."""
    from sparknet.models.llama import LlamaConfig, TPLlama

    def model():
        m = TPLlama(LlamaConfig.tiny(layers=2), rank=0, world=1, device=device, batch=3, max_len=48, gemm=gemm,
                    kv_cache="fp8", page_size=16)
        m.fill_prompt_cache(14)
        m.tokens.copy_(torch.tensor([1, 2, 3], device=device))
        return m

    m, eager = model(), []
    for _ in range(5):
        m.step_kernels()
        eager.append(m.tokens.tolist())
    assert m.table.lengths.tolist() == [19] * 3 and int(m.table.free_count) == 9 - 3 * 2
    want, _, bound = attention_by_definition(m.q[:, None], m.layers[-1]["cache"], m.table.block_tables,
                                             m.table.lengths)
    assert bool(((m.attn.double().cpu()[:, None] - want).abs() <= bound).all())
    g, replayed = model(), []
    g.capture()
    for _ in range(5):
        g.replay()
        replayed.append(g.tokens.tolist())
    assert replayed == eager
    assert g.launches_per_step() > 0
    g.layers[0]["cache"].check()
    for _ in range(40):  # past max_len: tokens without slots, nothing grows
        g.replay()
    assert g.table.lengths.tolist() == [48] * 3
    g.release()


def test_tiny_model_refuses(device):
    from sparknet.models.llama import LlamaConfig, TPLlama

    for bad in ({"kv_cache": "int8"}, {"kv_cache": "fp8", "attention": "simt"}, {"kv_cache": "fp8", "page_size": 24}):
        with pytest.raises(ValueError):
            TPLlama(LlamaConfig.tiny(layers=1), rank=0, world=1, device=device, batch=1, max_len=48, **bad)

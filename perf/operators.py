"""What is measured of the operators that serve attention from an 8-bit paged cache.

Three operators make one serving step after the projections:

* ``plan``   -- paged_plan: from the requests' lengths, the pages that their new
  tokens need (taken from a free list), the block table, the slot of each token;
* ``append`` -- paged_append: the step's keys and values into the cache, as 8-bit
  floats (e4m3) with one power-of-two scale for each page and head;
* ``attend`` -- paged_attention: the step's queries over that cache.

``run`` computes them in plain torch operations where ``own`` is false and through
``pmkl_function`` where it is true, on the same state.

Layout: a cache is [pages, kv_heads, block, hidden] (its memory may hold the rows of a
page outside its heads: ``rows_first``), its scales are [pages, kv_heads]; queries, new
keys and values are packed by request, [tokens, heads, hidden].
"""
import math
import random

import torch

own = False

DTYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
E4M3_MAX = 448.0
#: Scales are 2^-64 to 2^64.
SCALE_EXP = 64


# ---------------------------------------------------------------- cases
def listed():
    return [
        # One token for each of a small batch of requests: the call that every decode step makes, bound by latency.
        {"name": "plan-step-16", "op": "plan", "batch": 16, "block": 16, "min_len": 0, "max_len": 4096,
         "min_new": 1, "max_new": 1, "lens_seed": 1, "spare": 64, "pad": 0},
        # Prompts, chunks and single tokens mixed in one large batch, and a slot map with room to spare (a captured graph's).
        {"name": "plan-mixed-1024", "op": "plan", "batch": 1024, "block": 16, "min_len": 0, "max_len": 8192,
         "min_new": 0, "max_new": 129, "lens_seed": 2, "spare": 100, "pad": 4096},
        # The keys and values of one decode step: a row a request, most into pages that hold rows already.
        {"name": "append-step-16", "op": "append", "batch": 16, "kv_heads": 32, "hidden": 128, "block": 16,
         "dtype": "bfloat16", "min_len": 0, "max_len": 255, "min_new": 1, "max_new": 1, "lens_seed": 3, "rows_first": False},
        # Ragged chunks of prompts behind cached tokens, head size 64.
        {"name": "append-chunks-f16", "op": "append", "batch": 8, "kv_heads": 16, "hidden": 64, "block": 32,
         "dtype": "float16", "min_len": 0, "max_len": 1000, "min_new": 1, "max_new": 1024, "lens_seed": 4, "rows_first": True},
        # Whole prompts: 16 requests of 4096 tokens, 32 heads of 128.
        {"name": "append-prompts-bf16", "op": "append", "batch": 16, "kv_heads": 32, "hidden": 128, "block": 16,
         "dtype": "bfloat16", "min_len": 0, "max_len": 0, "min_new": 4096, "max_new": 4096, "lens_seed": 5, "rows_first": False},
        # The smallest: two requests of 128 tokens, 4 heads of 64, fp32.
        {"name": "attend-f32-tiny", "op": "attend", "batch": 2, "heads": 4, "kv_heads": 4, "hidden": 64, "block": 16,
         "dtype": "float32", "min_len": 128, "max_len": 128, "min_q": 1, "max_q": 1, "lens_seed": 6, "rows_first": False},
        # A decode step of a small model.
        {"name": "attend-f16-1k", "op": "attend", "batch": 8, "heads": 16, "kv_heads": 16, "hidden": 64, "block": 16,
         "dtype": "float16", "min_len": 1024, "max_len": 1024, "min_q": 1, "max_q": 1, "lens_seed": 7, "rows_first": False},
        # A decode step with as many K/V heads as query heads.
        {"name": "attend-mha-4k", "op": "attend", "batch": 16, "heads": 32, "kv_heads": 32, "hidden": 128, "block": 16,
         "dtype": "bfloat16", "min_len": 4096, "max_len": 4096, "min_q": 1, "max_q": 1, "lens_seed": 8, "rows_first": False},
        # A decode step of many requests of very different lengths, grouped heads.
        {"name": "attend-ragged-64", "op": "attend", "batch": 64, "heads": 32, "kv_heads": 8, "hidden": 128, "block": 64,
         "dtype": "bfloat16", "min_len": 1, "max_len": 16384, "min_q": 1, "max_q": 1, "lens_seed": 9, "rows_first": True},
        # One request with a long context: the work has to be split along the cache.
        {"name": "attend-long-1", "op": "attend", "batch": 1, "heads": 32, "kv_heads": 8, "hidden": 128, "block": 128,
         "dtype": "bfloat16", "min_len": 131071, "max_len": 131071, "min_q": 1, "max_q": 1, "lens_seed": 10, "rows_first": False},
        # Drafted tokens checked: a few query rows a request, eight query heads a K/V head.
        {"name": "attend-verify-16", "op": "attend", "batch": 16, "heads": 32, "kv_heads": 4, "hidden": 128, "block": 32,
         "dtype": "float16", "min_len": 500, "max_len": 8192, "min_q": 1, "max_q": 5, "lens_seed": 11, "rows_first": True},
        # Chunks of long prompts over what is cached of them: bound by arithmetic.
        {"name": "attend-chunk-1024", "op": "attend", "batch": 4, "heads": 32, "kv_heads": 8, "hidden": 128, "block": 16,
         "dtype": "bfloat16", "min_len": 3001, "max_len": 8192, "min_q": 700, "max_q": 1024, "lens_seed": 12, "rows_first": False},
    ]


def _log(rng, lo, hi):
    """A whole number of lo to hi, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["plan", "append", "attend", "attend", "attend"])
    lens_seed = rng.randrange(1 << 30)
    block = rng.choice([16, 16, 32, 64, 128])
    if op == "plan":
        new = _log(rng, 1, 512)
        return {"op": op, "batch": _log(rng, 1, 1024), "block": block, "min_len": 0, "max_len": _log(rng, 1, 8192),
                "min_new": rng.choice([0, 1, new]), "max_new": new, "lens_seed": lens_seed,
                "spare": rng.choice([0, 3, 1000]), "pad": rng.choice([0, 17, 1000])}
    hidden = rng.choice([64, 128, 128])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 8, 16, 32])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if op == "append":
        batch = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, min(4096, (1 << 27) // (batch * kv_heads * hidden))))
        return {"op": op, "batch": batch, "kv_heads": kv_heads, "hidden": hidden, "block": block, "dtype": dtype,
                "min_len": 0, "max_len": _log(rng, 1, 1000), "min_new": rng.choice([1, 1, new]), "max_new": new,
                "lens_seed": lens_seed, "rows_first": rng.random() < 0.5}
    group = rng.choice([1, 1, 2, 3, 4, 4, 7, 8])
    heads = kv_heads * group
    shape = rng.choice(["step", "step", "few", "chunk"])
    if shape == "chunk":
        batch = _log(rng, 1, 4)
        q = _log(rng, 16, 1024)
        longest = _log(rng, q, max(q, min(8192, (1 << 30) // (batch * heads * q))))
    else:
        batch = _log(rng, 1, 128)
        q = 1 if shape == "step" else rng.randrange(2, 9)
        longest = max(q, _log(rng, 16, max(16, min(131072, (1 << 29) // (batch * kv_heads * hidden), (1 << 31) // (batch * heads * q * 32)))))
    return {"op": op, "batch": batch, "heads": heads, "kv_heads": kv_heads, "hidden": hidden, "block": block, "dtype": dtype,
            "min_len": rng.choice([q, max(q, longest // 2), longest]), "max_len": longest, "min_q": rng.choice([1, q]), "max_q": q,
            "lens_seed": lens_seed, "rows_first": rng.random() < 0.5}


# ---------------------------------------------------------------- lengths (of the case, not of the seed)
def _spread(r, lo, hi):
    return lo if hi <= lo else r.randint(lo, hi)


def _lengths(case):
    """(tokens in the cache, new tokens) of each request; for ``attend`` the first counts the second's."""
    r = random.Random(case["lens_seed"])
    lens, new = [], []
    for _ in range(case["batch"]):
        if case["op"] == "attend":
            n = _spread(r, case["min_q"], case["max_q"])
            lens.append(max(n, _spread(r, case["min_len"], case["max_len"])))
        else:
            n = _spread(r, case["min_new"], case["max_new"])
            lens.append(_spread(r, case["min_len"], case["max_len"]))
        new.append(n)
    return lens, new


def _pages(n, block):
    return -(-n // block)


# ---------------------------------------------------------------- work
def work(case):
    lens, new = _lengths(case)
    b, block = case["batch"], case["block"]
    if case["op"] == "plan":
        tokens = sum(new) + case["pad"]
        taken = sum(_pages(c + n, block) - _pages(c, block) for c, n in zip(lens, new))
        last = sum(1 for c, n in zip(lens, new) if n and c % block)  # the page that a request goes on in is looked up
        return {"bytes": 8 * b + 4 * last + 4 + 8 * taken + 8 * tokens + 4 * b + 4 * (b + 1) + 4 * b + 4, "flops": 0}
    size = DTYPES[case["dtype"]].itemsize
    row = case["kv_heads"] * case["hidden"]
    if case["op"] == "append":
        touched = sum(_pages(c + n, block) - c // block for c, n in zip(lens, new) if n)
        return {"bytes": sum(new) * (2 * row * size + 2 * row + 8) + touched * case["kv_heads"] * 2 * 4, "flops": 0}
    heads, hidden = case["heads"], case["hidden"]
    pages = sum(_pages(c, block) for c in lens)
    seen = sum(n * (c - n) + n * (n + 1) // 2 for c, n in zip(lens, new))
    return {"bytes": sum(lens) * 2 * row + pages * (8 * case["kv_heads"] + 4) + sum(new) * heads * (2 * hidden * size + 4) + 8 * b,
            "flops": 4 * seen * heads * hidden}


# ---------------------------------------------------------------- inputs
def _ints(values, dtype=torch.int32):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _table(lens, block, width, gen, more=0):
    """A block table over a shuffled pool of pages ([batch, width], -1 where a request has no page), and the pages that no request has."""
    per = torch.tensor([_pages(n, block) for n in lens])
    held = int(per.sum())
    pool = torch.randperm(held + more, generator=gen, device="cuda").to(torch.int32)
    at = torch.arange(width)[None, :] < per[:, None]
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device="cuda")
    table[at.cuda()] = pool[:held]
    return table, pool[held:]


def _values(shape, gen):
    """Normal values whose rows differ in size, as a model's keys and values do."""
    x = torch.randn(shape, generator=gen, device="cuda")
    return x.mul_(torch.exp(torch.randn(shape[:-1] + (1,), generator=gen, device="cuda").mul_(0.5)))


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s, from 2^-64 to 2^64."""
    fraction, exponent = torch.frexp(amax)  # fraction of [0.5, 1); 448 is 0.875 * 2^9
    e = torch.where(fraction > 0.875, exponent - 8, exponent - 9).clamp(-SCALE_EXP, SCALE_EXP)
    return torch.exp2(torch.where(amax > 0, e, -SCALE_EXP).float())


def _cache(case, pages, gen):
    """A cache with every row of every page written, and its scales."""
    heads, block, hidden = case["kv_heads"], case["block"], case["hidden"]
    cache = torch.empty((pages, block, heads, hidden) if case["rows_first"] else (pages, heads, block, hidden),
                        dtype=torch.float8_e4m3fn, device="cuda")
    cache = cache.transpose(1, 2) if case["rows_first"] else cache
    scale = torch.empty(pages, heads, device="cuda")
    step = max(1, (1 << 27) // (heads * block * hidden))
    for p in range(0, pages, step):
        x = _values((min(step, pages - p), heads, block, hidden), gen)
        scale[p:p + step] = s = _scale_of(x.abs().amax((2, 3)))
        cache[p:p + step] = (x / s[:, :, None, None]).to(torch.float8_e4m3fn)
    return cache, scale


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    lens, new = _lengths(case)
    block = case["block"]
    state = {"op": case["op"], "block": block}
    if case["op"] == "plan":
        # The pool also holds what the new tokens need, and some pages more.
        need = sum(_pages(c + n, block) - _pages(c, block) for c, n in zip(lens, new))
        width = max(1, max(_pages(c + n, block) for c, n in zip(lens, new)))
        table, free = _table(lens, block, width, gen, need + case["spare"])
        state |= {"cached_lens": _ints(lens), "new_lens": _ints(new), "block_table": table, "free_blocks": free,
                  "free_count": _ints([free.numel()]), "max_tokens": sum(new) + case["pad"]}
        return state
    dtype = DTYPES[case["dtype"]]
    if case["op"] == "append":
        total = [c + n for c, n in zip(lens, new)]
        width = max(1, max(_pages(t, block) for t in total))
        table, _ = _table(total, block, width, gen)
        pages = max(1, sum(_pages(t, block) for t in total))
        ends = torch.tensor(new).cumsum(0)
        at = torch.arange(int(ends[-1]))
        owner = torch.searchsorted(ends, at, right=True)
        place = at - (ends - torch.tensor(new))[owner] + torch.tensor(lens)[owner]
        page = table.cpu()[owner, place // block].long()
        shape = (at.numel(), case["kv_heads"], case["hidden"])
        state["k_cache"], state["k_scale"] = _cache(case, pages, gen)
        state["v_cache"], state["v_scale"] = _cache(case, pages, gen)
        state |= {"k": _values(shape, gen).to(dtype), "v": _values(shape, gen).to(dtype), "slot_map": (page * block + place % block).cuda()}
        return state
    width = max(1, max(_pages(c, block) for c in lens))
    table, _ = _table(lens, block, width, gen)
    pages = max(1, sum(_pages(c, block) for c in lens))
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    state["k_cache"], state["k_scale"] = _cache(case, pages, gen)
    state["v_cache"], state["v_scale"] = _cache(case, pages, gen)
    state |= {"q": torch.randn(starts[-1], case["heads"], case["hidden"], generator=gen, device="cuda").to(dtype),
              "block_table": table, "seq_lens": _ints(lens), "query_starts": _ints(starts), "max_query_len": max(new)}
    return state


# ---------------------------------------------------------------- one pass
def run(state):
    if own:
        return _run_own(state)
    return {"plan": _plan, "append": _append, "attend": _attend}[state["op"]](state)


def _run_own(s):
    import pmkl_b200  # noqa: F401  (puts the binding on the path)
    from pmkl_function import paged_append, paged_attention, paged_plan

    if s["op"] == "plan":
        seq_lens, query_starts, slot_map, free_count, status = paged_plan(
            s["cached_lens"], s["new_lens"], s["block_table"], s["free_blocks"], s["free_count"], s["block"], s["max_tokens"])
        return [seq_lens, query_starts, slot_map, free_count, status, s["block_table"]]
    if s["op"] == "append":
        paged_append(s["k"], s["v"], s["slot_map"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"])
        return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]
    out, lse = paged_attention(s["q"], s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"], s["block_table"], s["seq_lens"],
                               s["query_starts"], s["max_query_len"])
    return [out, lse]


# ---------------------------------------------------------------- plain forms
def _plan(s):
    block, table, count = s["block"], s["block_table"], s["free_count"].long()
    width, tokens = table.shape[1], s["max_tokens"]
    cached, new = s["cached_lens"].long().clamp_min(0), s["new_lens"].long().clamp_min(0)
    ends = new.cumsum(0)
    starts, total = ends - new, cached + new
    first, last = (cached + block - 1) // block, (total + block - 1) // block
    past, wide = ends > tokens, last > width
    need = torch.where(past | wide, 0, last - first)
    taken = need.cumsum(0)
    short = (need > 0) & (taken > count)
    ok = ~(past | wide | short)
    status = torch.where(past, 3, torch.where(wide, 2, torch.where(short, 1, 0))).to(torch.int32)
    left = count - torch.where(ok & (need > 0), taken, 0).max()
    # the pages: the i-th that is taken is the i-th from the end of the free list
    column = torch.arange(width, device=table.device)[None, :]
    fresh = ok[:, None] & (column >= first[:, None]) & (column < last[:, None])
    order = (count - 1 - (taken - need)[:, None] - (column - first[:, None])).clamp(0, max(0, s["free_blocks"].numel() - 1))
    if s["free_blocks"].numel():
        table.copy_(torch.where(fresh, s["free_blocks"][order], table))
    # the slots
    at = torch.arange(tokens, device=table.device)
    owner = torch.searchsorted(ends, at, right=True)
    real = owner < ends.numel()
    owner = owner.clamp_max(ends.numel() - 1)
    place = cached[owner] + at - starts[owner]
    real &= ok[owner]
    page = table[owner, torch.where(real, place // block, 0)].long()
    slots = torch.where(real, page * block + place % block, -1)
    query_starts = torch.cat([ends.new_zeros(1), ends]).to(torch.int32)
    return [torch.where(ok, total, cached).to(torch.int32), query_starts, slots, left.to(torch.int32), status, table]


def _append_one(x, slots, cache, scale):
    block = cache.shape[2]
    x = x.float()
    page, row = slots // block, slots % block
    amax = torch.zeros_like(scale).index_reduce_(0, page, x.abs().amax(2), "amax", include_self=True)
    touched = torch.zeros_like(scale[:, 0]).index_fill_(0, page, 1.0)[:, None] > 0
    begun = torch.zeros_like(scale[:, 0]).index_fill_(0, page[row == 0], 1.0)[:, None] > 0  # written from its first row on: what it held is gone
    held = torch.where(begun, 0.0, scale)
    grown = torch.where(touched, torch.maximum(held, _scale_of(amax)), scale)
    # rows that a page holds already, where its scale grows
    lead = torch.ones_like(page, dtype=torch.bool)
    lead[1:] = page[1:] != page[:-1]
    lead &= row > 0
    there, first = page[lead], row[lead]
    old = cache[there].float()
    moved = (old * (held[there] / grown[there])[:, :, None, None]).to(cache.dtype)
    keep = torch.arange(block, device=x.device)[None, None, :, None] < first[:, None, None, None]
    cache[there] = torch.where(keep, moved.float(), old).to(cache.dtype)
    cache[page, :, row] = (x / grown[page][:, :, None]).clamp(-E4M3_MAX, E4M3_MAX).to(cache.dtype)
    scale.copy_(grown)


def _append(s):
    _append_one(s["k"], s["slot_map"], s["k_cache"], s["k_scale"])
    _append_one(s["v"], s["slot_map"], s["v_cache"], s["v_scale"])
    return [s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]]


def _gathered(cache, scale, pages):
    """[batch, kv_heads, keys, hidden] in 32 bits."""
    x = cache[pages].float().mul_(scale[pages][..., None, None])  # [batch, pages, kv_heads, block, hidden]
    b, w, h, p, d = x.shape
    return x.permute(0, 2, 1, 3, 4).reshape(b, h, w * p, d)


def _attend(s):
    q, lens, starts = s["q"], s["seq_lens"].long(), s["query_starts"].long()
    tokens, heads, hidden = q.shape
    batch, kv_heads = lens.numel(), s["k_cache"].shape[1]
    group, rows = heads // kv_heads, s["max_query_len"]
    pages = s["block_table"].long().clamp_min(0)
    keys, values = _gathered(s["k_cache"], s["k_scale"], pages), _gathered(s["v_cache"], s["v_scale"], pages)
    count = keys.shape[2]
    # queries, [batch, kv_heads, group * rows, hidden]
    news = starts[1:] - starts[:-1]
    row = torch.arange(rows, device=q.device)
    at = (starts[:-1, None] + row).clamp_max(tokens - 1)
    x = q.float()[at].view(batch, rows, kv_heads, group, hidden).permute(0, 2, 3, 1, 4).reshape(batch, kv_heads, group * rows, hidden)
    scores = torch.matmul(x, keys.transpose(2, 3)).mul_(1 / math.sqrt(hidden)).view(batch, kv_heads, group, rows, count)
    place = (lens - news)[:, None] + row  # [batch, rows]
    hidden_keys = torch.arange(count, device=q.device) > place[:, :, None]
    scores.masked_fill_(hidden_keys[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top.isinf(), 0.0, top)).exp_()
    total = scores.sum(-1, keepdim=True)
    values.masked_fill_((torch.arange(count, device=q.device) >= lens[:, None])[:, None, :, None], 0.0)
    out = torch.matmul(scores.view(batch, kv_heads, group * rows, count), values).view(batch, kv_heads, group, rows, hidden)
    out = torch.where(total > 0, out / total, 0.0)
    lse = (top + total.log())[..., 0]
    # packed again: [tokens, heads, hidden]
    token = torch.arange(tokens, device=q.device)
    owner = torch.searchsorted(starts[1:], token, right=True)
    line = token - starts[owner]
    out = out.permute(0, 3, 1, 2, 4)[owner, line].reshape(tokens, heads, hidden).to(q.dtype)
    return [out, lse.permute(0, 3, 1, 2)[owner, line].reshape(tokens, heads)]


# ---------------------------------------------------------------- 64 bits, from the definitions
def _e4m3(x):
    """The nearest e4m3 value (ties to even): 3 bits behind the leading one, exponents from -6."""
    a = x.abs()
    e = torch.floor(torch.log2(torch.where(a > 0, a, 1.0))).clamp(-6, 8)
    q = torch.exp2(e - 3)
    return (torch.round(x / q) * q).clamp(-E4M3_MAX, E4M3_MAX)


def _exact_append(x, cache, scale, table, lens, new, block):
    values, scales = cache.double(), scale.double()
    x, t = x.double(), 0
    for b, (c, n) in enumerate(zip(lens, new)):
        at = c
        while at < c + n:
            page, row = int(table[b, at // block]), at % block
            # the first page of a request may be partly filled; the whole ones behind it go at once
            many = 1 if row else max(1, (c + n - at) // block)
            pages = table[b, at // block:at // block + many].long().cuda()
            rows = min(block - row, c + n - at) if many == 1 else block
            y = x[t:t + many * rows].view(many, rows, x.shape[1], x.shape[2]).transpose(1, 2)
            amax = y.abs().amax((2, 3))
            s = torch.full_like(amax, 2.0 ** -SCALE_EXP)
            for _ in range(2 * SCALE_EXP):
                s = torch.where(E4M3_MAX * s < amax, 2 * s, s)
            if row:
                s = torch.maximum(s, scales[pages])
                values[page, :, :row] = _e4m3(values[page, :, :row] * (scales[page] / s[0])[:, None, None])
            scales[pages] = s
            values[pages, :, row:row + rows] = _e4m3(y / s[:, :, None, None])
            at, t = at + many * rows, t + many * rows
    return values, scales


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    lens, new = _lengths(case)
    block = case["block"]
    if case["op"] == "append":
        # the block table that prepare() made its slots from, by the same drawing
        total = [c + n for c, n in zip(lens, new)]
        table = _table(total, block, max(1, max(_pages(t, block) for t in total)), torch.Generator(device="cuda").manual_seed(seed))[0].cpu()
        k, ks = _exact_append(s["k"], s["k_cache"], s["k_scale"], table, lens, new, block)
        v, vs = _exact_append(s["v"], s["v_cache"], s["v_scale"], table, lens, new, block)
        return [k, v, ks, vs]
    group = case["heads"] // case["kv_heads"]
    outs, lses, t = [], [], 0
    for b, (c, n) in enumerate(zip(lens, new)):
        pages = s["block_table"][b, :_pages(c, block)].long()
        k, v = ((s[a + "_cache"][pages].double() * s[a + "_scale"][pages].double()[:, :, None, None]).transpose(1, 2).reshape(
            -1, case["kv_heads"], case["hidden"])[:c] for a in "kv")
        o = torch.empty(n, case["heads"], case["hidden"], dtype=torch.float64, device="cuda")
        lse = torch.empty(n, case["heads"], dtype=torch.float64, device="cuda")
        for h in range(case["heads"]):
            z = s["q"][t:t + n, h].double() @ k[:, h // group].T / math.sqrt(case["hidden"])
            z = z + torch.full_like(z, -math.inf).triu(c - n + 1)
            lse[:, h] = torch.logsumexp(z, 1)
            o[:, h] = torch.softmax(z, 1) @ v[:, h // group]
        outs.append(o)
        lses.append(lse)
        t += n
    return [torch.cat(outs), torch.cat(lses)]

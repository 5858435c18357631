"""Plain 64-bit implementations of the paged 8-bit cache's operators, and the
inputs and error bounds of their tests."""
from __future__ import annotations

import math

import torch

E4M3_MAX = 448.0


def plan(cached, new, table, free, count, block, max_tokens):
    """paged_plan on Python lists: (seq_lens, query_starts, slots, free left, status, table)."""
    table = [list(r) for r in table]
    width = len(table[0]) if table else 0
    seq, starts, slots, status = [], [0], [-1] * max_tokens, []
    taken, granted = 0, 0
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(0, c), max(0, n)
        begin, end = starts[-1], starts[-1] + n
        starts.append(end)
        first, last = -(-c // block), -(-(c + n) // block)
        why = 3 if end > max_tokens else 2 if last > width else 0
        need = 0 if why else last - first
        taken += need
        if not why and need and taken > count:
            why = 1
        status.append(why)
        seq.append(c if why else c + n)
        if why:
            continue
        if need:
            granted = taken
        for i in range(need):
            table[b][first + i] = free[count - 1 - (taken - need) - i]
        for i in range(n):
            slots[begin + i] = table[b][(c + i) // block] * block + (c + i) % block
    return seq, starts, slots, count - granted, status, table


def e4m3(x):
    """The nearest e4m3 value of float64 x, ties to even, saturating; NaN stays."""
    a = x.abs()
    e = torch.floor(torch.log2(torch.where((a > 0) & a.isfinite(), a, torch.ones_like(a)))).clamp(-6, 8)
    q = torch.exp2(e - 3)
    return (torch.round(x / q) * q).clamp(-E4M3_MAX, E4M3_MAX)


def scale_for(amax):
    s = 2.0 ** -64
    while E4M3_MAX * s < amax and s < 2.0 ** 64:
        s *= 2
    return s


def append(x, slots, cache, scale):
    """paged_append of one side, float64 on the CPU: cache [pages, heads, block,
    hidden] as stored values, scale [pages, heads]; returns new copies."""
    cache, scale = cache.double().clone(), scale.double().clone()
    pages, heads, block, _ = cache.shape
    t, x = 0, x.double()
    while t < len(slots):
        s = slots[t]
        if s < 0 or s >= pages * block:
            t += 1
            continue
        page, row, n = s // block, s % block, 1
        while row + n < block and t + n < len(slots) and slots[t + n] == s + n:
            n += 1
        for h in range(heads):
            y = x[t:t + n, h]
            a = y.abs()
            a = a[a.isfinite()]
            new = scale_for(float(a.max()) if a.numel() else 0.0)
            if row:
                old = float(scale[page, h])
                new = max(new, old)
                if new > old:
                    cache[page, h, :row] = e4m3(cache[page, h, :row] * (old / new))
            scale[page, h] = new
            cache[page, h, row:row + n] = e4m3(y / new)
        t += n
    return cache, scale


def attention(q, k_cache, v_cache, k_scale, v_scale, table, lens, starts, causal=True, scale=0.0):
    """paged_attention in float64 on the CPU.  Returns (out, lse, weight), weight
    = sum of p |v|, what the rounding of p is relative to; rows of no request
    give 0, -inf, 0."""
    T, H, D = q.shape
    pages, Hkv, block, _ = k_cache.shape
    sc = scale if scale > 0 else 1 / math.sqrt(D)
    out = torch.zeros(T, H, D, dtype=torch.float64)
    lse = torch.full((T, H), -math.inf, dtype=torch.float64)
    weight = torch.zeros(T, H, D, dtype=torch.float64)
    q = q.double()
    for b, n_keys in enumerate(lens):
        n_q = starts[b + 1] - starts[b]
        ks, vs, there = [], [], []
        for j in range(0, n_keys, block):
            page = table[b][j // block]
            rows = min(block, n_keys - j)
            ok = 0 <= page < pages
            there += [ok] * rows
            page = page if ok else 0
            ks.append(k_cache[page, :, :rows].double() * k_scale[page].double()[:, None, None])
            vs.append(v_cache[page, :, :rows].double() * v_scale[page].double()[:, None, None])
        if not ks:
            continue
        k, v = torch.cat(ks, 1), torch.cat(vs, 1)  # [Hkv, keys, D]
        there = torch.tensor(there)
        k, v = torch.where(there[None, :, None], k, 0.0), torch.where(there[None, :, None], v, 0.0)
        for i in range(n_q):
            seen = there & (torch.arange(n_keys) <= n_keys - n_q + i) if causal else there
            if not bool(seen.any()):
                continue
            t = starts[b] + i
            for h in range(H):
                kv = h // (H // Hkv)
                s = (k[kv][seen] @ q[t, h]) * sc
                p = torch.softmax(s, 0)
                lse[t, h] = torch.logsumexp(s, 0)
                out[t, h] = p @ v[kv][seen]
                weight[t, h] = p @ v[kv][seen].abs()
    return out, lse, weight


def ulp(x, dtype):
    mant, low = {torch.bfloat16: (7, -126), torch.float16: (10, -14), torch.float32: (23, -126)}[dtype]
    e = torch.floor(torch.log2(x.abs().clamp_min(2.0 ** low)))
    return torch.exp2(e - mant)


def out_bound(ref, weight, lse, dtype, n_keys):
    """What an output may be off, by how it is computed.

    16-bit queries: the weights p are rounded to 11 significant bits against a
    reference near their maximum (relative error 2^-11 each, or 2^-25 of the
    reference where they are subnormal), the output once to its type.  All: the
    scores carry fp32 rounding, (D + 4) 2^-24 of sum |q k| at worst and its
    square root in practice; 2^-16 covers it for the sizes here (|s| < 30), a
    change of d in a score changes p by d."""
    # fp32 queries and weights are held in 22 bits or more.
    p = 2.0 ** -11 + n_keys * 2.0 ** -25 if dtype != torch.float32 else 2.0 ** -20
    return (p + 2.0 ** -15) * weight + 0.5 * ulp(ref, dtype) + 1e-30


def lse_bound(lse):
    return 2.0 ** -15 * (1 + lse.abs().clamp_max(1e30))


def make_cache(pages, heads, block, hidden, seed, rows_first=False, poison=None, spread=0.5):
    """(cache, scale) on the CPU with normal values; poison: the byte that rows get
    before they are written (0x7F is NaN) -- the caller writes the valid ones."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(pages, heads, block, hidden, generator=g)
    x = x * torch.exp(spread * torch.randn(pages, heads, 1, 1, generator=g))
    scale = torch.tensor([[scale_for(float(x[p, h].abs().max())) for h in range(heads)] for p in range(pages)])
    cache = (x / scale[:, :, None, None]).to(torch.float8_e4m3fn)
    if rows_first:
        cache = cache.transpose(1, 2).contiguous().transpose(1, 2)
    if poison is not None:
        cache.view(torch.uint8).fill_(poison)
    return cache, scale.float()

"""Answers with a small random attention layer from an 8-bit paged cache.

Every step plans the new tokens' pages (paged_plan), appends their keys and
values (paged_append) and attends with their queries (paged_attention): first
the prompts, then one token a request, all through one code path.  A request
that ends gives its pages back.  With --check each step's output is compared
with attention over the unquantised keys and values.

    python examples/paged_decode.py [--steps 32] [--check]
"""
import argparse
import math
import sys
from pathlib import Path

import torch

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))
import pmkl_b200  # noqa: E402,F401  (puts the binding on the path)
from pmkl_function import paged_append, paged_attention, paged_plan  # noqa: E402


class PagedCache:
    """Pages, free list and block table of `batch` requests."""

    def __init__(self, pages, kv_heads, block, hidden, batch, columns):
        dev = "cuda"
        self.block = block
        self.k = torch.zeros(pages, kv_heads, block, hidden, device=dev).to(torch.float8_e4m3fn)
        self.v = torch.zeros_like(self.k)
        self.k_scale, self.v_scale = torch.ones(pages, kv_heads, device=dev), torch.ones(pages, kv_heads, device=dev)
        self.table = torch.full((batch, columns), -1, dtype=torch.int32, device=dev)
        self.lens = torch.zeros(batch, dtype=torch.int32, device=dev)
        self.free = torch.arange(pages, dtype=torch.int32, device=dev)
        self.free_count = torch.tensor([pages], dtype=torch.int32, device=dev)

    def step(self, q, k, v, new_lens, max_new):
        """The step's tokens, packed by request: their attention output."""
        self.lens, starts, slots, self.free_count, status = paged_plan(
            self.lens, new_lens, self.table, self.free, self.free_count, self.block, q.shape[0])
        paged_append(k, v, slots, self.k, self.v, self.k_scale, self.v_scale)
        out, _ = paged_attention(q, self.k, self.v, self.k_scale, self.v_scale, self.table, self.lens, starts, max_new)
        return out, status

    def release(self, b):
        """Gives request b's pages back (host-side bookkeeping: between steps)."""
        pages = -(-int(self.lens[b]) // self.block)
        count = int(self.free_count)
        self.free[count:count + pages] = self.table[b, :pages]
        self.free_count += pages
        self.table[b] = -1
        self.lens[b] = 0


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--steps", type=int, default=32)
    ap.add_argument("--check", action="store_true")
    args = ap.parse_args()
    heads, kv_heads, hidden, block = 32, 8, 128, 16
    prompts = [300, 17, 128, 1]
    gen = torch.Generator(device="cuda").manual_seed(0)
    cache = PagedCache(256, kv_heads, block, hidden, len(prompts), 64)
    past = [([], []) for _ in prompts]
    worst = 0.0
    for step in range(args.steps):
        new = prompts if step == 0 else [1] * len(prompts)
        tokens = sum(new)
        q = torch.randn(tokens, heads, hidden, generator=gen, device="cuda", dtype=torch.bfloat16)
        k, v = (torch.randn(tokens, kv_heads, hidden, generator=gen, device="cuda", dtype=torch.bfloat16) for _ in range(2))
        out, status = cache.step(q, k, v, torch.tensor(new, dtype=torch.int32, device="cuda"), max(new))
        if args.check:
            assert not status.any(), "a request was left out"
            at = 0
            for b, n in enumerate(new):
                past[b][0].append(k[at:at + n].double())
                past[b][1].append(v[at:at + n].double())
                ks, vs = (torch.cat(x).repeat_interleave(heads // kv_heads, 1) for x in past[b])
                s = torch.einsum("qhd,khd->hqk", q[at:at + n].double(), ks) / math.sqrt(hidden)
                s += torch.full_like(s, -math.inf).triu(s.shape[2] - n + 1)
                want = torch.einsum("hqk,khd->qhd", s.softmax(-1), vs)
                worst = max(worst, float((out[at:at + n].double() - want).norm() / want.norm()))
                at += n
        if step == args.steps // 2:  # the second request ends, and a new one takes its place
            cache.release(1)
            past[1] = ([], [])
    torch.cuda.synchronize()
    if args.check:
        # e4m3 keeps 3 bits behind the leading one: 2^-4 a value, less over sums
        print(f"largest relative difference from unquantised attention: {worst:.4f}")
        assert worst < 0.1, worst
    print(f"{args.steps} steps, {int(cache.free_count)} of {cache.free.numel()} pages free, lengths {cache.lens.tolist()}")


if __name__ == "__main__":
    main()

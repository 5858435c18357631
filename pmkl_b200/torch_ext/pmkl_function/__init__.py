"""Autograd wrapper around ``pmkl_pytorch_ext`` -- the reference's public
Python API for fused self-attention, kept name for name
(``pmkl_pytorch_ext/pmkl_function/__init__.py:12-33``):

    out, out_m, out_l = fused_self_attention(q, k, v, is_casual, debug=False)

Differences from the reference, all deliberate:

* CUDA tensors run the B200 kernels whatever ``debug`` is (the reference
  raises ``NotImplementedError`` unless the tensors are on the CPU and
  ``debug`` is true, ``__init__.py:15-18``);
* CPU tensors raise ``NotImplementedError``: this build has no CPU path;
* the backward runs the B200 backward kernels on CUDA tensors (the
  reference's raises ``NotImplementedError`` for any non-CPU tensor,
  ``__init__.py:27-31``).  Like the reference it ignores the gradients
  arriving for ``out_m`` and ``out_l``;
* strided q, k, v (e.g. ``[B, S, H, D]`` tensors viewed as ``[B, H, S, D]``)
  are read in place by the forward and the backward, and the gradients come
  back in their inputs' layout.

One addition without a reference counterpart:

    out, out_m, out_l = fused_self_attention_ex(q, k, v, is_causal, scale=0.0)

takes k, v with fewer heads than q (grouped-query / multi-query attention:
query head h reads K/V head h // (H // H_kv)) and an explicit score scale
(<= 0: 1/sqrt(D)); its backward returns dk, dv with k's and v's head count,
each the sum over the query heads that read it.

For answering with a model, three operators over a paged cache of keys and
values in 8 bits (no reference counterpart); a step calls them in this order:

    seq_lens, query_starts, slot_map, free_count, status = paged_plan(
        cached_lens, new_lens, block_table, free_blocks, free_count, block_size, max_tokens)
    paged_append(k, v, slot_map, k_cache, v_cache, k_scale, v_scale)
    out, lse = paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                               query_starts=None, max_query_len=None, is_causal=True, scale=0.0)

See each function's text; ``examples/paged_decode.py`` runs them together.
"""
import torch
from torch.autograd import Function

import pmkl_pytorch_ext

__all__ = [
    'fused_self_attention',
    'fused_self_attention_ex',
    'paged_append',
    'paged_attention',
    'paged_plan',
]


class fused_self_attention_(Function):
    @staticmethod
    def forward(q, k, v, is_casual, debug=False):
        if q.is_cuda:
            return pmkl_pytorch_ext.fused_self_attention_fw(q, k, v, is_casual)
        raise NotImplementedError("pmkl_b200 runs on CUDA tensors only (no CPU path)")

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, v, is_casual, debug = inputs
        out, out_m, out_l = output
        ctx.save_for_backward(q, k, v, torch.BoolTensor([is_casual]), torch.BoolTensor([debug]), out_m, out_l)

    @staticmethod
    def backward(ctx, grad_output, grad_m, grad_l):
        q, k, v, is_casual, debug, out_m, out_l = ctx.saved_tensors
        # Strided q, k, v and grad_output are read in place (the reference
        # makes them contiguous, fused_self_attention.cpp:179).
        dq, dk, dv = pmkl_pytorch_ext.fused_self_attention_bw(
            grad_output, q, k, v, out_m, out_l, is_casual.item())
        return dq, dk, dv, None, None


fused_self_attention = fused_self_attention_.apply


class fused_self_attention_ex_(Function):
    """Grouped-query form with an explicit score scale; see the module text."""

    @staticmethod
    def forward(q, k, v, is_causal, scale=0.0):
        if q.is_cuda:
            return pmkl_pytorch_ext.fused_self_attention_fw_ex(q, k, v, is_causal, False, 0, scale)
        raise NotImplementedError("pmkl_b200 runs on CUDA tensors only (no CPU path)")

    @staticmethod
    def setup_context(ctx, inputs, output):
        q, k, v, is_causal, scale = inputs
        out, out_m, out_l = output
        ctx.is_causal = bool(is_causal)
        ctx.scale = float(scale)
        ctx.save_for_backward(q, k, v, out_m, out_l)

    @staticmethod
    def backward(ctx, grad_output, grad_m, grad_l):
        q, k, v, out_m, out_l = ctx.saved_tensors
        dq, dk, dv = pmkl_pytorch_ext.fused_self_attention_bw_ex(
            grad_output, q, k, v, out_m, out_l, ctx.is_causal, 0, ctx.scale)
        return dq, dk, dv, None, None


fused_self_attention_ex = fused_self_attention_ex_.apply


def paged_plan(cached_lens, new_lens, block_table, free_blocks, free_count, block_size, max_tokens):
    """Pages, block table and slot map for a step's new tokens, on the device.

    ``cached_lens``, ``new_lens``: [batch] int32, each request's rows in the
    cache and tokens to add.  ``block_table``: [batch, pages] int32, written in
    place where a request gets new pages.  ``free_blocks`` [n] and
    ``free_count`` [1] int32: the free pages, taken from the end of the first
    ``free_count``.  ``max_tokens``: length of the slot map, at least the new
    tokens' number.

    Returns ``seq_lens`` [batch] (cached + new), ``query_starts`` [batch + 1]
    (running sums of ``new_lens``), ``slot_map`` [max_tokens] int64 (page *
    block_size + row of each token, -1 behind the last), ``free_count`` [1] (a
    new tensor: pages left) and ``status`` [batch]: 0, or why the request was
    left out, with no page taken and -1 for its tokens (1 not enough free
    pages, 2 ``block_table`` too narrow or the length past 2^31 - 1, 3 past
    ``max_tokens``); what an attention computes for its tokens means nothing."""
    return pmkl_pytorch_ext.paged_plan(cached_lens, new_lens, block_table, free_blocks, free_count, block_size,
                                       max_tokens)


def paged_append(k, v, slot_map, k_cache, v_cache, k_scale, v_scale):
    """Writes new keys and values [tokens, kv_heads, hidden] into the cache.

    ``k_cache``, ``v_cache``: float8_e4m3fn [pages, kv_heads, block, hidden]
    (any strides with a contiguous last dimension); ``k_scale``, ``v_scale``:
    float32 [pages, kv_heads], powers of two.  ``slot_map`` int64 as from
    ``paged_plan``; tokens with a slot of -1 are skipped.  All four cache
    tensors are updated in place: the scale of a page grows with its rows, and
    rows written earlier are then rounded again to the larger scale.

    Tokens that follow one another in a page's rows are written together; a page
    may get one such run a call (``paged_plan``'s slot maps are so): two runs in
    one page would race on its scale."""
    pmkl_pytorch_ext.paged_append(k, v, slot_map, k_cache, v_cache, k_scale, v_scale)


def paged_attention(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens, query_starts=None, max_query_len=None,
                    is_causal=True, scale=0.0):
    """Attention of a step's queries [tokens, heads, hidden] over the cache.

    ``seq_lens`` [batch] counts each request's rows in the cache, the step's
    own included; request b's queries are rows ``query_starts[b]`` to
    ``query_starts[b + 1]`` of ``q`` (without ``query_starts``: row b) and stand
    at the end of its rows; with ``is_causal`` each sees the keys up to its own
    place.  ``max_query_len``, the most tokens that a request has, chooses the
    kernel and nothing else (a wrong one costs time, not results); without it
    the requests' average is taken.  Query head h reads K/V head h // (heads //
    kv_heads).  ``scale`` <= 0: 1/sqrt(hidden).

    Returns ``out`` like q and ``lse`` [tokens, heads] float32, the log of the
    sum of the exponentials (-inf, with ``out`` 0, where no key is visible and in
    rows of no request).
    Forward only: the cache is not differentiable."""
    return pmkl_pytorch_ext.paged_attention_fw(q, k_cache, v_cache, k_scale, v_scale, block_table, seq_lens,
                                               query_starts, max_query_len, is_causal, scale)

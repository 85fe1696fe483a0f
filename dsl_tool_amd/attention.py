"""Attention over the paged 8-bit cache (:mod:`dsl_tool_amd.kvcache`).

``kv8_attention`` serves single new tokens, a few drafted ones and whole
prompts by one call: ``softmax(scale * q k^T) v`` over each sequence's cached
tokens, grouped query heads included.  Scores, the softmax and the sums are
fp32; the codes enter the products exactly, and the probabilities are rounded
to bf16 for the second one (to two bf16 numbers for fp16 results).
``kv8_shared_attention`` is the same where groups of sequences share a
prefix, up to 16 query rows of a group and cache head.  Above, the probabilities are
rounded to fp16 (to two fp16 numbers for fp16 results), bf16 queries are brought to fp16 by a
power of two for each row, within 2^-32 of the row's largest, value scales below 2^-90 count as 0,
and those of one context are to lie within 2^100 of each other.  The reference's attention (triton/qwen3next/qwen3next_kernels.py) has no cache.
"""
from __future__ import annotations

import math

import torch

from . import _native as N
from .kvcache import _SRC, KV8Cache, _ints, cache_args, head_rows, most_new


def _queries(fn: str, q, cache: KV8Cache, q_starts, lens, out):
    """q as the kernels read it, and the checked or new result."""
    heads, dim = cache.k.shape[1], cache.k.shape[3]
    if not isinstance(q, torch.Tensor) or q.dim() != 3 or q.shape[1] == 0 or q.shape[1] % heads:
        raise ValueError(f"{fn}: q must be [rows, q_heads, dim], q_heads a multiple of {heads}")
    q = head_rows(q, "q", cache, q.shape[1])
    rows, q_heads, _ = q.shape
    if q_starts is None and rows != lens.shape[0]:
        raise ValueError(f"{fn}: without q_starts there is one row per sequence")
    if out is None:
        out = torch.empty((rows, q_heads, dim), dtype=q.dtype, device=q.device)
    elif (not isinstance(out, torch.Tensor) or out.shape != q.shape or out.dtype != q.dtype or out.device != q.device):
        raise ValueError(f"{fn}: out must match q in shape, type and device")
    elif out.numel() and (out.stride(2) != 1 or out.stride(1) < dim or out.stride(0) < dim or out.stride(0) % 8
                          or out.stride(1) % 8 or out.data_ptr() % 16):
        raise ValueError(f"{fn}: out needs unit stride in dim and 16-byte aligned rows and heads")
    return q, out


def kv8_attention(q: torch.Tensor, cache: KV8Cache, seq_lens: torch.Tensor, page_table: torch.Tensor, *,
                  q_starts: torch.Tensor | None = None, max_q_len: int | None = None, scale: float | None = None,
                  causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """``q [rows, q_heads, dim]`` (bf16 or fp16) attends to the cache; the
    result has q's shape and type.

    Rows ``q_starts[b] .. q_starts[b+1]`` are the queries of the last tokens of
    sequence b (None: one each, row b), ``seq_lens[b]`` its cached tokens, those
    included.  Query head h reads cache head ``h // (q_heads // heads)``.  With
    ``causal`` a row sees the tokens up to its own, else all of them; a row that
    sees none is zeros, and rows outside every sequence are not specified (``out``'s
    may be written).  ``scale`` defaults to ``1/sqrt(dim)``.  ``max_q_len``
    (the most new tokens of a sequence) sizes the launch and its workspace; the
    result does not depend on it, but the default, all rows where there are
    ``q_starts``, launches many idle workgroups for a batch of prompts (64 of 512
    tokens, 32 heads on 8: 1000 us, 416 with it).  Contexts are split by the width
    of ``page_table``: one much wider than the longest costs time (500 tokens behind
    7500: 100 us, 250 with a table for 131072), and no more than that.
    """
    if out is None:
        r = N.fast().kv8_attention(q, *cache, seq_lens, page_table, q_starts, max_q_len, scale, causal)
        if r is not None:
            return r
    args, alive = cache_args("kv8_attention", cache, seq_lens, page_table, q_starts)
    q, out = _queries("kv8_attention", q, cache, q_starts, alive[0], out)
    (rows, q_heads, _), heads, dim = q.shape, cache.k.shape[1], cache.k.shape[3]
    most = most_new(rows, q_starts, max_q_len)
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    with torch.cuda.device(q.device):
        nb = N.lib().dsl_kv8_attention_workspace_bytes(heads, cache.page, dim, args[11], args[14], rows, q_heads, most)
        ws = torch.empty(nb // 4, dtype=torch.float32, device=q.device) if nb else None
        N.call("dsl_kv8_attention", N.ptr(q), q.stride(0), q.stride(1), q_heads, *args, N.ptr(out), out.stride(0),
               out.stride(1), rows, most, scale, int(causal), _SRC[q.dtype], N.ptr(ws), nb, N.stream_of(q.device))
    return out


def kv8_shared_attention(q: torch.Tensor, cache: KV8Cache, seq_lens: torch.Tensor, page_table: torch.Tensor,
                         group_starts: torch.Tensor, shared_lens: torch.Tensor, *, q_starts: torch.Tensor | None = None,
                         max_q_len: int | None = None, max_group: int | None = None, scale: float | None = None,
                         causal: bool = True, out: torch.Tensor | None = None) -> torch.Tensor:
    """:func:`kv8_attention` where groups of sequences share a prefix, which is
    read and scored once for each group.

    Sequences ``group_starts[g] .. group_starts[g+1]`` (``[groups + 1]`` int32,
    ascending) hold the same pages for their first ``shared_lens[g]`` tokens
    (``[groups]`` int32; cut to whole pages), as :func:`kvcache.kv8_fork` leaves the
    children of one prompt.  The prefix is read by the table row of the group's first sequence
    that is as long, and what lies behind it by each sequence's own.  Sequences
    outside every group share nothing.  ``max_group``, the most sequences of a
    group (default: all of them), sizes the launch with ``max_q_len``; a wrong one costs
    speed and changes no more than roundings.  Everything else, ``out`` and the rows that
    see nothing included, is as in :func:`kv8_attention`.

    Sequences of many new tokens (more than 96 query rows to a cache head, or 64 of 64
    columns, by ``max_q_len``, so give it) fill the matrix units by themselves and are
    computed as by :func:`kv8_attention`, which is also faster for few sequences behind
    a short prefix (six of four heads to a cache head behind 1000 tokens).  All others' rows
    times query heads are 2^22 at most; their workspace is eight bytes for each element of q, up
    to 32 MB more.
    """
    if out is None:
        r = N.fast().kv8_shared_attention(q, *cache, seq_lens, page_table, q_starts, max_q_len, scale, causal,
                                          group_starts, shared_lens, max_group)
        if r is not None:
            return r
    fn = "kv8_shared_attention"
    args, alive = cache_args(fn, cache, seq_lens, page_table, q_starts)
    q, out = _queries(fn, q, cache, q_starts, alive[0], out)
    (rows, q_heads, _), heads, dim = q.shape, cache.k.shape[1], cache.k.shape[3]
    groups = _ints(group_starts, "group_starts", q.device).contiguous()
    shared = _ints(shared_lens, "shared_lens", q.device).contiguous()
    if groups.dim() != 1 or shared.dim() != 1 or groups.shape[0] != shared.shape[0] + 1:
        raise ValueError(f"{fn}: group_starts must be [groups + 1] and shared_lens [groups]")
    if max_group is None:
        max_group = alive[0].shape[0]
    elif not isinstance(max_group, int) or max_group < 0:
        raise ValueError(f"{fn}: max_group must be a number >= 0 (got {max_group!r})")
    most = most_new(rows, q_starts, max_q_len)
    scale = 1.0 / math.sqrt(dim) if scale is None else float(scale)
    with torch.cuda.device(q.device):
        nb = N.lib().dsl_kv8_shared_attention_workspace_bytes(heads, cache.page, dim, args[11], args[14], rows, q_heads,
                                                              most, shared.shape[0], max_group)
        ws = torch.empty(-(-nb // 4), dtype=torch.float32, device=q.device)
        N.call("dsl_kv8_shared_attention", N.ptr(q), q.stride(0), q.stride(1), q_heads, *args, N.ptr(groups),
               N.ptr(shared), shared.shape[0], max_group, N.ptr(out), out.stride(0), out.stride(1), rows, most, scale,
               int(causal), _SRC[q.dtype], N.ptr(ws), nb, N.stream_of(q.device))
    return out

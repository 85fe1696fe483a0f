"""A paged key/value cache in 8 bits: one scale for each page and head.

A page holds ``page`` consecutive tokens of one sequence (16, 32, 64, 128 or
256), ``page_table [seqs, width]`` names each sequence's pages in order, and a
code stands for ``code * scale[page, head]``:

    cache = new_kv8_cache(pages, kv_heads, head_dim, page=64, fmt="int8")
    kv8_write(cache, k, v, seq_lens, page_table)           # one new token each
    kv8_write(cache, k, v, seq_lens, page_table, q_starts=starts)   # prompts
    o = attention.kv8_attention(q, cache, seq_lens, page_table)
    k, v = kv8_read(cache, seq_lens, page_table, starts, total)

``seq_lens`` counts a sequence's tokens with the new ones, which are its last.
Lengths, starts and the table are int32 tensors on the device and nothing is
copied to the host: page numbers outside the cache, tokens past a table row
and rows outside the tensors are skipped.  Everything runs in
``libdsl_gemm.so``.  The reference has no cache.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N

PAGES = (16, 32, 64, 128, 256)
HEAD_DIMS = (64, 128, 256)
_FMT = {torch.int8: N.KV_INT8, torch.float8_e4m3fn: N.KV_FP8}
_SRC = {torch.bfloat16: N.IN_BF16, torch.float16: N.IN_F16}


class KV8Cache(NamedTuple):
    k: torch.Tensor          # [pages, heads, page, dim] int8 or float8_e4m3fn
    v: torch.Tensor          # [pages, heads, dim, page]
    k_scale: torch.Tensor    # [pages, heads] float32
    v_scale: torch.Tensor

    @property
    def page(self) -> int:
        return self.k.shape[2]


def new_kv8_cache(pages: int, heads: int, dim: int, *, page: int = 64, fmt: str = "int8", device="cuda") -> KV8Cache:
    """An empty cache (zero codes and scales); fmt "int8" or "fp8" (E4M3)."""
    if fmt not in ("int8", "fp8"):
        raise ValueError(f"fmt must be 'int8' or 'fp8', got {fmt!r}")
    if page not in PAGES or dim not in HEAD_DIMS:
        raise ValueError(f"page must be one of {PAGES} and dim one of {HEAD_DIMS} (got {page}, {dim})")
    if pages < 0 or heads <= 0:
        raise ValueError("need pages >= 0 and heads > 0")
    dt = torch.int8 if fmt == "int8" else torch.float8_e4m3fn
    k = torch.zeros((pages, heads, page, dim), dtype=torch.int8, device=device).view(dt)
    v = torch.zeros((pages, heads, dim, page), dtype=torch.int8, device=device).view(dt)
    scales = torch.zeros((2, pages, heads), dtype=torch.float32, device=device)
    return KV8Cache(k, v, scales[0], scales[1])


def _ints(t, name: str, dev) -> torch.Tensor:
    if not isinstance(t, torch.Tensor) or t.device != dev:
        raise ValueError(f"{name} must be an integer tensor on {dev}")
    if t.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"{name} must be int32 (got {t.dtype})")
    return t.to(torch.int32)


def cache_args(fn: str, cache: KV8Cache, seq_lens, page_table, starts):
    """The cache and sequence arguments of the C entry points, checked; the
    second result keeps converted tensors alive for the call."""
    k, v, ks, vs = cache
    for t, name in zip(cache, KV8Cache._fields):
        if not isinstance(t, torch.Tensor) or t.device.type != "cuda":
            raise ValueError(f"{fn}: cache.{name} must be a tensor on a GPU device")
        if t.device != k.device or not t.is_contiguous():
            raise ValueError(f"{fn}: cache tensors must be contiguous and on one device")
    if k.dtype not in _FMT or v.dtype != k.dtype:
        raise TypeError(f"{fn}: cache codes must be int8 or float8_e4m3fn (got {k.dtype}, {v.dtype})")
    if ks.dtype != torch.float32 or vs.dtype != torch.float32:
        raise TypeError(f"{fn}: cache scales must be float32")
    if k.dim() != 4:
        raise ValueError(f"{fn}: cache.k must be [pages, heads, page, dim]")
    pages, heads, page, dim = k.shape
    if tuple(v.shape) != (pages, heads, dim, page) or tuple(ks.shape) != (pages, heads) or ks.shape != vs.shape:
        raise ValueError(f"{fn}: cache.v must be [pages, heads, dim, page], the scales [pages, heads]")
    if page not in PAGES or dim not in HEAD_DIMS:
        raise ValueError(f"{fn}: page must be one of {PAGES} and dim one of {HEAD_DIMS} (got {page}, {dim})")
    lens = _ints(seq_lens, "seq_lens", k.device).contiguous()
    table = _ints(page_table, "page_table", k.device)
    if lens.dim() != 1 or table.dim() != 2 or table.shape[0] != lens.shape[0]:
        raise ValueError(f"{fn}: seq_lens must be [seqs] and page_table [seqs, width]")
    if table.stride(1) != 1 or table.stride(0) < table.shape[1]:
        table = table.contiguous()
    if starts is not None:
        starts = _ints(starts, "starts", k.device).contiguous()
        if starts.dim() != 1 or starts.shape[0] != lens.shape[0] + 1:
            raise ValueError(f"{fn}: starts must be [seqs + 1]")
    ptrs = [N.ptr(k), N.ptr(v), N.ptr(ks), N.ptr(vs)]
    rest = [pages, heads, page, dim, _FMT[k.dtype], N.ptr(table), table.stride(0) if table.shape[0] > 1 else
            max(table.shape[1], 1), table.shape[1], N.ptr(lens), N.ptr(starts), lens.shape[0]]
    return ptrs + rest, (lens, table, starts)


def head_rows(t, name: str, cache: KV8Cache, heads: int) -> torch.Tensor:
    """``t [rows, heads, dim]`` in a layout the kernels read in place: unit
    stride in dim, 16-byte aligned rows and heads; else a contiguous copy."""
    if not isinstance(t, torch.Tensor) or t.dim() != 3 or t.device != cache.k.device:
        raise ValueError(f"{name} must be [rows, heads, dim] on {cache.k.device}")
    if t.dtype not in _SRC:
        raise TypeError(f"{name} must be bfloat16 or float16 (got {t.dtype})")
    if t.shape[2] != cache.k.shape[3] or t.shape[1] != heads:
        raise ValueError(f"{name} must have {heads} heads of {cache.k.shape[3]} (got {list(t.shape)})")
    if (t.stride(2) == 1 and t.stride(1) % 8 == 0 and t.stride(0) % 8 == 0 and t.stride(0) >= 0
            and (heads == 1 or t.stride(1) >= t.shape[2]) and t.data_ptr() % 16 == 0):
        return t
    return torch.empty(t.shape, dtype=t.dtype, device=t.device).copy_(t)


def most_new(rows: int, starts, max_q_len) -> int:
    if max_q_len is None:
        return 1 if starts is None else rows
    if not isinstance(max_q_len, int) or max_q_len < 0:
        raise ValueError(f"max_q_len must be a number >= 0 (got {max_q_len!r})")
    return max_q_len


def kv8_write(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor, seq_lens: torch.Tensor, page_table: torch.Tensor,
              *, q_starts: torch.Tensor | None = None, max_q_len: int | None = None) -> None:
    """Quantize the new tokens' keys and values ``[rows, heads, dim]`` (bf16 or
    fp16, views of a fused projection included) into the cache.

    Rows ``q_starts[b] .. q_starts[b+1]`` (ascending) are the last tokens of
    sequence b (None: one token each, row b).  The scale of a page and head becomes
    ``max(kept, amax(new)/top, 1e-12)``; ``kept`` is the one it had where older
    tokens stay in the page, and their codes move to a larger scale.  Two
    sequences must not write one page in the same call.  ``max_q_len`` (the most
    new tokens of a sequence) is taken so that one set of arguments serves this
    call and ``kv8_attention``; the launch is sized by the rows.
    """
    r = N.fast().kv8_write(*cache, k, v, seq_lens, page_table, q_starts, max_q_len)
    if r is not None:
        return
    args, alive = cache_args("kv8_write", cache, seq_lens, page_table, q_starts)
    heads = cache.k.shape[1]
    k, v = head_rows(k, "k", cache, heads), head_rows(v, "v", cache, heads)
    if k.shape[0] != v.shape[0] or k.dtype != v.dtype:
        raise ValueError("kv8_write: k and v must have the same rows and type")
    if q_starts is None and k.shape[0] != alive[0].shape[0]:
        raise ValueError("kv8_write: without q_starts there is one row per sequence")
    with torch.cuda.device(k.device):
        N.call("dsl_kv8_write", *args, N.ptr(k), k.stride(0), k.stride(1), N.ptr(v), v.stride(0), v.stride(1),
               k.shape[0], most_new(k.shape[0], q_starts, max_q_len), _SRC[k.dtype], N.stream_of(k.device))


def kv8_read(cache: KV8Cache, seq_lens: torch.Tensor, page_table: torch.Tensor, starts: torch.Tensor, total: int, *,
             dtype: torch.dtype = torch.bfloat16):
    """The cached tokens back in 16 bits: ``(k, v)``, each ``[total, heads,
    dim]``; rows ``starts[b] .. starts[b+1]`` (ascending) are sequence b's tokens from its
    first on (rows past its length are zeros; rows outside every
    sequence are not written)."""
    if dtype not in _SRC:
        raise TypeError(f"kv8_read: dtype must be bfloat16 or float16 (got {dtype})")
    if not isinstance(total, int) or total < 0:
        raise ValueError(f"kv8_read: total must be a number >= 0 (got {total!r})")
    r = N.fast().kv8_read(*cache, seq_lens, page_table, starts, total, dtype)
    if r is not None:
        return r
    if starts is None:
        raise ValueError("kv8_read: starts must be [seqs + 1]")
    args, alive = cache_args("kv8_read", cache, seq_lens, page_table, starts)
    shape = (total, cache.k.shape[1], cache.k.shape[3])
    k, v = (torch.empty(shape, dtype=dtype, device=cache.k.device) for _ in range(2))
    with torch.cuda.device(k.device):
        N.call("dsl_kv8_read", *args, N.ptr(k), N.ptr(v), total, _SRC[dtype], N.stream_of(k.device))
    del alive
    return k, v

"""A causal self-attention layer in 8 bits, from the operators it is made of:

    residual norm -> int8 codes        fused.add_rmsnorm_quant
    -> query, key, value projection    gemm.int8_gemm_packed
    -> positions                       rotary.rotary
    -> keys and values into the cache  kvcache.kv8_write
    -> attention over the cache        attention.kv8_attention, or kv8_shared_attention
    -> int8 codes                      quant.quant_int8_rows
    -> output projection               gemm.int8_gemm_packed

Prompts and single tokens take the same call, which allocates from torch's
pool only and copies nothing to the host, so that a step can be captured in a
graph.
"""
from __future__ import annotations

import torch

from . import attention as A
from . import fused as FU
from . import gemm as G
from . import kvcache as KV
from . import quant as Q
from . import rotary as R


def _product(q, w, s, sw, dtype):
    """The int8 product in the activations' type.  Its results are bf16 or fp32, so
    fp16 comes from fp32 by a pass of its own: one rounding, and fp16's bits."""
    if dtype == torch.bfloat16:
        return G.int8_gemm_packed(q, w, s, sw, out_dtype=dtype)
    return G.int8_gemm_packed(q, w, s, sw, out_dtype=torch.float32).to(dtype)


class Int8AttentionLayer:
    """``w_qkv [(q_heads + 2 kv_heads) * dim, hidden]`` (queries, keys, values in
    this order), ``w_out [hidden, q_heads * dim]`` and ``norm [hidden]``: bf16,
    fp16 or fp32, on the GPU.  The weights are quantized once, per output
    channel; ``rotate(q, k) -> (q, k)`` is applied to the projected heads
    (``[rows, heads, dim]``) before they are used: a position encoding.  With
    ``freqs`` (and ``axis_of``, ``adjacent``: :func:`rotary.rotary`) they are turned by the
    call's positions instead."""

    def __init__(self, w_qkv: torch.Tensor, w_out: torch.Tensor, norm: torch.Tensor, *, q_heads: int, kv_heads: int,
                 dim: int, eps: float = 1e-6, rotate=None, freqs: torch.Tensor | None = None,
                 axis_of: torch.Tensor | None = None, adjacent: bool = False):
        if q_heads <= 0 or kv_heads <= 0 or q_heads % kv_heads:
            raise ValueError(f"q_heads must be a multiple of kv_heads (got {q_heads}, {kv_heads})")
        if rotate is not None and freqs is not None:
            raise ValueError("positions are encoded by rotate or by freqs, not by both")
        if freqs is None and (axis_of is not None or adjacent):
            raise ValueError("axis_of and adjacent say how freqs turn the heads: give freqs too")
        hidden = norm.shape[0]
        if w_qkv.shape != ((q_heads + 2 * kv_heads) * dim, hidden) or w_out.shape != (hidden, q_heads * dim):
            raise ValueError(f"w_qkv must be [{(q_heads + 2 * kv_heads) * dim}, {hidden}] and w_out "
                             f"[{hidden}, {q_heads * dim}] (got {tuple(w_qkv.shape)}, {tuple(w_out.shape)})")
        self.q_heads, self.kv_heads, self.dim, self.eps, self.rotate = q_heads, kv_heads, dim, eps, rotate
        self.freqs, self.axis_of, self.adjacent = freqs, axis_of, adjacent
        self.norm = norm.float() if norm.dtype == torch.float16 else norm      # once: the kernels take bf16 and fp32
        self.w_qkv, self.s_qkv = Q.quant_int8_rows(w_qkv)
        self.w_out, self.s_out = Q.quant_int8_rows(w_out)

    def __call__(self, x: torch.Tensor, residual: torch.Tensor | None, cache: KV.KV8Cache, seq_lens: torch.Tensor,
                 page_table: torch.Tensor, *, q_starts: torch.Tensor | None = None, max_q_len: int | None = None,
                 positions: torch.Tensor | None = None, group_starts: torch.Tensor | None = None,
                 shared_lens: torch.Tensor | None = None, max_group: int | None = None):
        """The layer's output for the new tokens ``x [rows, hidden]`` (bf16 or fp16)
        and the new residual: ``(out, h)``, both of x's type, as the next layer
        takes them.  Their keys and values go into the cache; ``seq_lens`` counts
        them, rows and starts are those of :func:`kvcache.kv8_write`.  ``positions``
        are the rows', of a layer with ``freqs``; ``group_starts``, ``shared_lens`` and
        ``max_group`` name sequences that share a prefix, as
        :func:`attention.kv8_shared_attention` takes them."""
        if (self.freqs is None) != (positions is None):
            raise ValueError("a layer with freqs needs the rows' positions, and one without takes none")
        if (group_starts is None) != (shared_lens is None) or (group_starts is None and max_group is not None):
            raise ValueError("group_starts and shared_lens come together, max_group only with them")
        codes, scales, h = FU.add_rmsnorm_quant(x, residual, self.norm, self.eps)
        qkv = _product(codes, self.w_qkv, scales, self.s_qkv, x.dtype)
        qkv = qkv.view(x.shape[0], self.q_heads + 2 * self.kv_heads, self.dim)
        q, k, v = qkv.split([self.q_heads, self.kv_heads, self.kv_heads], dim=1)
        if self.rotate is not None:
            q, k = self.rotate(q, k)
        elif self.freqs is not None:
            q, k = R.rotary(q, k, positions, self.freqs, axis_of=self.axis_of, adjacent=self.adjacent)
        KV.kv8_write(cache, k, v, seq_lens, page_table, q_starts=q_starts, max_q_len=max_q_len)
        if group_starts is None:
            o = A.kv8_attention(q, cache, seq_lens, page_table, q_starts=q_starts, max_q_len=max_q_len)
        else:
            o = A.kv8_shared_attention(q, cache, seq_lens, page_table, group_starts, shared_lens, q_starts=q_starts,
                                       max_q_len=max_q_len, max_group=max_group)
        codes, scales = Q.quant_int8_rows(o.view(x.shape[0], self.q_heads * self.dim))
        return _product(codes, self.w_out, scales, self.s_out, x.dtype), h

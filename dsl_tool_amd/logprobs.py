"""Log probabilities of given tokens, the entropy and the best alternatives
of logits (:func:`gemm.bf16_gemm`, say, of the last hidden states), in one pass
over them.  Everything runs in ``libdsl_gemm.so``; the reference has none of it.
"""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N

TOP = 32                     # most alternatives of a row
_SRC = {torch.bfloat16: N.IN_BF16, torch.float16: N.IN_F16, torch.float32: N.IN_F32}


class TokenLogprobs(NamedTuple):
    logp: torch.Tensor           # of the given tokens, float32, the shape of ids
    entropy: torch.Tensor        # [rows] float32
    top_logp: torch.Tensor       # [rows, top] float32, falling
    top_ids: torch.Tensor        # [rows, top] int32


def token_logprobs(logits: torch.Tensor, ids: torch.Tensor | None = None, *, top: int = 0,
                   scale: float = 1.0) -> TokenLogprobs:
    """Of ``softmax(scale * logits)``, ``logits [rows, vocab]`` bf16, fp16 or
    fp32 (``scale``: 1 / temperature, below 2^126): natural log probabilities of the tokens ``ids``
    (int32, ``[rows]`` or ``[rows, n]``; None: none, ``logp [rows, 0]``), the entropy, and the
    ``top`` (up to 32) likeliest tokens, ties by the lowest number.

    Logits of -inf (tokens that are not allowed) have probability 0, log -inf;
    so have ids outside the vocabulary.  A row of nothing else has entropy 0.  Finite logits of any
    size are what they are: tokens masked by the type's lowest value have about that for their
    log probability, and a row of nothing else is uniform.  NaN or
    +inf make all of a row's results NaN but ``top_ids``.
    """
    r = N.fast().token_logprobs(logits, ids, top, scale)
    if r is not None:
        return TokenLogprobs(*r)
    if not isinstance(logits, torch.Tensor) or logits.dim() != 2:
        raise ValueError("token_logprobs: logits must be [rows, vocab]")
    if logits.device.type != "cuda":
        raise ValueError(f"token_logprobs: tensor must be on a GPU device (got {logits.device})")
    if logits.dtype not in _SRC:
        raise TypeError(f"token_logprobs: logits must be bfloat16, float16 or float32 (got {logits.dtype})")
    rows, vocab = logits.shape
    if vocab == 0:
        raise ValueError("token_logprobs: the vocabulary is empty")
    if not isinstance(top, int) or isinstance(top, bool) or not 0 <= top <= min(TOP, vocab):
        raise ValueError(f"token_logprobs: top must be 0 .. {min(TOP, vocab)} (got {top!r})")
    scale = float(scale)
    if not 0 < scale < 2.0 ** 126:
        raise ValueError(f"token_logprobs: scale must be > 0 and below 2^126 (got {scale!r})")
    dev = logits.device
    if ids is None:
        ids = torch.empty((rows, 0), dtype=torch.int32, device=dev)
    if not isinstance(ids, torch.Tensor) or ids.device != dev or ids.dim() not in (1, 2) or ids.shape[0] != rows:
        raise ValueError(f"token_logprobs: ids must be [{rows}] or [{rows}, n] on {dev}")
    if ids.dtype not in (torch.int32, torch.int64):
        raise TypeError(f"token_logprobs: ids must be int32 (got {ids.dtype})")
    # (numbers past 32 bits are no tokens: not wrapped into ones that are)
    ids32 = (ids if ids.dtype == torch.int32 else ids.clamp(-1, 2 ** 31 - 1).to(torch.int32)).contiguous()
    n_ids = ids32.numel() // rows if rows else 0
    if logits.stride(1) != 1 and vocab > 1 or (rows > 1 and logits.stride(0) < vocab):
        logits = logits.contiguous()
    out = TokenLogprobs(torch.empty(ids.shape, dtype=torch.float32, device=dev),
                        torch.empty(rows, dtype=torch.float32, device=dev),
                        torch.empty((rows, top), dtype=torch.float32, device=dev),
                        torch.empty((rows, top), dtype=torch.int32, device=dev))
    with torch.cuda.device(dev):
        nb = N.lib().dsl_token_logprobs_workspace_bytes(rows, vocab, top, _SRC[logits.dtype])
        ws = torch.empty(-(-nb // 4), dtype=torch.int32, device=dev) if nb else None
        N.call("dsl_token_logprobs", N.ptr(logits), rows, vocab, max(logits.stride(0), vocab), _SRC[logits.dtype],
               N.ptr(ids32), n_ids, n_ids, scale, top, *(N.ptr(t) for t in out), N.ptr(ws), nb, N.stream_of(dev))
    return out

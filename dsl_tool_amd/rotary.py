"""Rotary positions of queries and keys, with one axis or several (time,
height and width of a frame's patches, say).

Pair i of a head is turned by the angle ``positions[axis_of[i]] * freqs[i]``:

    freqs = rotary_freqs(128)                       # 10000 ** (-i / 64), float64
    axis_of = rotary_axes([16, 24, 24])             # which axis turns which pair
    q, k = rotary(q, k, positions, freqs, axis_of=axis_of)

Angles are formed in 64 bits, so far positions keep their digits: an angle of a
radians is off by ``|a| * 2 ** -51`` and the 2^-22 of its turn in 32 bits.  Everything
runs in ``libdsl_gemm.so``.  The reference's RoPE
(triton/rope/rope_kernel.py:11-145) has one axis.
"""
from __future__ import annotations

from collections.abc import Sequence

import torch

from . import _native as N

_SRC = {torch.bfloat16: N.IN_BF16, torch.float16: N.IN_F16}


def rotary_freqs(rotary_dim: int, theta: float = 10000.0, device="cuda") -> torch.Tensor:
    """``theta ** (-2 i / rotary_dim)`` for the pairs i of ``rotary_dim`` dimensions."""
    if not isinstance(rotary_dim, int) or rotary_dim < 0 or rotary_dim % 2 or not theta > 0:
        raise ValueError(f"rotary_freqs: need an even rotary_dim >= 0 and theta > 0 (got {rotary_dim!r}, {theta!r})")
    return theta ** (torch.arange(0, rotary_dim, 2, dtype=torch.float64, device=device) / -max(rotary_dim, 1))


def rotary_axes(sections: Sequence[int], *, interleaved: bool = False, device="cuda") -> torch.Tensor:
    """The axis of each pair, int32: ``sections[a]`` pairs of axis a, one axis
    after another, or dealt in turn (an axis whose pairs are dealt is passed
    over)."""
    if not sections or any(not isinstance(n, int) or n < 0 for n in sections):
        raise ValueError(f"rotary_axes: sections must be numbers >= 0 (got {sections!r})")
    if interleaved:
        order = [a for i in range(max(sections)) for a, n in enumerate(sections) if i < n]
    else:
        order = [a for a, n in enumerate(sections) for _ in range(n)]
    return torch.tensor(order, dtype=torch.int32, device=device)


def _heads(t, name: str, like=None):
    if not isinstance(t, torch.Tensor) or t.dim() != 3:
        raise ValueError(f"rotary: {name} must be [rows, heads, dim]")
    if t.device.type != "cuda":
        raise ValueError(f"rotary: tensor must be on a GPU device (got {t.device})")
    if t.dtype not in _SRC:
        raise TypeError(f"rotary: {name} must be bfloat16 or float16 (got {t.dtype})")
    if like is not None and (t.dtype != like.dtype or t.device != like.device or t.shape[0] != like.shape[0]
                             or t.shape[2] != like.shape[2]):
        raise ValueError("rotary: k must match q in rows, dim, type and device")


def _in_place(t) -> bool:
    """Rows and heads that the kernel writes in place: unit stride in dim, none overlapping."""
    rows, heads, dim = t.shape
    return ((t.stride(2) == 1 or dim == 1) and (heads == 1 or t.stride(1) >= dim)
            and (rows == 1 or t.stride(0) >= (heads - 1) * t.stride(1) + dim))


def rotary(q: torch.Tensor, k: torch.Tensor | None, positions: torch.Tensor, freqs: torch.Tensor, *,
           axis_of: torch.Tensor | None = None, adjacent: bool = False, magnitude: float = 1.0, inplace: bool = False):
    """``(q, k)`` turned by their positions: q ``[rows, heads, dim]`` bf16 or
    fp16, k (None: none) the same with its own heads.

    ``positions`` ``[rows]``, or ``[axes, rows]`` with ``axis_of [pairs]`` int32
    (:func:`rotary_axes`), is int32 or int64; ``freqs [pairs]``
    float64 (:func:`rotary_freqs`; other types are widened, once a call).  Pairs are
    the dimensions ``(i, i + pairs)``, or ``(2 i, 2 i + 1)`` with ``adjacent``; those
    from ``2 * pairs`` on stay.  Results are multiplied by ``magnitude`` (of the turned
    dimensions) and rounded once.  ``inplace`` writes them over q and k, views of a
    fused projection included.
    """
    if not inplace:
        r = N.fast().rotary(q, k, positions, freqs, axis_of, adjacent, magnitude)
        if r is not None:
            return r
    _heads(q, "q")
    if k is not None:
        _heads(k, "k", q)
    dev, (rows, heads, dim) = q.device, q.shape
    if heads == 0 or dim == 0 or (k is not None and k.shape[1] == 0):
        raise ValueError("rotary: q and k must have heads and dimensions")
    for t, name, dtypes in ((positions, "positions", (torch.int32, torch.int64)),
                            (freqs, "freqs", (torch.float64, torch.float32, torch.float16, torch.bfloat16))):
        if not isinstance(t, torch.Tensor) or t.device != dev:
            raise ValueError(f"rotary: {name} must be a tensor on {dev}")
        if t.dtype not in dtypes:
            raise TypeError(f"rotary: {name} has an unsupported type ({t.dtype})")
    if positions.dim() not in (1, 2) or positions.shape[-1] != rows or positions.shape[0] == 0 and rows:
        raise ValueError(f"rotary: positions must be [{rows}] or [axes, {rows}] (got {list(positions.shape)})")
    pos = positions.view(1, rows) if positions.dim() == 1 and positions.is_contiguous() else positions
    if pos.dim() == 1:
        pos = pos.contiguous().view(1, rows)
    if pos.stride(1) != 1 or pos.stride(0) < rows:
        pos = pos.contiguous()
    if freqs.dim() != 1 or 2 * freqs.shape[0] > dim:
        raise ValueError(f"rotary: freqs must be [pairs], 2 * pairs <= {dim} (got {list(freqs.shape)})")
    freqs = freqs.double().contiguous()
    if axis_of is None:
        if pos.shape[0] != 1:
            raise ValueError("rotary: positions of several axes need axis_of")
    else:
        if not isinstance(axis_of, torch.Tensor) or axis_of.device != dev or axis_of.shape != freqs.shape:
            raise ValueError("rotary: axis_of must be [pairs] on the device of q")
        if axis_of.dtype not in (torch.int32, torch.int64):
            raise TypeError(f"rotary: axis_of must be int32 (got {axis_of.dtype})")
        axis_of = axis_of.to(torch.int32).contiguous()
    magnitude = float(magnitude)
    if inplace:
        if any(t is not None and t.numel() and not _in_place(t) for t in (q, k)):
            raise ValueError("rotary: in place needs unit stride in dim and heads and rows that do not overlap")
        src, out = [q, k], [q, k]
    else:
        src = [t if t is None or (t.stride(2) == 1 and t.stride(0) >= 0 and (t.shape[1] == 1 or t.stride(1) >= dim))
               else t.contiguous() for t in (q, k)]
        out = [None if t is None else torch.empty(t.shape, dtype=t.dtype, device=dev) for t in (q, k)]
    args = [a for t in src for a in ((N.ptr(t), t.stride(0), t.stride(1), t.shape[1]) if t is not None else (None, 0, 0, 0))]
    outs = [a for t in out for a in ((N.ptr(t), t.stride(0), t.stride(1)) if t is not None else (None, 0, 0))]
    with torch.cuda.device(dev):
        N.call("dsl_rotary", *args, rows, dim, freqs.shape[0], N.ptr(pos), int(pos.dtype == torch.int64),
               max(pos.stride(0), rows), pos.shape[0], N.ptr(axis_of), N.ptr(freqs), magnitude, int(adjacent),
               _SRC[q.dtype], *outs, N.stream_of(dev))
    return out[0], out[1]

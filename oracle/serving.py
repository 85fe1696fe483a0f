"""The 8-bit attention layer's operators, plainly (CPU) -- TEST INFRASTRUCTURE ONLY.

Loops over sequences, pages and heads in 64 bits; the quantizers, whose codes
are pinned bit for bit, in IEEE fp32.
"""
from __future__ import annotations

import math

import torch

TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
FLOOR = torch.tensor(1e-12, dtype=torch.float32)


def encode(x: torch.Tensor, s: torch.Tensor, dtype) -> torch.Tensor:
    """Codes of the IEEE fp32 quotient x / s."""
    y = x / s
    return y.round().clamp(-127, 127).to(torch.int8) if dtype == torch.int8 else y.to(torch.float8_e4m3fn)


def scale_of(amax: torch.Tensor, dtype) -> torch.Tensor:
    return torch.maximum(amax.float() / torch.tensor(TOP[dtype]), FLOOR)


def quant_rows(x: torch.Tensor):
    s = scale_of(x.float().abs().amax(1), torch.int8)
    return encode(x.float(), s[:, None], torch.int8), s


def norm(x, residual, w, eps):
    """(h, y) in 64 bits."""
    h = x.double() if residual is None else x.double() + residual.double()
    return h, h / (h.pow(2).mean(1, keepdim=True) + eps).sqrt() * w.double()


def sequences(lens, starts, rows):
    """(sequence, length, first position, first row, new tokens) of each."""
    for b, n in enumerate(lens.tolist()):
        n = max(n, 0)
        lo, hi = (b, b + 1) if starts is None else (starts[b].item(), starts[b + 1].item())
        lo, hi = min(max(lo, 0), rows), min(max(hi, 0), rows)
        new = max(hi - lo, 0)
        yield b, n, n - new, lo, new


def write(cache, k, v, lens, table, starts=None):
    """kv8_write on CPU tensors, in place."""
    kc, vc, ks, vs = cache
    pages, heads, page, _ = kc.shape
    for b, n, first, row0, new in sequences(lens, starts, k.shape[0]):
        if new == 0:
            continue
        begin = max(first, 0)
        for i in range(begin // page, (n + page - 1) // page):
            if i >= table.shape[1] or not 0 <= table[b, i] < pages:
                continue
            p = table[b, i].item()
            lo, hi = max(begin - i * page, 0), min(n - i * page, page)
            rows = slice(row0 + i * page + lo - first, row0 + i * page + hi - first)
            for codes, scales, x in ((kc[p], ks, k), (vc[p].transpose(1, 2), vs, v)):
                new = x[rows].float().transpose(0, 1)                # [heads, tokens, dim]
                kept = scales[p].clone() if lo > 0 else torch.zeros(heads)
                s = torch.maximum(kept, scale_of(new.abs().amax((1, 2)), codes.dtype))
                if lo > 0:
                    old = codes[:, :lo].float()
                    moved = encode(old * kept[:, None, None], s[:, None, None], codes.dtype)
                    grew = (s > kept)[:, None, None]
                    codes[:, :lo] = torch.where(grew, moved.float(), old).to(codes.dtype)
                codes[:, lo:hi] = encode(new, s[:, None, None], codes.dtype)
                scales[p] = s


def tokens(cache, length, pages_of):
    """Keys, values [heads, length, dim] in 64 bits, and which tokens there are."""
    kc, vc, ks, vs = cache
    pages, heads, page, dim = kc.shape
    k = torch.zeros((heads, length, dim), dtype=torch.float64)
    v, there = torch.zeros_like(k), torch.zeros(length, dtype=torch.bool)
    for i in range((length + page - 1) // page):
        if i >= len(pages_of) or not 0 <= pages_of[i] < pages:
            continue
        p, lo, hi = pages_of[i], i * page, min((i + 1) * page, length)
        k[:, lo:hi] = kc[p, :, :hi - lo].double() * ks[p].double()[:, None, None]
        v[:, lo:hi] = vc[p, :, :, :hi - lo].double().transpose(1, 2) * vs[p].double()[:, None, None]
        there[lo:hi] = True
    return k, v, there


def read(cache, lens, table, starts, total):
    heads, dim = cache[0].shape[1], cache[0].shape[3]
    out = torch.zeros((2, total, heads, dim), dtype=torch.float64)
    for b, n, _, row0, new in sequences(lens, starts, total):
        k, v, _ = tokens(cache, min(n, new), table[b].tolist())
        out[0, row0:row0 + k.shape[1]] = k.transpose(0, 1)
        out[1, row0:row0 + k.shape[1]] = v.transpose(0, 1)
    return out[0], out[1]


def attention(q, cache, lens, table, starts=None, scale=None, causal=True):
    """(o, a, reach) in 64 bits: the result; sum of p |v|, what the rounding of
    the probabilities is relative to; and the largest sum of |scale q k|, what
    the fp32 scores' error is relative to, per row and head."""
    rows, hq, dim = q.shape
    heads = cache[0].shape[1]
    group = hq // heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    o = torch.zeros((rows, hq, dim), dtype=torch.float64)
    a, reach = torch.zeros_like(o), torch.zeros((rows, hq, 1), dtype=torch.float64)
    for b, n, first, row0, new in sequences(lens, starts, rows):
        n = min(n, table.shape[1] * cache[0].shape[2])
        if new == 0 or n == 0:
            continue
        k, v, there = tokens(cache, n, table[b].tolist())
        x = q[row0:row0 + new].double().reshape(new, heads, group, dim)
        z = torch.einsum("ihgd,htd->ihgt", x, k) * scale
        far = torch.einsum("ihgd,htd->ihgt", x.abs(), k.abs()).amax(-1) * abs(scale)
        seen = there[None, :].expand(new, n)
        if causal:
            seen = seen & (torch.arange(n)[None, :] <= first + torch.arange(new)[:, None])
        z = z.masked_fill(~seen[:, None, None, :], -math.inf)
        top = z.amax(-1, keepdim=True).clamp_min(-1e300)
        p = (z - top).exp()
        p = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
        o[row0:row0 + new] = torch.einsum("ihgt,htd->ihgd", p, v).reshape(new, hq, dim)
        a[row0:row0 + new] = torch.einsum("ihgt,htd->ihgd", p, v.abs()).reshape(new, hq, dim)
        reach[row0:row0 + new] = far.reshape(new, hq, 1)
    return o, a, reach

"""What generates several continuations of a prompt, plainly (CPU) -- TEST
INFRASTRUCTURE ONLY.

Loops over sequences, pages, pairs and rows; numbers in 64 bits.  Attention over
shared prefixes has :func:`oracle.serving.attention` for its oracle: every
sequence's own row of the table names all of its pages.
"""
from __future__ import annotations

import math

import torch

INT_MAX = 2 ** 31 - 1


def fork(cache, lens, table, parents, refs, new):
    """kv8_fork on CPU tensors: (lens, table, refs, lacking); the cache in place."""
    pages, page, (seqs, width) = refs.shape[0], cache[0].shape[2], table.shape
    rows = [[p if 0 <= p < pages else -1 for p in row] for row in table.tolist()]
    counts = refs.tolist()
    for row in rows:
        for p in row:
            if p >= 0:
                counts[p] -= 1
    out, out_lens, wanted, kept, lacking = [], [], [], set(), 0
    for c, a in enumerate(parents.tolist()):
        there = 0 <= a < seqs
        n = max(lens[a].item(), 0) if there else 0
        more = max(int(new[c]) if isinstance(new, torch.Tensor) else new, 0)
        row = [-1] * width
        for i in range(min(n // page, width)):
            row[i] = rows[a][i]
        part = n // page
        if n % page and part < width and rows[a][part] >= 0:
            if a in kept:
                wanted.append((c, part, rows[a][part]))
            else:
                row[part] = rows[a][part]
            kept.add(a)
        begin, end = -(-n // page), -(-(n + more) // page)
        wanted += [(c, i, -1) for i in range(begin, min(end, width))]
        lacking += max(end - max(begin, width), 0)
        for p in row:
            if p >= 0:
                counts[p] += 1
        out.append(row)
        out_lens.append(min(n + more, INT_MAX))
    free = [p for p, n in enumerate(counts) if n == 0]
    for k, (c, i, source) in enumerate(wanted):
        if k >= len(free):
            lacking += 1
            continue
        out[c][i] = free[k]
        counts[free[k]] += 1
        if source >= 0:
            for t in cache:
                raw = t.view(torch.uint8) if t.element_size() == 1 else t
                raw[free[k]] = raw[source]
    return (torch.tensor(out_lens, dtype=torch.int32), torch.tensor(out, dtype=torch.int32).view(len(out), width),
            torch.tensor(counts, dtype=torch.int32), torch.tensor([min(lacking, INT_MAX)], dtype=torch.int32))


def compact(cache, table, refs):
    """kv8_compact on CPU tensors: (table, refs, moved, live); the cache in place."""
    counts = refs.tolist()
    live = [p for p, n in enumerate(counts) if n > 0]
    holes = [p for p in range(len(live)) if counts[p] <= 0]
    moved = [p if n > 0 else -1 for p, n in enumerate(counts)]
    for p in live[len(live) - len(holes):]:
        moved[p] = holes[len([q for q in live if q < p and q >= len(live)])]
        for t in cache:
            raw = t.view(torch.uint8) if t.element_size() == 1 else t
            raw[moved[p]] = raw[p]
    now = [0] * len(counts)
    for p in live:
        now[moved[p]] = counts[p]
    rows = [[moved[p] if 0 <= p < len(counts) else -1 for p in row] for row in table.tolist()]
    return (torch.tensor(rows, dtype=torch.int32).view(table.shape), torch.tensor(now, dtype=torch.int32),
            torch.tensor(moved, dtype=torch.int32), torch.tensor([len(live)], dtype=torch.int32))


def rotary(x, positions, freqs, axis_of=None, adjacent=False, magnitude=1.0):
    """x [rows, heads, dim] turned, in 64 bits."""
    y, half = x.double().clone(), freqs.shape[0]
    pos = positions.view(-1, x.shape[0]).double()
    for i in range(half):
        axis = 0 if axis_of is None else axis_of[i].item()
        angle = (pos[axis] if 0 <= axis < pos.shape[0] else torch.zeros(x.shape[0]).double()) * freqs[i].double()
        c, s = (magnitude * angle.cos())[:, None], (magnitude * angle.sin())[:, None]
        a, b = (2 * i, 2 * i + 1) if adjacent else (i, i + half)
        u, v = x[..., a].double(), x[..., b].double()
        y[..., a], y[..., b] = u * c - v * s, v * c + u * s
    return y


def logprobs(logits, ids, top, scale=1.0):
    """(logp [rows, n], entropy [rows], top_logp, top_ids [rows, top]) in 64 bits; rows
    without NaN or +inf."""
    rows, vocab = logits.shape
    logp = torch.full(ids.shape, -math.inf, dtype=torch.float64)
    entropy = torch.zeros(rows, dtype=torch.float64)
    best, at = torch.full((rows, top), -math.inf, dtype=torch.float64), torch.zeros((rows, top), dtype=torch.int32)
    for r in range(rows):
        order = sorted(range(vocab), key=lambda i: (-logits[r, i].item(), i))[:top]
        at[r] = torch.tensor(order, dtype=torch.int32)
        most = logits[r].double().max()
        if most == -math.inf:
            continue
        z = (logits[r].double() - most) * scale         # (differences first: those of logits next to 1e38 matter)
        z = z - z.logsumexp(0)
        p = z.exp()
        entropy[r] = -(p * z)[p > 0].sum()
        best[r] = z[order]
        for i, t in enumerate(ids[r].tolist()):
            if 0 <= t < vocab:
                logp[r, i] = z[t]
    return logp, entropy, best, at

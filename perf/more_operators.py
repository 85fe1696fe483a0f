"""Performance cases of the operators that generate several continuations of a
prompt over the paged 8-bit cache.

A step of samples, beams or scored candidates runs, around an 8-bit attention
layer: the step's sequences are made from the last step's (``fork``: shared
pages are counted, a partly filled page is copied for all but one of its
children, pages of dropped sequences become free, new tokens get pages); their
queries and keys are rotated by positions of one or several axes (``rotary``);
attention reads a prefix that a group of sequences shares once for all of them
(``attn``); and the head's logits become the log probabilities of given
tokens, the entropy and the best alternatives (``logp``).  Between batches the
live pages move to the cache's front (``compact``).

``run`` computes each in elementary torch operations, or, with ``own``, makes
the calls that a user of the package makes.  A page holds ``page`` tokens of a
sequence; its keys are ``k[page][head][token][dim]``, its values
``v[page][head][dim][token]``.
"""
from __future__ import annotations

import math
import random

import torch

own = False

DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "fp8": 448.0}


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # One step of eight beams: some are dropped, some fork.
        dict(name="fork_beams", op="fork", seqs=8, children=8, ctx=700, new=1, spare=64, hkv=8, d=128, page=64,
             fmt="int8"),
        # Sixteen prompts fan out into sixteen samples each, in a large cache.
        dict(name="fork_samples", op="fork", seqs=16, children=256, ctx=4001, new=5, spare=6000, hkv=8, d=128,
             page=64, fmt="fp8"),
        # A small cache's live pages move to its front.
        dict(name="compact_small", op="compact", pages=99, live=50, seqs=4, hkv=4, d=64, page=16, fmt="fp8"),
        # A cache of 1 GB, half of it live.
        dict(name="compact_large", op="compact", pages=8191, live=4000, seqs=64, hkv=8, d=128, page=64, fmt="int8"),
        # Four samples of one short prompt: latency counts.
        dict(name="attn_few", op="attn", groups=1, seqs=4, qlen=1, prefix=1000, suffix=40, hq=16, hkv=4, d=128,
             page=32, fmt="int8", src="bf16"),
        # 32 samples of one document.
        dict(name="attn_samples", op="attn", groups=1, seqs=32, qlen=1, prefix=30001, suffix=500, hq=32, hkv=8, d=128,
             page=64, fmt="int8", src="bf16"),
        # Eight prompts with eight samples each, up to three drafted tokens, small pages and heads, fp16.
        dict(name="attn_groups", op="attn", groups=8, seqs=8, qlen=3, prefix=6000, suffix=300, hq=32, hkv=8, d=64,
             page=16, fmt="fp8", src="fp16"),
        # 64 samples behind a very long document.
        dict(name="attn_long", op="attn", groups=1, seqs=64, qlen=1, prefix=66313, suffix=1000, hq=32, hkv=8, d=128,
             page=128, fmt="fp8", src="bf16"),
        # The new tokens of 32 sequences at far positions.
        dict(name="rotary_step", op="rotary", rows=32, hq=32, hkv=8, d=128, rot=128, axes=1, far=1 << 20,
             adjacent=False, src="bf16"),
        # A prompt of frames: time, height and width.
        dict(name="rotary_frames", op="rotary", rows=20001, hq=32, hkv=8, d=128, rot=128, axes=3, far=4096,
             adjacent=False, src="bf16"),
        # The sampled tokens of 16 sequences, with the 20 best alternatives.
        dict(name="logp_step", op="logp", rows=16, vocab=131071, ids=1, top=20, scale=1.25, masked=False, src="fp32"),
        # All tokens of a prompt, odd vocabulary.
        dict(name="logp_prompt", op="logp", rows=3001, vocab=100003, ids=1, top=5, scale=1.0, masked=False, src="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["fork", "compact", "attn", "attn", "attn", "rotary", "logp", "logp"])
    src = rng.choice(["bf16", "bf16", "fp16"])
    if op == "rotary":
        d = rng.choice([64, 128, 128, 256])
        hkv = rng.choice([1, 2, 4, 8])
        hq = hkv * rng.choice([1, 2, 4, 7, 8])
        rot = d if rng.random() < 0.6 else rng.choice([d // 2, d // 4, d - 16])
        return dict(op=op, rows=min(_log(rng, 1, 32768), 100_000_000 // ((hq + hkv) * d)), hq=hq, hkv=hkv, d=d, rot=rot,
                    axes=rng.choice([1, 1, 2, 3, 4]), far=_log(rng, 1000, 1 << 22), adjacent=rng.random() < 0.3, src=src)
    if op == "logp":
        vocab = _log(rng, 1000, 260000)
        src = rng.choice(["bf16", "bf16", "fp16", "fp32", "fp32"])
        return dict(op=op, rows=min(_log(rng, 1, 8192), (150_000_000 if src == "fp32" else 300_000_000) // vocab),
                    vocab=vocab, ids=rng.choice([1, 1, 3]), top=rng.choice([0, 1, 5, 20, 32]),
                    scale=rng.choice([1.0, 1.0, 0.7, 1.6]), masked=rng.random() < 0.3, src=src)
    d = rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    fmt = rng.choice(["int8", "fp8"])
    size = hkv * page * d                            # bytes of a page's keys
    if op == "fork":
        seqs = _log(rng, 1, 128)
        children = min(_log(rng, 1, 512), max(1, 15_000_000 // size))
        ctx = max(1, min(_log(rng, 1, 8192), (400_000_000 // size - 1) * page // seqs))
        new = rng.choice([0, 1, 1, 5])
        # now and then fewer free pages than the step asks for
        spare = max(0, children * (2 + new // page) - 1) if rng.random() < 0.2 else _log(rng, 4 * children + 4, 4096)
        return dict(op=op, seqs=seqs, children=children, ctx=ctx, new=new,
                    spare=max(0, min(spare, 200_000_000 // size)), hkv=hkv, d=d, page=page, fmt=fmt)
    if op == "compact":
        pages = max(2, min(_log(rng, 8, 16384), 500_000_000 // size))
        return dict(op=op, pages=pages, live=max(1, int(pages * rng.uniform(0.05, 0.95))), seqs=_log(rng, 1, 64),
                    hkv=hkv, d=d, page=page, fmt=fmt)
    hq = hkv * rng.choice([1, 2, 4, 7, 8])
    groups = rng.choice([1, 1, 2, 5, 16])
    seqs = max(1, _log(rng, 1, 128) // groups)
    qlen = rng.choice([1, 1, 1, 4, _log(rng, 2, 64)])
    most = int(1.2e10 / (groups * seqs * qlen * hq * d))
    prefix = max(1, min(_log(rng, 64, 65536), most, (1 << 26) // (hkv * d) // groups))
    suffix = qlen + min(_log(rng, 1, 2000), most // 4, (1 << 25) // (hkv * d) // (groups * seqs))
    return dict(op=op, groups=groups, seqs=seqs, qlen=qlen, prefix=prefix, suffix=suffix, hq=hq, hkv=hkv, d=d,
                page=page, fmt=fmt, src=src)


# ----------------------------------------------------------------- inputs --

def _case_rng(case):
    """What a case leaves open and its work depends on, the same for every seed."""
    return random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))


def _fork_plan(case):
    """(lengths, prefix pages shared by groups of four sequences, parents)."""
    rng = _case_rng(case)
    lens = [case["ctx"]] + [max(1, int(case["ctx"] * rng.uniform(0.25, 1.0))) for _ in range(case["seqs"] - 1)]
    shared = [min(lens[b - b % 4:b - b % 4 + 4]) // case["page"] // 2 for b in range(case["seqs"])]
    if case["children"] > case["seqs"]:              # fan out, in order
        parents = [c * case["seqs"] // case["children"] for c in range(case["children"])]
    else:                                            # beams; now and then a finished one
        parents = [-1 if rng.random() < 0.05 else rng.randrange(case["seqs"]) for _ in range(case["children"])]
    return lens, shared, parents


def _attn_plan(case):
    """For each group its prefix, for each of its sequences (new tokens, tokens behind the prefix)."""
    rng = _case_rng(case)
    plan = []
    for i in range(case["groups"]):
        prefix = case["prefix"] if i == 0 else max(1, int(case["prefix"] * rng.uniform(0.25, 1.0)))
        behind = []
        for j in range(case["seqs"]):
            n = case["qlen"] if j == 0 else rng.randint(max(1, case["qlen"] // 2), case["qlen"])
            behind.append((n, case["suffix"] if j == 0 else max(n, int(case["suffix"] * rng.random()))))
        plan.append((prefix, behind))
    return plan


def _cache(case, pages, g, device):
    hkv, d, page, fmt = case["hkv"], case["d"], case["page"], case["fmt"]
    top = TOP[fmt]

    def codes(shape, channel):
        x = torch.empty(shape, device=device, dtype=torch.float16)
        x.normal_(generator=g)
        x.mul_(channel)
        x = x.mul_(top / 6).clamp_(-top, top)
        return x.round_().to(torch.int8) if fmt == "int8" else x.to(CODE[fmt])

    # a few channels are larger than the rest, as they are in keys
    channel = (1 + (torch.rand((hkv, 1, d), generator=g, device=device) < 0.03).half() * 2) * 0.8
    k = codes((pages, hkv, page, d), channel)
    v = codes((pages, hkv, d, page), 1.0)
    ks, vs = (torch.rand((pages, hkv), generator=g, device=device) * 0.5 + 0.75 for _ in range(2))
    return dict(k=k, v=v, k_scale=ks * (6 / top), v_scale=vs * (6 / top))


def _table(rows, pages, g, device):
    """The page table of sequences whose pages are numbered in turn, in any order in the cache."""
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    width = max(max(len(r) for r in rows), 1)
    at = torch.tensor([r + [-1] * (width - len(r)) for r in rows], device=device)
    return torch.where(at < 0, -1, order[at.clamp_min(0)]).to(torch.int32), order


def _counts(table, pages):
    held = table[table >= 0].long()
    return torch.zeros(pages, dtype=torch.int32, device=table.device).index_add_(
        0, held, torch.ones_like(held, dtype=torch.int32))


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(shape):
        return torch.randn(shape, generator=g, device=dev)

    def ints(x):
        return torch.tensor(x, dtype=torch.int32, device=dev)

    s = dict(case=case, op=case["op"])
    if case["op"] == "rotary":
        rows, hq, hkv, d, axes, rot = (case[n] for n in ("rows", "hq", "hkv", "d", "axes", "rot"))
        half = rot // 2
        # queries and keys lie in one projection's rows, beside the values
        qkv = (randn((rows, hq + 2 * hkv, d)) * 1.5).to(DT[case["src"]])
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
        pos = torch.randint(0, case["far"], (axes, rows), generator=g, device=dev)
        s["positions"] = pos[0] if axes == 1 else pos
        s["freqs"] = 10000.0 ** (-torch.arange(half, dtype=torch.float64, device=dev) / half)
        # the first axis has a quarter of the frequencies, the others share the rest
        cut = [half] if axes == 1 else [half // 4] + [(half - half // 4) // (axes - 1)] * (axes - 1)
        owner = [a for a, n in enumerate(cut) for _ in range(n)]
        s["axis_of"] = None if axes == 1 else ints(owner + [axes - 1] * (half - len(owner)))
        return s
    if case["op"] == "logp":
        rows, vocab = case["rows"], case["vocab"]
        x = randn((rows, vocab))
        x.mul_(1.5 + 1.5 * torch.rand((rows, 1), generator=g, device=dev))        # flat and sharp rows
        x = x.to(DT[case["src"]])
        best = torch.randint(0, vocab, (rows, 1), generator=g, device=dev)        # one likely token
        x.scatter_(1, best, torch.full((rows, 1), 14.0, dtype=x.dtype, device=dev))
        if case["masked"]:                           # a constrained step: most tokens are not allowed
            x.masked_fill_(torch.rand((1, vocab), generator=g, device=dev) < 0.9, -math.inf)
        s["logits"] = x
        ids = torch.randint(0, vocab, (rows, case["ids"]), generator=g, device=dev)
        ids[:, 0] = torch.where(torch.rand((rows,), generator=g, device=dev) < 0.5, best[:, 0], ids[:, 0])
        s["ids"] = ids.to(torch.int32)[:, 0].contiguous() if case["ids"] == 1 else ids.to(torch.int32)
        return s
    page = case["page"]
    if case["op"] == "fork":
        lens, shared, parents = _fork_plan(case)
        rows, at = [], 0
        for b, n in enumerate(lens):
            mine = -(-n // page)
            same = shared[b] if b % 4 else 0
            rows.append((rows[b - b % 4][:same] if same else []) + list(range(at, at + mine - same)))
            at += mine - same
        pages = at + case["spare"]
        width = -(-(max(lens) + case["new"]) // page)
        s["table"], _ = _table([r + [-1] * (width - len(r)) for r in rows], pages, g, dev)
        s["seq_lens"], s["parents"] = ints(lens), ints(parents)
        s["new"] = ints([case["new"]] * len(parents))
        s["refs"] = _counts(s["table"], pages)
        s["cache"] = _cache(case, pages, g, dev)
        return s
    if case["op"] == "compact":
        rng, pages = _case_rng(case), case["pages"]
        live = rng.sample(range(pages), case["live"])
        per = -(-len(live) // case["seqs"])
        rows = [live[b * per:(b + 1) * per] for b in range(case["seqs"])]
        width = max(len(r) for r in rows)
        table = [r + [-1] * (width - len(r)) for r in rows]
        for r in table[1::2]:                        # every other sequence shares its first pages with the one before
            same = [p for p in table[table.index(r) - 1][:width // 4] if p >= 0]
            r[:] = (same + [p for p in r if p >= 0])[:width] + [-1] * max(0, width - len(same) - sum(p >= 0 for p in r))
        s["table"] = ints(table)
        s["refs"] = _counts(s["table"], pages)
        # what no sequence holds any more is kept by its writer
        s["refs"][torch.tensor(live, device=dev)] += 1
        s["cache"] = _cache(case, pages, g, dev)
        return s
    plan = _attn_plan(case)
    rows, lens, new, starts, at = [], [], [], [0], 0
    for prefix, behind in plan:
        whole = prefix // page
        first = list(range(at, at + whole))
        at += whole
        for n, t in behind:
            mine = -(-(prefix + t) // page) - whole
            rows.append(first + list(range(at, at + mine)))
            at += mine
            lens.append(prefix + t)
            new.append(n)
        starts.append(len(lens))
    s["table"], _ = _table(rows, at + 3, g, dev)
    s["seq_lens"], s["group_starts"] = ints(lens), ints(starts)
    s["shared_lens"] = ints([p for p, _ in plan])
    s["q_starts"] = None if case["qlen"] == 1 else ints([0] + torch.tensor(new).cumsum(0).tolist())
    s["cache"] = _cache(case, at + 3, g, dev)
    s["q"] = (randn((sum(new), case["hq"], case["d"])) * 1.5).to(DT[case["src"]])
    return s


# ------------------------------------------------------------ plain forms --

def _plain_fork(s):
    cache, lens, table, refs = s["cache"], s["seq_lens"].long().clamp_min(0), s["table"].long(), s["refs"]
    page, (seqs, width), pages, dev = s["case"]["page"], table.shape, refs.shape[0], table.device
    parents, i = s["parents"].long(), torch.arange(width, device=dev)
    c = torch.arange(len(parents), device=dev)
    there = (parents >= 0) & (parents < seqs)
    a = parents.clamp(0, seqs - 1)
    n = torch.where(there, lens[a], 0)
    full = (n // page).clamp_max(width)
    first = torch.full((seqs,), len(parents), device=dev).scatter_reduce(
        0, a, torch.where(there, c, len(parents)), "amin")[a] == c
    row = table[a]
    row = torch.where((row >= 0) & (row < pages), row, -1)
    split = (n % page != 0) & (n // page < width) & (i == full[:, None]).logical_and(row >= 0).any(1)
    held = torch.where((i < full[:, None]) | ((i == full[:, None]) & (split & first)[:, None]), row, -1)
    copied = (split & ~first)[:, None] & (i == full[:, None])
    begin, end = -(-n // page), -(-(n + s["new"].long().clamp_min(0)) // page)
    fresh = copied | ((i >= begin[:, None]) & (i < end[:, None]))

    def count(entries):
        ok = (entries >= 0) & (entries < pages)
        return torch.zeros(pages, dtype=torch.int32, device=dev).index_add_(
            0, torch.where(ok, entries, 0).flatten(), ok.flatten().int())

    kept = refs - count(table) + count(held)
    free = torch.argsort((kept != 0).int(), stable=True)
    left = (kept == 0).sum()
    rank = fresh.flatten().long().cumsum(0).view_as(fresh) - 1
    given = fresh & (rank < left)
    out = torch.where(given, free[rank.clamp(0, pages - 1)], held)
    to = (given & copied).nonzero()
    source, target = row[to[:, 0], to[:, 1]], out[to[:, 0], to[:, 1]]
    for t in (cache["k"], cache["v"]):
        t.view(torch.uint8)[target] = t.view(torch.uint8)[source]
    for t in (cache["k_scale"], cache["v_scale"]):
        t[target] = t[source]
    wanted = copied.sum() + (end - begin).clamp_min(0).sum()
    refs = kept + count(torch.where(given, out, -1))
    return ((n + s["new"].long().clamp_min(0)).int(), out.int(), refs, (wanted - given.sum()).int().view(1),
            cache["k"], cache["v"], cache["k_scale"], cache["v_scale"])


def _plain_compact(s):
    cache, table, refs = s["cache"], s["table"].long(), s["refs"]
    pages = refs.shape[0]
    live = refs > 0
    n, p = live.sum(), torch.arange(pages, device=refs.device)
    holes, movers = (~live & (p < n)).nonzero()[:, 0], (live & (p >= n)).nonzero()[:, 0]
    moved = torch.where(live, p, -1)
    moved[movers] = holes
    ok = (table >= 0) & (table < pages)
    out = torch.where(ok, moved[table.clamp(0, pages - 1)], -1)
    for t in (cache["k"], cache["v"]):
        t.view(torch.uint8)[holes] = t.view(torch.uint8)[movers]
    for t in (cache["k_scale"], cache["v_scale"]):
        t[holes] = t[movers]
    now = torch.zeros_like(refs)
    now[moved[live]] = refs[live]
    return (out.int(), now, moved.int(), n.int().view(1),
            cache["k"], cache["v"], cache["k_scale"], cache["v_scale"])


def _values(cache, table):
    """Keys and values of the tables' pages in 32 bits, [..., heads, tokens, dim]."""
    pid = table.long().clamp_min(0)
    k = cache["k"].view(torch.uint8)[pid].view(cache["k"].dtype).float() * cache["k_scale"][pid][..., None, None]
    v = cache["v"].view(torch.uint8)[pid].view(cache["v"].dtype).float() * cache["v_scale"][pid][..., None, None]
    return k, v.transpose(-1, -2)


def _plain_attn(s):
    """Each group: scores of all its queries against the prefix, and of each
    sequence's against its own tokens behind it; one softmax over both."""
    c, cache, q, dev = s["case"], s["cache"], s["q"], s["q"].device
    hkv, d, page, gqa = c["hkv"], c["d"], c["page"], c["hq"] // c["hkv"]
    out, at, b = [], 0, 0
    for prefix, behind in _attn_plan(c):
        whole, seqs, most = prefix // page, len(behind), max(n for n, _ in behind)
        news, own_ = [n for n, _ in behind], [t + prefix % page for _, t in behind]
        rows = q[at:at + sum(news)].float()
        x = rows.view(-1, hkv, gqa, d).permute(1, 0, 2, 3).reshape(hkv, -1, d)           # [heads, rows * gqa, d]
        pk, pv = _values(cache, s["table"][b, :whole])
        pk, pv = (t.transpose(0, 1).reshape(hkv, whole * page, d) for t in (pk, pv))
        left = (x @ pk.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(hkv, sum(news), gqa, whole * page)
        wide = -(-max(own_) // page)
        part = s["table"][b:b + seqs, whole:whole + wide]
        sk, sv = _values(cache, part)
        sk, sv = (t.transpose(1, 2).reshape(seqs, hkv, -1, d) for t in (sk, sv))
        start = torch.tensor([0] + news, device=dev).cumsum(0)
        i = torch.arange(most, device=dev)
        n, t = torch.tensor(news, device=dev), torch.tensor(own_, device=dev)
        pick = (start[:-1, None] + i).clamp_max(sum(news) - 1)
        y = rows[pick].view(seqs, most, hkv, gqa, d).permute(0, 2, 1, 3, 4).reshape(seqs, hkv, most * gqa, d)
        right = (y @ sk.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(seqs, hkv, most, gqa, wide * page)
        j = torch.arange(wide * page, device=dev)
        seen = j <= (t - n)[:, None, None] + i[:, None]
        right.masked_fill_(~seen[:, None, :, None], -math.inf)
        who = torch.repeat_interleave(torch.arange(seqs, device=dev), n)
        nth = torch.arange(sum(news), device=dev) - start[who]
        right = right[who, :, nth].transpose(0, 1)                                       # [heads, rows, gqa, tokens]
        top = right.amax(-1, keepdim=True)
        if whole:
            top = torch.maximum(top, left.amax(-1, keepdim=True))
        left, right = left.sub_(top).exp_(), (right - top).exp_()
        total = left.sum(-1, keepdim=True) + right.sum(-1, keepdim=True)
        o = (left.view(hkv, sum(news) * gqa, whole * page) @ pv).view(hkv, -1, gqa, d)
        back = torch.zeros((seqs, hkv, most, gqa, wide * page), device=dev)
        back[who, :, nth] = right.transpose(0, 1)
        r = (back.view(seqs, hkv, most * gqa, -1) @ sv).view(seqs, hkv, most, gqa, d)
        o = (o + r[who, :, nth].transpose(0, 1)) / total
        out.append(o.permute(1, 0, 2, 3).reshape(-1, c["hq"], d).to(q.dtype))
        at, b = at + sum(news), b + seqs
    return torch.cat(out)


def _plain_rotary(s):
    c, half = s["case"], s["case"]["rot"] // 2
    pos = s["positions"].double().view(c["axes"], -1)
    angle = (pos[0][:, None] if s["axis_of"] is None else pos[s["axis_of"].long()].t()) * s["freqs"]
    cos, sin = angle.cos().float()[:, None], angle.sin().float()[:, None]

    def turned(x):
        y = x.float()
        if c["adjacent"]:
            a, b = y[..., 0:2 * half:2], y[..., 1:2 * half:2]
        else:
            a, b = y[..., :half], y[..., half:2 * half]
        a, b = a * cos - b * sin, b * cos + a * sin
        pair = torch.stack((a, b), -1).flatten(-2) if c["adjacent"] else torch.cat((a, b), -1)
        return torch.cat((pair, y[..., 2 * half:]), -1).to(x.dtype)

    return turned(s["q"]), turned(s["k"])


def _plain_logp(s):
    c, x = s["case"], s["logits"].float()
    ids = s["ids"].long().view(c["rows"], -1)
    z = x * c["scale"]
    top = z.amax(1, keepdim=True)
    z -= top
    e = z.exp()
    total = e.sum(1, keepdim=True, dtype=torch.float64)              # long sums
    logp = (z.gather(1, ids).double() - total.log()).float()
    ze = e.mul_(z).nan_to_num_(0.0)                                  # (a masked token has no part in it)
    entropy = (total.log() - ze.sum(1, keepdim=True, dtype=torch.float64) / total)[:, 0].float()
    if c["ids"] == 1:
        logp = logp[:, 0]
    if c["top"] == 0:
        return logp, entropy
    del e, ze
    # ties by index: keys of the value's order, then the index from the last on
    bits = (x + 0.0).view(torch.int32).long()
    bits = torch.where(bits < 0, -(bits & 0x7fffffff), bits)
    keys = bits * (1 << 31) + (c["vocab"] - 1 - torch.arange(c["vocab"], device=x.device))
    at = c["vocab"] - 1 - keys.topk(c["top"], 1).values % (1 << 31)
    return logp, entropy, (z.gather(1, at).double() - total.log()).float(), at.int()


# -------------------------------------------------------------------- run --

def run(s):
    if own:
        return _own(s, s["case"])
    return {"fork": _plain_fork, "compact": _plain_compact, "attn": _plain_attn, "rotary": _plain_rotary,
            "logp": _plain_logp}[s["op"]](s)


def _own(s, c):
    from dsl_tool_amd import attention, kvcache, logprobs, rotary
    if c["op"] == "rotary":
        return rotary.rotary(s["q"], s["k"], s["positions"], s["freqs"], axis_of=s["axis_of"], adjacent=c["adjacent"])
    if c["op"] == "logp":
        r = logprobs.token_logprobs(s["logits"], s["ids"], top=c["top"], scale=c["scale"])
        return tuple(r)[:4 if c["top"] else 2]
    t = s["cache"]
    cache = kvcache.KV8Cache(t["k"], t["v"], t["k_scale"], t["v_scale"])
    if c["op"] == "fork":
        return tuple(kvcache.kv8_fork(cache, s["seq_lens"], s["table"], s["parents"], s["refs"], new=s["new"])) + tuple(cache)
    if c["op"] == "compact":
        return tuple(kvcache.kv8_compact(cache, s["table"], s["refs"])) + tuple(cache)
    return attention.kv8_shared_attention(s["q"], cache, s["seq_lens"], s["table"], s["group_starts"], s["shared_lens"],
                                          q_starts=s["q_starts"], max_q_len=c["qlen"], max_group=c["seqs"])


# ------------------------------------------------------------------- work --

def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "rotary":
        n = case["rows"] * (case["hq"] + case["hkv"]) * case["d"]
        return {"bytes": 2 * n * size[case["src"]] + 8 * case["axes"] * case["rows"] + 4 * case["rot"], "flops": 3 * n}
    if case["op"] == "logp":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * size[case["src"]] + case["rows"] * (8 * case["ids"] + 4 + 8 * case["top"]), "flops": 6 * n}
    hkv, d, page = case["hkv"], case["d"], case["page"]
    of_page = 2 * hkv * d * page + 8 * hkv
    if case["op"] == "fork":
        lens, shared, parents = _fork_plan(case)
        held = [a for a in parents if a >= 0]
        copies = sum(lens[a] % page != 0 for a in held) - sum(lens[a] % page != 0 for a in set(held))
        entries = -(-(max(lens) + case["new"]) // page)
        pages = sum(-(-n // page) - (m if b % 4 else 0) for b, (n, m) in enumerate(zip(lens, shared))) + case["spare"]
        return {"bytes": 4 * entries * (len(lens) + len(parents)) + 8 * pages + 4 * (len(lens) + 3 * len(parents)) +
                2 * of_page * min(copies, pages), "flops": 0}
    if case["op"] == "compact":
        live = _case_rng(case).sample(range(case["pages"]), case["live"])
        entries = case["seqs"] * -(-case["live"] // case["seqs"])
        return {"bytes": 8 * entries + 12 * case["pages"] + 2 * of_page * sum(p >= case["live"] for p in live),
                "flops": 0}
    tokens = pairs = rows = pages = 0
    for prefix, behind in _attn_plan(case):
        tokens += prefix // page * page
        pages += prefix // page
        for n, t in behind:
            rows += n
            tokens += t + prefix % page
            pages += -(-(t + prefix % page) // page)
            pairs += n * (prefix + t) - n * (n - 1) // 2
    return {"bytes": 2 * hkv * d * tokens + pages * (8 * hkv + 4) + 2 * case["hq"] * d * rows * size[case["src"]],
            "flops": 4 * case["hq"] * d * pairs}


# ------------------------------------------------------------------ exact --

def _exact_fork(case, s):
    """The bookkeeping by loops; the cache's codes and scales as they then stand."""
    page, dev = case["page"], s["refs"].device
    lens, table, refs, parents = (s[n].tolist() for n in ("seq_lens", "table", "refs", "parents"))
    width, seen, wants, rows, out_lens = len(table[0]), set(), [], [], []
    for row in table:
        for p in row:
            if p >= 0:
                refs[p] -= 1
    lacking = 0
    for c, (a, m) in enumerate(zip(parents, s["new"].tolist())):
        n = lens[a] if a >= 0 else 0
        row = [-1] * width
        for i in range(min(n // page, width)):
            row[i] = table[a][i]
        i = n // page
        if n % page and i < width and table[a][i] >= 0:
            if a in seen:
                wants.append((c, i, table[a][i]))
            else:
                row[i] = table[a][i]
            seen.add(a)
        for i in range(-(-n // page), -(-(n + m) // page)):
            if i < width:
                wants.append((c, i, None))
            else:
                lacking += 1
        for p in row:
            if p >= 0:
                refs[p] += 1
        rows.append(row)
        out_lens.append(n + m)
    free = [p for p, r in enumerate(refs) if r == 0]
    cache = {n: t.clone() for n, t in s["cache"].items()}
    for k, (c, i, source) in enumerate(wants):
        if k >= len(free):
            lacking += 1
            continue
        rows[c][i] = free[k]
        refs[free[k]] += 1
        if source is not None:
            for t in cache.values():
                t[free[k]] = t[source]
    return (torch.tensor(out_lens, dtype=torch.int32, device=dev), torch.tensor(rows, dtype=torch.int32, device=dev),
            torch.tensor(refs, dtype=torch.int32, device=dev), torch.tensor([lacking], dtype=torch.int32, device=dev),
            cache["k"], cache["v"], cache["k_scale"], cache["v_scale"])


def _exact_compact(case, s):
    refs, dev = s["refs"].tolist(), s["refs"].device
    live = [p for p, r in enumerate(refs) if r > 0]
    holes = [p for p in range(len(live)) if refs[p] <= 0]
    moved = [p if r > 0 else -1 for p, r in enumerate(refs)]
    for p in live:
        if p >= len(live):
            moved[p] = holes.pop(0)
    now = [0] * len(refs)
    for p in live:
        now[moved[p]] = refs[p]
    table = [[moved[p] if p >= 0 else -1 for p in row] for row in s["table"].tolist()]
    cache = {n: t.clone() for n, t in s["cache"].items()}
    source = torch.tensor(live, device=dev)
    target = torch.tensor([moved[p] for p in live], device=dev)
    for n, t in cache.items():
        raw, old = (t.view(torch.uint8), s["cache"][n].view(torch.uint8)) if t.element_size() == 1 else (t, s["cache"][n])
        raw[target] = old[source]
    ints = [torch.tensor(x, dtype=torch.int32, device=dev) for x in (table, now, moved, [len(live)])]
    return (*ints, cache["k"], cache["v"], cache["k_scale"], cache["v_scale"])


def _exact_attn(case, s):
    """Sequence by sequence over its whole context, as its own row of the table has it."""
    cache, page, fmt, out, at, b = s["cache"], case["page"], case["fmt"], [], 0, 0
    gqa = case["hq"] // case["hkv"]
    ks, vs = cache["k_scale"].double(), cache["v_scale"].double()
    for prefix, behind in _attn_plan(case):
        for n, t in behind:
            t += prefix
            pid = s["table"][b, :-(-t // page)].long()
            heads = []
            for h in range(case["hkv"]):
                k = cache["k"].view(torch.uint8)[pid, h].view(CODE[fmt]).double() * ks[pid, h][:, None, None]
                v = cache["v"].view(torch.uint8)[pid, h].view(CODE[fmt]).double() * vs[pid, h][:, None, None]
                k, v = k.flatten(0, 1)[:t], v.transpose(1, 2).flatten(0, 1)[:t]
                q = s["q"][at:at + n, h * gqa:(h + 1) * gqa].double().transpose(0, 1)
                z = q.reshape(-1, case["d"]) @ k.t() / math.sqrt(case["d"])
                hidden = torch.ones((n, t), dtype=torch.bool, device=z.device).triu(t - n + 1)
                p = z.view(gqa, n, t).masked_fill(hidden, -math.inf).softmax(-1)
                heads.append((p.view(-1, t) @ v).view(gqa, n, -1))
            out.append(torch.cat(heads).transpose(0, 1))
            at, b = at + n, b + 1
    return torch.cat(out)


def _exact_rotary(case, s):
    half = case["rot"] // 2
    pos = s["positions"].view(case["axes"], -1)
    angle = torch.zeros((pos.shape[1], half), dtype=torch.float64, device=pos.device)
    for i in range(half):
        axis = 0 if s["axis_of"] is None else int(s["axis_of"][i])
        angle[:, i] = pos[axis].double() * float(s["freqs"][i])
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]
    out = []
    for x in (s["q"], s["k"]):
        y = x.double().clone()
        first, second = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if case["adjacent"] else (slice(0, half), slice(half, 2 * half))
        z = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn
        y[..., first], y[..., second] = z.real, z.imag
        out.append(y)
    return tuple(out)


def _exact_logp(case, s):
    logp, entropy, best, at = [], [], [], []
    for r in range(0, case["rows"], 64):
        x = s["logits"][r:r + 64].double()
        z = (x * case["scale"]).log_softmax(1)
        p = z.exp()
        entropy.append(-(p * z).where(p > 0, 0.0).sum(1))
        logp.append(z.gather(1, s["ids"].long().view(case["rows"], -1)[r:r + 64]))
        if case["top"]:
            order = x.sort(dim=1, descending=True, stable=True).indices[:, :case["top"]]
            at.append(order.int())
            best.append(z.gather(1, order))
    logp = torch.cat(logp)
    first = (logp[:, 0] if case["ids"] == 1 else logp), torch.cat(entropy)
    return first if not case["top"] else (*first, torch.cat(best), torch.cat(at))


def exact(case, seed):
    return {"fork": _exact_fork, "compact": _exact_compact, "attn": _exact_attn, "rotary": _exact_rotary,
            "logp": _exact_logp}[case["op"]](case, prepare(case, seed))

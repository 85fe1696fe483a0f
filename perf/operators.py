"""Performance cases of the operators of an 8-bit attention layer.

A decoder layer served in 8 bits runs, around its attention: the residual's
addition with the RMS norm and an 8-bit result (``norm``); the projections as
products of 8-bit integers with a scale for each token and each channel
(``int8``); the new keys and values quantised into a paged cache with one
scale for each page and head (``write``), and read back where a prefix is
needed in 16 bits (``read``); and attention over that cache (``attn``), for
single new tokens and for prompts.

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
TOP = {"int8": 127.0, "fp8": 448.0, "fp8_row": 448.0}
FLOOR = 1e-12            # the smallest scale
EPS = 1e-6


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # The norm in front of a block-scaled FP8 projection, one decode step
        # of a batch of 16: E4M3 codes, a scale for each 128 columns.
        dict(name="norm_decode", op="norm", rows=16, cols=4096, fmt="fp8", src="bf16", weight="bf16"),
        # The same over a prompt of an odd number of tokens, fp16, one scale
        # for each token.
        dict(name="norm_prefill", op="norm", rows=3001, cols=7168, fmt="fp8_row", src="fp16", weight="fp32"),
        # A projection of 16 tokens by int8 weights: the weights' bytes.
        dict(name="int8_decode", op="int8", m=16, n=7168, k=4096, out="bf16"),
        # The same over a prompt whose length is no whole tile.
        dict(name="int8_prefill", op="int8", m=4001, n=7168, k=4096, out="bf16"),
        # One new token for each of 64 sequences goes into half-filled pages.
        dict(name="write_decode", op="write", seqs=64, qlen=1, ctx=2048, hkv=8, d=128, page=64, fmt="fp8",
             src="bf16"),
        # Prompts of about 2000 tokens, behind a few that are in the cache.
        dict(name="write_prefill", op="write", seqs=4, qlen=2000, ctx=2100, hkv=8, d=128, page=64, fmt="fp8",
             src="bf16"),
        # The cached prefixes of eight sequences, back in bf16.
        dict(name="read_prefixes", op="read", seqs=8, ctx=8192, hkv=8, d=128, page=16, fmt="int8", src="bf16"),
        # One short prefix, small pages and heads.
        dict(name="read_one", op="read", seqs=1, ctx=777, hkv=4, d=64, page=32, fmt="fp8", src="fp16"),
        # The next token of one conversation: latency counts.
        dict(name="attn_decode_one", op="attn", seqs=1, qlen=1, ctx=5001, hq=32, hkv=8, d=128, page=64, fmt="int8",
             src="bf16"),
        # The next token of 64 of them, small pages: the cache's bytes.
        dict(name="attn_decode_batch", op="attn", seqs=64, qlen=1, ctx=8192, hq=32, hkv=8, d=128, page=16,
             fmt="int8", src="bf16"),
        # Two long documents, fp16 over an E4M3 cache.
        dict(name="attn_decode_long", op="attn", seqs=2, qlen=1, ctx=131072, hq=64, hkv=8, d=128, page=128,
             fmt="fp8", src="fp16"),
        # Two prompts in one call, each behind a cached prefix.
        dict(name="attn_prefill", op="attn", seqs=2, qlen=3600, ctx=4600, hq=32, hkv=8, d=128, page=64, fmt="fp8",
             src="bf16"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng, lo, hi, step):
    """A dimension: whole 128s mostly, else any multiple of `step`."""
    s = 128 if rng.random() < 0.6 else step
    return max(s, _log(rng, lo, hi) // s * s)


def draw(rng):
    op = rng.choice(["norm", "int8", "int8", "write", "read", "attn", "attn", "attn"])
    if op == "norm":
        cols = _width(rng, 256, 16384, 8)
        return dict(op=op, rows=min(_log(rng, 1, 8192), (1 << 25) // cols), cols=cols,
                    fmt=rng.choice(["int8", "fp8", "fp8_row"]), src=rng.choice(["bf16", "bf16", "fp16"]),
                    weight=rng.choice(["bf16", "fp32"]))
    if op == "int8":
        n = _width(rng, 256, 16384, rng.choice([8, 1]))
        k = _width(rng, 256, 16384, 16)
        m = min(_log(rng, 1, 8192), int(2.3e11 / (2 * n * k)), (1 << 26) // max(n, k))
        return dict(op=op, m=max(1, m), n=n, k=k, out=rng.choice(["bf16", "bf16", "fp32"]))
    d = rng.choice([64, 128, 128, 256])
    hkv = rng.choice([1, 2, 4, 8])
    page = rng.choice([16, 32, 64, 128])
    fmt, src = rng.choice(["int8", "fp8"]), rng.choice(["bf16", "bf16", "fp16"])
    most = (1 << 28) // (hkv * d)                    # tokens in the cache
    if op == "write":
        seqs = _log(rng, 1, 64)
        qlen = 1 if rng.random() < 0.5 else _log(rng, 2, 4096)
        qlen = max(1, min(qlen, (1 << 23) // (seqs * hkv * d)))
        ctx = min(qlen + _log(rng, 1, 2048), max(qlen, most // 4 // seqs))
        return dict(op=op, seqs=seqs, qlen=qlen, ctx=ctx, hkv=hkv, d=d, page=page, fmt=fmt, src=src)
    if op == "read":
        seqs = _log(rng, 1, 32)
        return dict(op=op, seqs=seqs, ctx=max(1, min(_log(rng, 16, 16384), most // 4 // seqs)), hkv=hkv, d=d,
                    page=page, fmt=fmt, src=src)
    hq = hkv * rng.choice([1, 2, 4, 7, 8])
    if rng.random() < 0.6:                           # decode, or a few drafted tokens
        seqs = _log(rng, 1, 64)
        ctx = max(16, min(_log(rng, 16, 65536), most // seqs))
        qlen = rng.choice([1, 1, 1, 4])
    else:
        seqs = rng.choice([1, 2, 4])
        qlen = _log(rng, 16, 4096)
        ctx = qlen + (0 if rng.random() < 0.4 else _log(rng, 1, 2048))
        over = seqs * hq * qlen * ctx * d / 128 / 4.5e8
        if over > 1:
            qlen, ctx = max(1, int(qlen / math.sqrt(over))), max(1, int(ctx / math.sqrt(over)))
    return dict(op=op, seqs=seqs, qlen=min(qlen, ctx), ctx=ctx, hq=hq, hkv=hkv, d=d, page=page, fmt=fmt, src=src)


# ----------------------------------------------------------------- inputs --

def _lens(case):
    """(new tokens, tokens in all) of each sequence, the same for every seed:
    the first is as long as the case says, the others up to 3/4 shorter
    (single new tokens stay single)."""
    rng = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    qlen = case.get("qlen", 0)
    new, total = [qlen], [case["ctx"]]
    for _ in range(case["seqs"] - 1):
        share = rng.uniform(0.25, 1.0)
        new.append(qlen if qlen <= 4 else max(1, int(qlen * share)))
        total.append(max(new[-1], 1, int(case["ctx"] * share)))
    return new, total


def _starts(lens, device):
    return torch.tensor([0] + lens, dtype=torch.int64).cumsum(0).to(torch.int32).to(device)


def _cache(case, total, g, device):
    """A paged cache whose pages lie in any order: codes, scales, and the
    table of each sequence's pages."""
    hkv, d, page, fmt = case["hkv"], case["d"], case["page"], case["fmt"]
    need = [-(-n // page) for n in total]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=device).to(torch.int32)
    table = torch.zeros((len(total), max(need)), dtype=torch.int32, device=device)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n

    def codes(shape, channel):
        x = torch.empty(shape, device=device, dtype=torch.float16)
        x.normal_(generator=g)
        x.mul_(channel)
        top = TOP[fmt]
        x = x.mul_(top / 6).clamp_(-top, top)
        return x.round_().to(torch.int8) if fmt == "int8" else x.to(CODE[fmt])

    # a few channels are larger than the rest, as they are in keys
    channel = (1 + (torch.rand((hkv, 1, d), generator=g, device=device) < 0.03).half() * 2) * 0.8
    k = codes((pages, hkv, page, d), channel)
    v = codes((pages, hkv, d, page), 1.0)
    ks, vs = (torch.rand((pages, hkv), generator=g, device=device) * 0.5 + 0.75 for _ in range(2))
    return dict(k=k, v=v, k_scale=ks * (6 / TOP[fmt]), v_scale=vs * (6 / TOP[fmt]), table=table)


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev).manual_seed(seed)

    def randn(shape, dtype=torch.float32):
        return torch.randn(shape, generator=g, device=dev, dtype=torch.float32).to(dtype)

    s = dict(case=case, op=case["op"])
    if case["op"] == "norm":
        rows, cols, dt = case["rows"], case["cols"], DT[case["src"]]
        s["x"] = randn((rows, cols), dt)
        heavy = 1 + (torch.rand((cols,), generator=g, device=dev) < 0.01).float() * 20   # outlier channels
        s["residual"] = (randn((rows, cols)) * 2 * heavy).to(dt)
        s["weight"] = (1 + 0.2 * randn((cols,))).to(DT[case["weight"]])
        return s
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        s["qa"] = (randn((m, k)) * 30).round_().clamp_(-127, 127).to(torch.int8)
        s["qw"] = (randn((n, k)) * 32).round_().clamp_(-127, 127).to(torch.int8)
        s["sa"] = torch.rand((m,), generator=g, device=dev) * 0.05 + 0.01
        s["sw"] = torch.rand((n,), generator=g, device=dev) * 1e-3 + 1e-4
        return s
    new, total = _lens(case)
    s["cache"] = _cache(case, total, g, dev)
    s["seq_lens"] = torch.tensor(total, dtype=torch.int32, device=dev)
    if case["op"] == "read":
        s["starts"], s["total"] = _starts(total, dev), sum(total)
        return s
    s["q_starts"] = None if case["qlen"] == 1 else _starts(new, dev)
    hq, hkv, d, dt, rows = case.get("hq", 0), case["hkv"], case["d"], DT[case["src"]], sum(new)
    if case["op"] == "write":
        # keys and values lie in one projection's rows, beside the queries
        qkv = randn((rows, 3 * hkv, d))
        qkv[:, :, ::31] *= 3
        qkv = qkv.to(dt)
        s["k_new"], s["v_new"] = qkv[:, hkv:2 * hkv], qkv[:, 2 * hkv:]
        return s
    s["q"] = (randn((rows, hq, d)) * 1.5).to(dt)
    return s


# ------------------------------------------------------------ plain forms --

def _div(x, top):
    """x / top, rounded once (a number as divisor would be a product)."""
    return x / torch.full((), top, dtype=x.dtype, device=x.device)


def _encode(x, scale, fmt):
    y = x / scale
    return y.round().clamp_(-127, 127).to(torch.int8) if fmt == "int8" else y.to(torch.float8_e4m3fn)


def _plain_norm(s):
    c = s["case"]
    fmt = c["fmt"]
    h = s["x"].float() + s["residual"].float()
    y = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["weight"].float()
    rows, cols = y.shape
    group = 128 if fmt == "fp8" else cols
    pad = -cols % group
    yg = torch.nn.functional.pad(y, (0, pad)).view(rows, -1, group)
    scale = _div(yg.abs().amax(-1), TOP[fmt]).clamp_min(FLOOR)
    q = _encode(yg, scale[..., None], "int8" if fmt == "int8" else "fp8").view(rows, -1)[:, :cols]
    return q, (scale if fmt == "fp8" else scale[:, 0]), h.to(s["x"].dtype)


def _plain_int8(s):
    # a sum of products of codes passes 24 bits: in 64
    acc = s["qa"].double() @ s["qw"].double().t()
    return (acc * s["sa"].double()[:, None] * s["sw"].double()).to(DT[s["case"]["out"]])


def _queries(s):
    """Row numbers [sequences, most new tokens] of the new tokens, which of
    them there are, and their positions."""
    c, lens = s["case"], s["seq_lens"].long()
    dev = lens.device
    i = torch.arange(c["qlen"], device=dev)
    if s["q_starts"] is None:
        starts, n = torch.arange(c["seqs"], device=dev), torch.ones_like(lens)
    else:
        starts = s["q_starts"][:-1].long()
        n = s["q_starts"][1:].long() - starts
    there = i < n[:, None]
    return (starts[:, None] + i).where(there, 0), there, (lens - n)[:, None] + i, starts, n


def _plain_write(s):
    c, cache, lens = s["case"], s["cache"], s["seq_lens"].long()
    fmt, page = c["fmt"], c["page"]
    dev = lens.device
    _, _, _, starts, n = _queries(s)
    first = lens - n                                        # position of the first new token
    # the pages that new tokens touch: `span` from the first one's on
    span = (c["qlen"] + page - 2) // page + 1
    number = first[:, None] // page + torch.arange(span, device=dev)
    live = number * page < lens[:, None]
    pid = cache["table"].long().gather(1, number.clamp_max(cache["table"].shape[1] - 1))
    pos = number[..., None] * page + torch.arange(page, device=dev)
    fresh = (pos >= first[:, None, None]) & (pos < lens[:, None, None])
    older = (pos < first[:, None, None])[:, :, None, :, None]
    row = (starts[:, None, None] + pos - first[:, None, None]).where(fresh, 0)
    b, p = live.nonzero(as_tuple=True)
    pid, fresh, older, row = pid[b, p], fresh[b, p][:, None, :, None], older[b, p], row[b, p]

    def put(codes, scales, new, turned):
        raw = codes.view(torch.uint8)
        old = raw[pid].view(codes.dtype).float()
        old = old.transpose(-1, -2) if turned else old
        x = new[row].float().transpose(1, 2).where(fresh, 0.0)
        kept = scales[pid].where(older.flatten(1).any(1)[:, None], 0.0)
        scale = torch.maximum(kept, _div(x.abs().amax((-1, -2)), TOP[fmt]).clamp_min(FLOOR))[..., None, None]
        # old codes move to the larger scale; places past the end stay
        moved = _encode(old * kept[..., None, None], scale, fmt).float()
        out = torch.where(fresh, _encode(x, scale, fmt).float(), torch.where(older, moved, old))
        out = (out.transpose(-1, -2) if turned else out).to(codes.dtype).contiguous()
        raw[pid] = out.view(torch.uint8)
        scales[pid] = scale[..., 0, 0]

    put(cache["k"], cache["k_scale"], s["k_new"], False)
    put(cache["v"], cache["v_scale"], s["v_new"], True)
    return _cache_values(cache)


def _cache_values(cache):
    """The cache's buffers; codes as numbers of a floating type."""
    k, v = cache["k"], cache["v"]
    if k.dtype == torch.int8:
        k, v = k.to(torch.bfloat16), v.to(torch.bfloat16)
    return k, v, cache["k_scale"], cache["v_scale"]


def _values(cache, table):
    """Keys and values of the tables' pages in 32 bits, [..., heads, tokens, dim]."""
    pid = table.long()
    k = cache["k"].view(torch.uint8)[pid].view(cache["k"].dtype).float() * cache["k_scale"][pid][..., None, None]
    v = cache["v"].view(torch.uint8)[pid].view(cache["v"].dtype).float() * cache["v_scale"][pid][..., None, None]
    return k, v.transpose(-1, -2)


def _plain_read(s):
    c, cache = s["case"], s["cache"]
    dt, page = DT[c["src"]], c["page"]
    t = torch.arange(s["total"], device=s["starts"].device)
    b = torch.searchsorted(s["starts"][1:].long(), t, right=True)
    pos = t - s["starts"].long()[b]
    pid, at = cache["table"].long()[b, pos // page], pos % page
    k = cache["k"].view(torch.uint8)[pid, :, at].view(cache["k"].dtype).float() * cache["k_scale"][pid][..., None]
    v = cache["v"].view(torch.uint8)[pid, :, :, at].view(cache["v"].dtype).float() * cache["v_scale"][pid][..., None]
    return k.to(dt), v.to(dt)


def _plain_attn(s):
    c, cache, q = s["case"], s["cache"], s["q"]
    hkv, d, lens = c["hkv"], c["d"], s["seq_lens"].long()
    row, there, pos, starts, _ = _queries(s)
    seqs, most = row.shape
    k, v = _values(cache, cache["table"])                   # [seqs, pages, heads, page, dim]
    k, v = (x.transpose(1, 2).reshape(seqs, hkv, -1, d) for x in (k, v))
    x = q[row].float().view(seqs, most, hkv, -1, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, -1, d)
    score = (x @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(seqs, hkv, -1, most, k.shape[2])
    j = torch.arange(k.shape[2], device=q.device)
    seen = (j <= pos[..., None]) & (j < lens[:, None, None])
    score.masked_fill_(~seen[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True).clamp_min(torch.finfo(torch.float32).min)
    p = score.sub_(top).exp_().view(seqs, hkv, -1, k.shape[2])
    total = p.sum(-1, keepdim=True)
    o = (p @ v) / total.clamp_min(1e-30)
    o = o.view(seqs, hkv, -1, most, d).permute(0, 3, 1, 2, 4).reshape(seqs, most, -1, d)
    t = torch.arange(q.shape[0], device=q.device)
    b = torch.searchsorted(starts, t, right=True) - 1
    return o[b, t - starts[b]].to(q.dtype)


# -------------------------------------------------------------------- run --

def run(s):
    c = s["case"]
    if own:
        return _own(s, c)
    return {"norm": _returned_norm, "int8": _plain_int8, "write": _plain_write, "read": _plain_read,
            "attn": _plain_attn}[s["op"]](s)


def _returned_norm(s):
    q, scale, h = _plain_norm(s)
    return (q.to(torch.bfloat16) if q.dtype == torch.int8 else q), scale, h


def _own(s, c):
    from dsl_tool_amd import attention, fused, gemm, kvcache
    if c["op"] == "norm":
        q, scale, h = fused.add_rmsnorm_quant(s["x"], s["residual"], s["weight"], EPS, fmt=c["fmt"])
        return (q.to(torch.bfloat16) if c["fmt"] == "int8" else q.view(torch.float8_e4m3fn)), scale, h
    if c["op"] == "int8":
        return gemm.int8_gemm_packed(s["qa"], s["qw"], s["sa"], s["sw"], out_dtype=DT[c["out"]])
    t = s["cache"]
    cache = kvcache.KV8Cache(t["k"], t["v"], t["k_scale"], t["v_scale"])
    if c["op"] == "write":
        kvcache.kv8_write(cache, s["k_new"], s["v_new"], s["seq_lens"], t["table"], q_starts=s["q_starts"],
                          max_q_len=c["qlen"])
        return _cache_values(t)
    if c["op"] == "read":
        return kvcache.kv8_read(cache, s["seq_lens"], t["table"], s["starts"], s["total"], dtype=DT[c["src"]])
    return attention.kv8_attention(s["q"], cache, s["seq_lens"], t["table"], q_starts=s["q_starts"],
                                   max_q_len=c["qlen"])


# ------------------------------------------------------------------- work --

def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "norm":
        rows, cols, e = case["rows"], case["cols"], size[case["src"]]
        scales = rows * (-(-cols // 128) if case["fmt"] == "fp8" else 1) * 4
        return {"bytes": rows * cols * (3 * e + 1) + scales + cols * size[case["weight"]], "flops": 8 * rows * cols}
    if case["op"] == "int8":
        m, n, k = case["m"], case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * (m + n) + m * n * size[case["out"]], "flops": 2 * m * n * k}
    new, total = _lens(case)
    hkv, d, page, e = case["hkv"], case["d"], case["page"], size[case["src"]]
    pages = sum(-(-n // page) for n in total)
    held = 2 * hkv * d * sum(total) + pages * (8 * hkv + 4)
    if case["op"] == "write":
        touched = sum((t - 1) // page - (t - n) // page + 1 for n, t in zip(new, total))
        return {"bytes": 2 * hkv * d * sum(new) * (e + 1) + touched * (8 * hkv + 4), "flops": 4 * hkv * d * sum(new)}
    if case["op"] == "read":
        return {"bytes": held + 2 * hkv * d * sum(total) * e, "flops": 2 * hkv * d * sum(total)}
    hq = case["hq"]
    pairs = sum(n * t - n * (n - 1) // 2 for n, t in zip(new, total))
    return {"bytes": held + 2 * hq * d * sum(new) * e, "flops": 4 * hq * d * pairs}


# ------------------------------------------------------------------ exact --

def _e4m3(x):
    """The nearest E4M3 value (ties to even), in 64 bits."""
    e = torch.frexp(x)[1].clamp_min(-5) - 4                # 3 bits behind the point
    return torch.ldexp(torch.ldexp(x, -e).round(), e)


def _nearest(x, fmt):
    return x.round() if fmt == "int8" else _e4m3(x)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        fmt = case["fmt"]
        h = s["x"].double() + s["residual"].double()
        y = h / (h.pow(2).sum(1, keepdim=True) / h.shape[1] + EPS).sqrt() * s["weight"].double()
        q, scales = torch.empty_like(y), []
        step = 128 if fmt == "fp8" else y.shape[1]
        for at in range(0, y.shape[1], step):
            part = y[:, at:at + step]
            scales.append((part.abs().max(1).values / TOP[fmt]).clamp_min(FLOOR))
            q[:, at:at + step] = _nearest(part / scales[-1][:, None], "int8" if fmt == "int8" else "fp8")
        return q, torch.stack(scales, 1) if fmt == "fp8" else scales[0], h
    if case["op"] == "int8":
        a, w = s["qa"].double() * s["sa"].double()[:, None], s["qw"].double() * s["sw"].double()[:, None]
        return torch.cat([a @ w[at:at + 2048].t() for at in range(0, w.shape[0], 2048)], 1)
    new, total = _lens(case)
    cache, page, fmt = s["cache"], case["page"], case["fmt"]
    table = cache["table"].tolist()
    k, v, ks, vs = (cache[n].double() for n in ("k", "v", "k_scale", "v_scale"))
    if case["op"] == "write":
        v = v.transpose(-1, -2).contiguous()
        at = 0
        for n, t, pages in zip(new, total, table):
            for i in range((t - n) // page, (t - 1) // page + 1):
                lo, hi = max(t - n, i * page), min(t, (i + 1) * page)
                old, p = max(0, t - n - i * page), pages[i]
                for codes, scale, rows in ((k, ks, s["k_new"]), (v, vs, s["v_new"])):
                    x = rows[at + lo - (t - n):at + hi - (t - n)].double().transpose(0, 1)
                    need = (x.abs().amax((1, 2)) / TOP[fmt]).clamp_min(FLOOR)
                    now = torch.maximum(scale[p], need) if old else need
                    codes[p, :, :old] = _nearest(codes[p, :, :old] * (scale[p] / now)[:, None, None], fmt)
                    codes[p, :, lo - i * page:hi - i * page] = _nearest(x / now[:, None, None], fmt)
                    scale[p] = now
            at += n
        return k, v.transpose(-1, -2).contiguous(), ks, vs
    if case["op"] == "read":
        out = [], []
        for t, pages in zip(total, table):
            pid = torch.tensor(pages[:-(-t // page)], device=k.device)
            x = (k[pid] * ks[pid][..., None, None]).permute(0, 2, 1, 3).flatten(0, 1)[:t]
            y = (v[pid] * vs[pid][..., None, None]).permute(0, 3, 1, 2).flatten(0, 1)[:t]
            out[0].append(x)
            out[1].append(y)
        return torch.cat(out[0]), torch.cat(out[1])
    del k, v
    at, out, group = 0, [], case["hq"] // case["hkv"]
    for n, t, pages in zip(new, total, table):
        pid = torch.tensor(pages[:-(-t // page)], device=ks.device)
        heads = []
        for h in range(case["hkv"]):
            x = (cache["k"].view(torch.uint8)[pid, h].view(CODE[fmt]).double() * ks[pid, h][:, None, None]).flatten(0, 1)[:t]
            y = cache["v"].view(torch.uint8)[pid, h].view(CODE[fmt]).double() * vs[pid, h][:, None, None]
            y = y.transpose(1, 2).flatten(0, 1)[:t]
            q = s["q"][at:at + n, h * group:(h + 1) * group].double().transpose(0, 1)
            z = q @ x.t() / math.sqrt(case["d"])
            hidden = torch.ones((n, t), dtype=torch.bool, device=z.device).triu(t - n + 1)
            heads.append(z.masked_fill(hidden, -math.inf).softmax(-1) @ y)
        out.append(torch.cat(heads).transpose(0, 1))
        at += n
    return torch.cat(out)

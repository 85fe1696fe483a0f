"""The 8-bit attention layer's operators on the GPU against their plain forms:
the residual norm and int8 rows, writing and reading the paged cache, and
attention over it."""
import random

import pytest
import torch

from dsl_tool_amd import attention as A
from dsl_tool_amd import fused as FU
from dsl_tool_amd import kvcache as KV
from dsl_tool_amd import quant as Q
from oracle import serving as O

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}     # half a step, relative


def gen(seed):
    return torch.Generator().manual_seed(seed)


def randn(shape, seed, dtype=torch.float32):
    return torch.randn(shape, generator=gen(seed)).to(dtype)


# ------------------------------------------------------------------- norm --

def check_codes(q, s, y, fmt):
    """Codes within half a step of y / s, scales within fp32 noise of
    amax / top.  y carries the noise of its own fp32 products and of the sum
    of squares: 2^-20 relative."""
    rows, cols = y.shape
    g = 128 if fmt == "fp8" else cols
    pad = -cols % g
    yg = torch.nn.functional.pad(y, (0, pad)).view(rows, -1, g)
    top = 127.0 if fmt == "int8" else 448.0
    want = (yg.abs().amax(-1) / top).clamp_min(1e-12)
    s = s.double().view(rows, -1)
    assert s.shape == want.shape
    assert ((s - want).abs() <= want * 2.0 ** -20).all()
    r = (yg / s[..., None]).view(rows, -1)[:, :cols]
    if fmt == "int8":
        assert ((q.double() - r).abs() <= 0.5 + 127 * 2.0 ** -20).all()
    else:
        v = q.view(torch.float8_e4m3fn).double()
        assert ((v - r).abs() <= torch.maximum(r.abs() * 2.0 ** -4, torch.tensor(2.0 ** -10)) * (1 + 2.0 ** -14)).all()


@pytest.mark.parametrize("fmt", ["int8", "fp8_row", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,cols", [(1, 8), (3, 136), (5, 520), (2, 1032), (7, 2048), (4, 4104), (3, 8192),
                                       (2, 16392), (1, 32768), (0, 64)])
def test_add_rmsnorm_quant(rows, cols, src, fmt):
    x, r = randn((rows, cols), 1, src), (randn((rows, cols), 2) * 3).to(src)
    if rows > 2:
        x[1], r[1] = 0, 0                       # a row of zeros: the floor of the scale
    for wdt in (torch.bfloat16, torch.float32, torch.float16):
        w = (1 + 0.1 * randn((cols,), 3)).to(wdt)
        q, s, h = FU.add_rmsnorm_quant(x.to(DEV), r.to(DEV), w.to(DEV), fmt=fmt)
        hx, y = O.norm(x, r, w, 1e-6)
        assert h.dtype == src and ((h.cpu().double() - hx).abs() <= HALF[src] * hx.abs() + 2.0 ** -25).all()
        if rows:
            check_codes(q.cpu(), s.cpu(), y, fmt)
        assert q.dtype == (torch.int8 if fmt == "int8" else torch.uint8) and q.shape == (rows, cols)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_add_rmsnorm_quant_views_and_no_residual(fmt):
    x, r, w = randn((9, 600), 4, torch.bfloat16), randn((9, 600), 5, torch.bfloat16), 1 + 0.1 * randn((512,), 6)
    xd, rd, wd = x.to(DEV), r.to(DEV), w.to(DEV)
    for a, b in ((slice(8, 520), slice(16, 528)), (slice(3, 515), slice(8, 520))):     # the second is unaligned
        q, s, h = FU.add_rmsnorm_quant(xd[:, a], rd[:, b], wd, fmt=fmt)
        q2, s2, h2 = FU.add_rmsnorm_quant(xd[:, a].contiguous(), rd[:, b].contiguous(), wd, fmt=fmt)
        assert torch.equal(q, q2) and torch.equal(s, s2) and torch.equal(h, h2)
    xc = xd[:, :512].contiguous()
    q, s, h = FU.add_rmsnorm_quant(xc, None, wd, fmt=fmt)
    assert h is xc
    check_codes(q.cpu(), s.cpu(), O.norm(x[:, :512], None, w, 1e-6)[1], fmt)


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 8), (6, 136), (33, 4096), (3, 9000), (2, 32768)])
def test_quant_int8_rows(rows, cols, src):
    x = (randn((rows, cols), 7) * torch.logspace(-3, 3, rows)[:, None]).to(src)
    x[0, : cols // 2] = 0
    q, s = Q.quant_int8_rows(x.to(DEV))
    q0, s0 = O.quant_rows(x)
    assert torch.equal(s.cpu(), s0) and torch.equal(q.cpu(), q0)


# ------------------------------------------------------------------ cache --

def table_of(lens, page, seed, spare=2, width=None):
    """A page table whose pages lie in any order, and the number of pages."""
    need = [(max(n, 0) + page - 1) // page for n in lens]
    pages = sum(need) + spare
    order = torch.randperm(pages, generator=gen(seed)).tolist()
    table = torch.full((len(lens), width or max(need + [1])), -1, dtype=torch.int32)
    for b, n in enumerate(need):
        for i in range(n):
            table[b, i] = order.pop()
    return table, pages


def to(cache, device):
    return KV.KV8Cache(*(t.to(device) for t in cache))


def same_cache(got, want):
    for a, b, name in zip(to(got, "cpu"), want, KV.KV8Cache._fields):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8)), name


def random_cache(pages, heads, dim, page, fmt, seed):
    """Codes and scales of every page, tails past the sequences' ends included;
    E4M3 tails hold NaN codes there too (:func:`spoil`)."""
    c = KV.new_kv8_cache(pages, heads, dim, page=page, fmt=fmt, device="cpu")
    for t, s in ((c.k, 8), (c.v, 9)):
        x = randn(t.shape, seed + s)
        if fmt == "int8":
            t.copy_((x * 40).round().clamp(-127, 127).to(torch.int8))
        else:
            t.copy_((x * 100).clamp(-448, 448).to(torch.float8_e4m3fn))
    c.k_scale.copy_(torch.rand((pages, heads), generator=gen(seed)) * 0.03 + 0.005)
    c.v_scale.copy_(torch.rand((pages, heads), generator=gen(seed + 1)) * 0.03 + 0.005)
    return c


def spoil(cache, lens, table):
    """NaN codes (E4M3) behind every sequence's last token."""
    if cache.k.dtype != torch.float8_e4m3fn:
        return
    page = cache.page
    for b, n in enumerate(lens):
        if n > 0 and n % page and 0 <= table[b, n // page] < cache.k.shape[0]:
            p = table[b, n // page].item()
            cache.k.view(torch.uint8)[p, :, n % page:] = 0x7f
            cache.v.view(torch.uint8)[p, :, :, n % page:] = 0xff


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 3), (32, 128, 2), (64, 256, 1), (128, 64, 1), (256, 128, 2)])
def test_kv8_write_steps(page, dim, heads, src, fmt):
    """Prompts of odd lengths, then single tokens: codes and scales bit for bit,
    growing scales included."""
    news = [page + 3, 1, 2 * page, 5]
    steps = [news] + [[1] * 4] * 3 + [[3, page, 1, 0]]
    total = [sum(s[b] for s in steps) for b in range(4)]
    table, pages = table_of(total, page, 11)
    want = random_cache(pages, heads, dim, page, fmt, 12)      # stale codes and scales in every page
    got = to(want, DEV)
    have = [0] * 4
    for i, new in enumerate(steps):
        have = [a + b for a, b in zip(have, new)]
        lens = torch.tensor(have, dtype=torch.int32)
        starts = None if new == [1] * 4 else torch.tensor([0] + new).cumsum(0).to(torch.int32)
        qkv = (randn((sum(new), 3 * heads, dim), 20 + i) * (1 + 2 * i)).to(src)     # each step is larger
        k, v = qkv[:, heads:2 * heads], qkv[:, 2 * heads:]
        O.write(want, k, v, lens, table, starts)
        dq = qkv.to(DEV)
        KV.kv8_write(got, dq[:, heads:2 * heads], dq[:, 2 * heads:], lens.to(DEV), table.to(DEV),
                     q_starts=None if starts is None else starts.to(DEV), max_q_len=max(new) if i % 2 else None)
        same_cache(got, want)


def test_kv8_write_skips_what_is_not_there():
    """Lengths of zero, page numbers outside the cache, tokens past the table
    row, more rows than tokens, starts outside the rows: skipped, and every
    other token is written."""
    page, heads, dim = 16, 2, 64
    lens = torch.tensor([0, 40, 70, 5, 20, -3], dtype=torch.int32)
    table = torch.tensor([[0, 1, 2], [3, 99, 4], [5, 6, 7], [8, -1, -1], [-7, 9, -1], [10, 11, 1]], dtype=torch.int32)
    starts = torch.tensor([0, 0, 30, 60, 72, 90, 400], dtype=torch.int32)
    want = random_cache(12, heads, dim, page, "int8", 30)
    got = to(want, DEV)
    k, v = randn((91, heads, dim), 31, torch.bfloat16), randn((91, heads, dim), 32, torch.bfloat16)
    O.write(want, k, v, lens, table, starts)
    KV.kv8_write(got, k.to(DEV), v.to(DEV), lens.to(DEV), table.to(DEV), q_starts=starts.to(DEV), max_q_len=1)
    same_cache(got, want)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 3), (32, 256, 1), (64, 128, 2), (256, 64, 1), (128, 128, 1)])
def test_kv8_read(page, dim, heads, dtype, fmt):
    lens = [0, 1, page, 3 * page + 7, 2 * page - 1]
    table, pages = table_of(lens, page, 40)
    table[3, 1] = 10 ** 6                                       # a page that is none: zeros
    cache = random_cache(pages, heads, dim, page, fmt, 41)
    rows = [0, 4, page, 2 * page + 9, 2 * page + 3]             # past the end, and less than the whole
    starts = torch.tensor([0] + rows).cumsum(0).to(torch.int32)
    lt = torch.tensor(lens, dtype=torch.int32)
    spoil(cache, lens, table)
    k, v = KV.kv8_read(to(cache, DEV), lt.to(DEV), table.to(DEV), starts.to(DEV), sum(rows), dtype=dtype)
    for got, want in zip((k, v), O.read(cache, lt, table, starts, sum(rows))):
        assert got.dtype == dtype
        # the fp32 product, then the type: half a step of each, and half of fp16's smallest step
        assert ((got.cpu().double() - want).abs() <= (HALF[dtype] + 2.0 ** -23) * want.abs() + 2.0 ** -25).all()


# -------------------------------------------------------------- attention --

def check_attention(q, cache, lens, table, starts=None, **kw):
    lt = torch.tensor(lens, dtype=torch.int32)
    st = None if starts is None else torch.tensor(starts, dtype=torch.int32)
    dkw = {k: v for k, v in kw.items() if k != "out_heads"}
    got = A.kv8_attention(q.to(DEV), to(cache, DEV), lt.to(DEV), table.to(DEV),
                          q_starts=None if st is None else st.to(DEV), **dkw)
    okw = {k: v for k, v in kw.items() if k in ("scale", "causal")}
    o, a, reach = O.attention(q, cache, lt, table, st, **okw)
    assert got.shape == q.shape and got.dtype == q.dtype
    within(got, o, a, reach)
    return got


def within(got, o, a, reach):
    """The result's half step; that of each probability (bf16; two bf16 numbers
    for fp16: 2^-16); and fp32 scores, sums and exponentials: 2^-20 of the
    largest score's terms for every probability and the sum, and 2^-16 for the
    sums over the context."""
    half = HALF[got.dtype]
    p = 2.0 ** -8 if got.dtype == torch.bfloat16 else 2.0 ** -16
    tol = half * o.abs() + a * (p + 2.0 ** -16 + 2.0 ** -19 * reach) * (1 + half) + 2.0 ** -25
    err = (got.cpu().double() - o).abs()
    assert torch.isfinite(got).all()
    assert (err <= tol).all(), (err / tol).max()


ATTN = [  # page, dim, cache heads, group
    (16, 64, 2, 1), (32, 128, 1, 7), (64, 128, 2, 4), (128, 256, 1, 2), (256, 64, 1, 16), (64, 128, 1, 40)]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads,group", ATTN)
def test_attention_single_tokens(page, dim, heads, group, src, fmt):
    lens = [1, 0, 63, 64, 65, 257, 1000]
    table, pages = table_of(lens, page, 50)
    cache = random_cache(pages, heads, dim, page, fmt, 51)
    spoil(cache, lens, table)
    got = check_attention(randn((len(lens), heads * group, dim), 52, src) * 1.5, cache, lens, table)
    assert (got[1] == 0).all()                                  # a row that sees nothing


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads,group", ATTN)
@pytest.mark.parametrize("causal", [True, False])
def test_attention_prompts(page, dim, heads, group, src, fmt, causal):
    """Several new tokens, whole prompts and parts, more rows than tokens."""
    lens, new = [3, 70, 200, 129, 0, 10], [3, 5, 200, 1, 2, 14]
    table, pages = table_of(lens, page, 60)
    cache = random_cache(pages, heads, dim, page, fmt, 61)
    spoil(cache, lens, table)
    starts = [0]
    for n in new:
        starts.append(starts[-1] + n)
    q = randn((starts[-1], heads * group, dim), 62, src)
    got = check_attention(q, cache, lens, table, starts, causal=causal, max_q_len=max(new))
    assert (got[starts[4]:starts[5]] == 0).all()
    if causal:
        assert (got[starts[5]:starts[5] + 4] == 0).all()        # positions before the first token


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_attention_long_context(fmt):
    """Contexts that are split over workgroups, of very different lengths, and a
    table far wider than any of them."""
    lens = [9000, 1, 4097, 64]
    table, pages = table_of(lens, 64, 70, width=300)
    cache = random_cache(pages, 2, 128, 64, fmt, 71)
    spoil(cache, lens, table)
    for src in (torch.bfloat16, torch.float16):
        check_attention(randn((4, 8, 128), 72, src) * 3, cache, lens, table)


def test_attention_scale_extremes():
    """Scores far apart (one token takes all), scores of zero (all alike), page
    scales decades apart, a negative softmax scale."""
    lens = [500, 333]
    table, pages = table_of(lens, 32, 80)
    for fmt in ("int8", "fp8"):
        cache = random_cache(pages, 2, 64, 32, fmt, 81)
        cache.v_scale.copy_(10.0 ** torch.linspace(-9, 2, pages)[:, None].expand(pages, 2))
        for src in (torch.bfloat16, torch.float16):
            q = randn((2, 4, 64), 82, src)
            for scale in (0.0, 1e-3, 5.0, -0.2):
                if src == torch.float16:
                    cache.v_scale.copy_(10.0 ** torch.linspace(-6, 0, pages)[:, None].expand(pages, 2))
                check_attention(q, cache, lens, table, scale=scale)


def test_attention_skips_pages_that_are_none():
    lens = [200, 90, 500]
    table, pages = table_of(lens, 16, 90)
    table[0, 3], table[0, 7], table[1, 0], table[2, 1:] = -1, pages, 2 ** 31 - 1, -5
    table = table[:, :20].contiguous()                          # the third's row ends before its tokens
    for fmt in ("int8", "fp8"):
        cache = random_cache(pages, 1, 128, 16, fmt, 91)
        for starts, new in ((None, None), ([0, 60, 150, 200], 90)):
            n = 3 if starts is None else 200
            check_attention(randn((n, 4, 128), 92, torch.bfloat16), cache, lens, table, starts)


def test_attention_strides_out_and_streams():
    """Queries inside a fused projection, a result inside a wider tensor, a
    stream of its own; each as from contiguous tensors, bit for bit."""
    lens, new = [130, 40], [5, 9]
    table, pages = table_of(lens, 16, 100)
    cache = to(random_cache(pages, 2, 128, 16, "int8", 101), DEV)
    qkv = randn((14, 12, 128), 102, torch.bfloat16).to(DEV)
    lt = torch.tensor(lens, dtype=torch.int32, device=DEV)
    st = torch.tensor([0, 5, 14], dtype=torch.int32, device=DEV)
    tb = table.to(DEV)
    want = A.kv8_attention(qkv[:, :8].contiguous(), cache, lt, tb, q_starts=st)
    wide = torch.zeros((14, 10, 136), dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = A.kv8_attention(qkv[:, :8], cache, lt, tb, q_starts=st)
        out = A.kv8_attention(qkv[:, :8], cache, lt.long(), tb.long(), q_starts=st, out=wide[:, 1:9, :128])
        odd = torch.zeros((14, 8, 129), dtype=torch.bfloat16, device=DEV)[:, :, 1:].copy_(qkv[:, :8])
        b = A.kv8_attention(odd, cache, lt, tb, q_starts=st, max_q_len=1)
    side.synchronize()
    assert out.data_ptr() == wide[:, 1:].data_ptr()
    assert torch.equal(a, want) and torch.equal(out, want)
    within(b, *O.attention(qkv[:, :8].cpu(), to(cache, "cpu"), lt.cpu(), table, st.cpu()))
    assert (wide[:, 0] == 0).all() and (wide[:, 9] == 0).all() and (wide[:, :, 128:] == 0).all()


def test_attention_the_same_twice():
    lens = [3000, 777, 1]
    table, pages = table_of(lens, 64, 110)
    cache = to(random_cache(pages, 4, 128, 64, "fp8", 111), DEV)
    q = randn((3, 32, 128), 112, torch.bfloat16).to(DEV)
    lt, tb = torch.tensor(lens, dtype=torch.int32, device=DEV), table.to(DEV)
    first = A.kv8_attention(q, cache, lt, tb)
    for _ in range(5):
        assert torch.equal(A.kv8_attention(q, cache, lt, tb), first)


def test_random_cases():
    """Seeded sizes of all kinds: a write, a read and attention over the same cache."""
    rng = random.Random(7)
    for case in range(24):
        page, dim = rng.choice(KV.PAGES), rng.choice(KV.HEAD_DIMS)
        heads, group = rng.choice([1, 2, 3]), rng.choice([1, 2, 3, 5, 8])
        fmt, src = rng.choice(["int8", "fp8"]), rng.choice([torch.bfloat16, torch.float16])
        lens = [rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 700)]) for _ in range(rng.randint(1, 6))]
        new = [rng.choice([min(n, 1), rng.randint(0, n)]) for n in lens]
        table, pages = table_of(lens, page, 200 + case)
        what = (case, page, dim, heads, group, fmt, src, lens, new)
        want = random_cache(pages, heads, dim, page, fmt, 300 + case)
        got = to(want, DEV)
        starts = torch.tensor([0] + new).cumsum(0).to(torch.int32)
        rows, lt = sum(new), torch.tensor(lens, dtype=torch.int32)
        k, v = randn((rows, heads, dim), 400 + case, src), randn((rows, heads, dim), 500 + case, src)
        args = (lt.to(DEV), table.to(DEV))
        KV.kv8_write(got, k.to(DEV), v.to(DEV), *args, q_starts=starts.to(DEV))
        O.write(want, k, v, lt, table, starts)
        same_cache(got, want)
        q = randn((rows, heads * group, dim), 600 + case, src)
        o = A.kv8_attention(q.to(DEV), got, *args, q_starts=starts.to(DEV), max_q_len=max(new + [1]))
        if rows:
            try:
                within(o, *O.attention(q, want, lt, table, starts))
            except AssertionError as e:
                raise AssertionError(what) from e

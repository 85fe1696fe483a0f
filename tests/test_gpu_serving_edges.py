"""The cache's and the attention's corners on the GPU: many sequences, codes and
scales that a row must not see, scales of every kind, prompts whose context is
split; and the layer that runs the operators together, eager and as a graph."""
import math

import pytest
import torch

from dsl_tool_amd import attention as A
from dsl_tool_amd import fused as FU
from dsl_tool_amd import gemm as G
from dsl_tool_amd import kvcache as KV
from dsl_tool_amd import layer8 as L
from dsl_tool_amd import quant as Q
from oracle import serving as O
from tests.test_gpu_serving import (ATTN, DEV, check_attention, random_cache, randn, same_cache, spoil, table_of, to,
                                    within)
from tests import test_gpu_serving as S

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["auto", "prompt"])
def route(request, monkeypatch):
    """Attention as the sizes have it, and all of it by the kernel of prompts."""
    if request.param == "prompt":
        monkeypatch.setenv("DSL_ATTN_FEW_ROWS", "0")
    return request.param


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def starts_of(new):
    return [sum(new[:i]) for i in range(len(new) + 1)]


# ------------------------------------------------------------------- cache --

@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("seqs", [65, 300])
def test_many_sequences(seqs, fmt):
    """More sequences than a wave looks at: empty ones, single tokens, prompts."""
    lens = [(b * 37) % 90 for b in range(seqs)]
    new = [n if b % 5 == 0 else min(n, b % 3) for b, n in enumerate(lens)]
    table, pages = table_of(lens, 16, 700)
    want = random_cache(pages, 1, 64, 16, fmt, 701)
    got = to(want, DEV)
    starts = starts_of(new)
    lt, st = ints(lens), ints(starts)
    k, v = randn((starts[-1], 1, 64), 702, torch.bfloat16), randn((starts[-1], 1, 64), 703, torch.bfloat16)
    KV.kv8_write(got, k.to(DEV), v.to(DEV), lt.to(DEV), table.to(DEV), q_starts=st.to(DEV))
    O.write(want, k, v, lt, table, st)
    same_cache(got, want)
    q = randn((starts[-1], 2, 64), 704, torch.bfloat16)
    check_attention(q, want, lens, table, starts, max_q_len=max(new))
    check_attention(q, want, lens, table, starts, max_q_len=1)          # a hint that is too small
    check_attention(randn((seqs, 2, 64), 705, torch.bfloat16), want, lens, table)
    total = starts_of(lens)
    a, b = KV.kv8_read(got, lt.to(DEV), table.to(DEV), ints(total).to(DEV), total[-1])
    x, y = O.read(want, lt, table, ints(total), total[-1])
    half = 2.0 ** -8
    for g, w in ((a, x), (b, y)):
        assert ((g.cpu().double() - w).abs() <= w.abs() * (half + 2.0 ** -23)).all()


def test_a_workgroup_per_unit():
    """More units than runs are worth, and contexts of a single round."""
    for seqs, heads, span in ((1100, 4, 300), (40, 2, 256)):
        lens = [(b * 71) % span + 1 for b in range(seqs)]
        table, pages = table_of(lens, 64, 710)
        cache = random_cache(pages, heads, 64, 64, "int8", 711)
        check_attention(randn((seqs, heads * 2, 64), 712, torch.bfloat16), cache, lens, table)
        new = [min(n, b % 4) if b % 7 else min(n, 40) for b, n in enumerate(lens)]
        starts = starts_of(new)
        q = randn((starts[-1], heads * 2, 64), 713, torch.bfloat16)
        check_attention(q, cache, lens, table, starts, max_q_len=40)
        check_attention(q, cache, lens, table, starts, max_q_len=1)
    check_attention(randn((seqs, heads * 20, 64), 714, torch.bfloat16), cache, lens, table)      # two blocks of rows


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_write_scales_of_every_kind(fmt):
    """Tokens of zeros, of subnormals, very large and negative zero
    ones; kept scales that no amax gives."""
    lens, new = [40, 40, 40, 40, 40, 40, 17], [40, 3, 40, 5, 5, 5, 1]
    table, pages = table_of(lens, 32, 720)
    want = random_cache(pages, 2, 64, 32, fmt, 721)
    starts = starts_of(new)
    k, v = randn((starts[-1], 2, 64), 722, torch.bfloat16), randn((starts[-1], 2, 64), 723, torch.bfloat16)
    for t in (k, v):
        t[starts[0]:starts[1]] = 0
        t[starts[0], :, ::3] = -0.0
        t[starts[1]:starts[2]] *= 2.0 ** -130
        t[starts[2]:starts[3]] *= 2.0 ** 120
    for s in (want.k_scale, want.v_scale):
        s[table[3, 1].item()] = 3e38                       # 1 / s is subnormal
        s[table[4, 1].item()] = math.inf
        s[table[5, 1].item()] = 1e-30
    got = to(want, DEV)
    args = (ints(lens), table, ints(starts))
    KV.kv8_write(got, k.to(DEV), v.to(DEV), args[0].to(DEV), args[1].to(DEV), q_starts=args[2].to(DEV))
    O.write(want, k, v, *args)
    same_cache(got, want)


# --------------------------------------------------------------- attention --

@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads,group", ATTN)
@pytest.mark.parametrize("causal", [True, False])
def test_every_size_by_the_prompts_kernel(page, dim, heads, group, src, fmt, causal, monkeypatch):
    monkeypatch.setenv("DSL_ATTN_FEW_ROWS", "0")
    S.test_attention_prompts(page, dim, heads, group, src, fmt, causal)
    if causal:
        S.test_attention_single_tokens(page, dim, heads, group, src, fmt)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim,group", [(64, 8), (128, 4), (256, 1)])
def test_prompts_of_many_blocks(dim, group, src, fmt):
    """Enough rows that the sizes themselves choose the kernel of prompts."""
    lens, new = [2100, 1300], [1100, 1300]
    table, pages = table_of(lens, 64, 770)
    cache = random_cache(pages, 4, dim, 64, fmt, 771)
    spoil(cache, lens, table)
    check_attention(randn((2400, 4 * group, dim), 772, src), cache, lens, table, [0, 1100, 2400], max_q_len=1300)


@pytest.mark.parametrize("group,new", [(1, 6), (4, 5), (8, 40), (1, 300)])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_hidden_nan_codes(dim, src, group, new, route):
    """An E4M3 NaN in a new token: the rows before it are as without it, the
    rows from it on are NaN (in its column, for a value; wholly, for a key)."""
    length = 70 + new
    table, pages = table_of([length], 16, 730)
    clean = random_cache(pages, 2, dim, 16, "fp8", 731)
    q = randn((new, 2 * group, dim), 732, src)
    lt, st = ints([length]), ints([0, new])
    want = O.attention(q, clean, lt, table, st)
    at = new // 2
    pos = length - new + at
    page, slot = table[0, pos // 16].item(), pos % 16
    col = 37
    for code in (0x7f, 0xff):
        for key in (False, True):
            c = KV.KV8Cache(*(t.clone() for t in clean))
            if key:
                c.k.view(torch.uint8)[page, 0, slot, col] = code
            else:
                c.v.view(torch.uint8)[page, 0, col, slot] = code
            got = A.kv8_attention(q.to(DEV), to(c, DEV), lt.to(DEV), table.to(DEV), q_starts=st.to(DEV)).cpu()
            nan = got.isnan()
            hit = torch.zeros_like(nan)
            if key:
                hit[at:, :group] = True
            else:
                hit[at:, :group, col] = True
            assert torch.equal(nan, hit)
            fixed = torch.where(hit, want[0], got.double()).to(src)
            within(fixed, *want)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("new", [1, 7, 100])
def test_nothing_past_the_end_is_seen(new, fmt, route):
    """Table entries behind the last token's page name pages whose scales are
    NaN; so does the last page of another sequence's row."""
    lens = [65 + new, 128 + new]
    table, pages = table_of(lens, 32, 740, spare=3, width=20)
    cache = random_cache(pages, 2, 128, 32, fmt, 741)
    spoil(cache, lens, table)
    used = set(table.flatten().tolist())
    bad = next(p for p in range(pages) if p not in used)
    cache.k_scale[bad] = cache.v_scale[bad] = math.nan
    table[table < 0] = bad
    q = randn((2 * new, 8, 128), 742, torch.bfloat16)
    for causal in (True, False):
        check_attention(q, cache, lens, table, [0, new, 2 * new], max_q_len=new, causal=causal)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,group", [(16, 64, 4), (64, 128, 4), (32, 128, 1), (128, 256, 2), (256, 64, 16)])
def test_long_prompts(page, dim, group, src, fmt, route):
    """Prompts over many tiles, whose context is split and joined; a page of none
    in the middle."""
    lens, new = [1500, 333, 64, 0], [150, 333, 1, 2]
    table, pages = table_of(lens, page, 750)
    cache = random_cache(pages, 1, dim, page, fmt, 751)
    spoil(cache, lens, table)
    table[0, 300 // page] = -1
    starts = starts_of(new)
    q = randn((starts[-1], group, dim), 752, src)
    for causal in (True, False):
        check_attention(q, cache, lens, table, starts, max_q_len=max(new), causal=causal)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_prompt_scales_of_every_kind(src, fmt, route):
    """Page scales of zero, negative ones, and ones decades apart, in prompts and
    for few rows."""
    lens = [700]
    table, pages = table_of(lens, 16, 760)
    cache = random_cache(pages, 1, 128, 16, fmt, 761)
    low = -6 if src == torch.float16 else -20
    cache.v_scale.copy_(10.0 ** torch.linspace(low, -1, pages)[:, None])
    for i in range(0, lens[0] // 16, 5):
        p = table[0, i].item()
        cache.v_scale[p] = 0.0 if i % 2 else -0.01
        cache.k_scale[table[0, i + 1].item()] = 0.0 if i % 3 else -0.004
    for new in (200, 3):
        check_attention(randn((new, 4, 128), 762, src), cache, lens, table, [0, new], max_q_len=new)


# ------------------------------------------------------------------- layer --

HQ, HKV, DIM, HIDDEN = 8, 2, 64, 512


def new_layer(rotate=None):
    w = [randn((n, k), 800 + i) / math.sqrt(k) for i, (n, k) in
         enumerate((((HQ + 2 * HKV) * DIM, HIDDEN), (HIDDEN, HQ * DIM)))]
    norm = 1 + 0.1 * randn((HIDDEN,), 802)
    layer = L.Int8AttentionLayer(*(t.to(DEV, torch.bfloat16) for t in w), norm.to(DEV), q_heads=HQ, kv_heads=HKV,
                                 dim=DIM, rotate=rotate)
    return layer, [t.to(torch.bfloat16).double() for t in w], norm.double()


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_layer(fmt):
    """A prompt, then single tokens: bit for bit the operators called one by
    one, and the plain layer in 64 bits.  A row quantized to int8 is off by a
    step of amax/127 over sqrt(12), at most 1.1% of its norm for normal values
    of up to 4.8 deviations; E4M3 codes are off by at most 2^-4 / sqrt(3),
    3.6%.  Six such roundings lie on the way (the norm's, both weights', the
    keys', the values', the attention's), two of them in the cache: 2.7% and
    5.6% in quadrature; twice that is allowed."""
    layer, (wq, wo), norm = new_layer()
    lens = [50, 7]
    full = [n + 3 for n in lens]
    table, pages = table_of(full, 16, 810)
    cache = KV.new_kv8_cache(pages, HKV, DIM, page=16, fmt=fmt, device=DEV)
    twin = to(cache, DEV)
    twin = KV.KV8Cache(*(t.clone() for t in twin))
    x = [randn((n + 3, HIDDEN), 820 + b, torch.bfloat16) for b, n in enumerate(lens)]
    r = [randn((n + 3, HIDDEN), 830 + b, torch.bfloat16) for b, n in enumerate(lens)]
    want = []
    for a, b in zip(x, r):
        h = a.double() + b.double()
        y = h / (h * h).mean(-1, keepdim=True).add(1e-6).sqrt() * norm
        q, k, v = (y @ wq.T).view(len(a), HQ + 2 * HKV, DIM).split([HQ, HKV, HKV], 1)
        k, v = (t.repeat_interleave(HQ // HKV, 1) for t in (k, v))
        z = torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(DIM)
        z = z.masked_fill(torch.ones(len(a), len(a)).triu(1).bool(), -math.inf).softmax(-1)
        want.append(torch.einsum("hij,jhd->ihd", z, v).reshape(len(a), -1) @ wo.T)
    got = [[], []]
    for step in range(4):
        new = lens if step == 0 else [1, 1]
        now = [n + step for n in lens]
        starts = starts_of(new)
        args = (ints(now).to(DEV), table.to(DEV))
        kw = dict(q_starts=ints(starts).to(DEV), max_q_len=max(new)) if step == 0 else {}
        xs, rs = (torch.cat([t[b][now[b] - new[b]:now[b]] for b in (0, 1)]).to(DEV) for t in (x, r))
        out, h = layer(xs, rs, cache, *args, **kw)
        codes, s, h2 = FU.add_rmsnorm_quant(xs, rs, layer.norm)
        qkv = G.int8_gemm_packed(codes, layer.w_qkv, s, layer.s_qkv).view(len(xs), -1, DIM)
        KV.kv8_write(twin, qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], *args, **kw)
        o = A.kv8_attention(qkv[:, :HQ], twin, *args, **kw)
        codes, s = Q.quant_int8_rows(o.view(len(xs), -1))
        assert torch.equal(out, G.int8_gemm_packed(codes, layer.w_out, s, layer.s_out)) and torch.equal(h, h2)
        for b in (0, 1):
            got[b].append(out[starts[b]:starts[b + 1]].cpu().double())
    for b in (0, 1):
        g = torch.cat(got[b])
        assert (g - want[b]).norm() <= (0.054 if fmt == "int8" else 0.112) * want[b].norm()


def test_layer_as_a_graph():
    """Single-token steps of a captured layer, with eager work between the
    replays, against the same steps run eagerly."""
    layer, _, _ = new_layer(rotate=lambda q, k: (q * 0.5, k * 2))
    lens, steps = [1000, 3, 77], 5
    table, pages = table_of([n + steps for n in lens], 64, 840)
    start = to(random_cache(pages, HKV, DIM, 64, "int8", 841), DEV)
    x = randn((steps, 3, HIDDEN), 842, torch.bfloat16).to(DEV)
    r = randn((steps, 3, HIDDEN), 843, torch.bfloat16).to(DEV)
    tb = table.to(DEV)
    eager_cache = KV.KV8Cache(*(t.clone() for t in start))
    eager = [layer(x[i], r[i], eager_cache, ints([n + i + 1 for n in lens]).to(DEV), tb) for i in range(steps)]
    cache = KV.KV8Cache(*(t.clone() for t in start))
    xs, rs, lt = x[0].clone(), r[0].clone(), ints([n + 1 for n in lens]).to(DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):                          # a first run outside the graph
        layer(xs, rs, cache, lt, tb)
    torch.cuda.current_stream().wait_stream(side)
    for t, s in zip(cache, start):
        t.copy_(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, h = layer(xs, rs, cache, lt, tb)
    for i in range(steps):
        xs.copy_(x[i])
        rs.copy_(r[i])
        lt.copy_(ints([n + i + 1 for n in lens]))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, eager[i][0]) and torch.equal(h, eager[i][1]), i
        (torch.randn(256, 256, device=DEV) @ torch.randn(256, 256, device=DEV)).sum()
    for a, b in zip(cache, eager_cache):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))

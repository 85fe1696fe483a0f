"""The 8-bit layer's operators at their limits on the GPU: rows that see
nothing, NaN over contexts that are split, launches of very many workgroups,
lengths and scores at the ends of their types."""
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
from tests.test_gpu_serving import DEV, check_attention, random_cache, randn, table_of, to, within
from tests.test_gpu_serving_edges import DIM, HIDDEN, HKV, HQ, ints, new_layer, route, starts_of  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------ rows that see nothing --

@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_blocks_that_see_nothing_after_nan_ones(dim, src, causal, monkeypatch):
    """Whole blocks of prompts' rows that see no token are zeros, whatever the
    workgroups' shared memory held before: a call all of whose rows get NaN
    columns goes first, with a workgroup or more for every CU."""
    monkeypatch.setenv("DSL_ATTN_FEW_ROWS", "0")
    seqs, heads, new = 40, 8, 70
    table, pages = table_of([new] * seqs, 64, 960)
    cache = random_cache(pages, heads, dim, 64, "fp8", 961)
    dirty = cache._replace(v=torch.full(cache.v.shape, 0x7f, dtype=torch.uint8).view(cache.v.dtype))
    starts = starts_of([new] * seqs)
    q = randn((starts[-1], heads * 4, dim), 962, src).to(DEV)
    st, tb = ints(starts).to(DEV), table.to(DEV)
    dirty, clean = to(dirty, DEV), to(cache, DEV)
    for lens in ([0] * seqs, [0 if b % 2 else 3 for b in range(seqs)]):
        full = A.kv8_attention(q, dirty, ints([new] * seqs).to(DEV), tb, q_starts=st, max_q_len=new)
        got = A.kv8_attention(q, clean, ints(lens).to(DEV), tb, q_starts=st, max_q_len=new, causal=causal)
        assert full.isnan().all()
        for b, n in enumerate(lens):
            none = got[starts[b]:starts[b + 1] - (n if causal else new if n else 0)]
            assert (none == 0).all(), b
    # two blocks, the first of which sees nothing and the second the only tokens
    lens, starts = [5, 0, 40], [0, 300, 600, 900]
    check_attention(randn((900, 4, dim), 963, src), random_cache(pages, 4, dim, 64, "fp8", 964), lens, table[:3],
                    starts, max_q_len=300, causal=causal)


# ------------------------------------------------------------------ scores --

@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("seqs", [1, 130])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_scores_that_overflow_below(dim, seqs, fmt, route):
    """Tokens whose products fall below the least fp32 number, several tiles of
    them before any other: probability 0, as in 64 bits.  One sequence, whose
    context is split, and enough that none is."""
    new = 9
    lens, starts = [720] * seqs, starts_of([new] * seqs)
    table, pages = table_of([720], 64, 930)
    table = table.repeat(seqs, 1)
    cache = random_cache(pages, 2, dim, 64, fmt, 931)
    early = table[0, :8].long()
    cache.k.view(torch.uint8)[:, :, :, 0] = 0
    cache.k[early, :, :, 0] = torch.full((), 100.0).to(cache.k.dtype)
    q = randn((starts[-1], 4, dim), 932, torch.bfloat16)
    q[:, :, 0] = -3e38
    lt, st = ints(lens), ints(starts)
    got = A.kv8_attention(q.to(DEV), to(cache, DEV), lt.to(DEV), table.to(DEV), q_starts=st.to(DEV), max_q_len=new)
    q[:, :, 0] = 0                                         # the others' scores do not have it
    late = table.clone()
    late[:, :8] = -1
    within(got, *O.attention(q, cache, lt, late, st))


# ------------------------------------------------------ NaN and joined parts --

def nan_where_it_belongs(q, cache, lens, table, starts=None, **kw):
    """The oracle's NaNs, no others; the rest within the tolerance."""
    lt, st = ints(lens), None if starts is None else ints(starts)
    got = A.kv8_attention(q.to(DEV), to(cache, DEV), lt.to(DEV), table.to(DEV),
                          q_starts=None if st is None else st.to(DEV), **kw).cpu()
    o, a, reach = O.attention(q, cache, lt, table, st, **kw)
    assert torch.equal(got.isnan(), o.isnan())
    rows = o.isnan().any(-1, keepdim=True).expand_as(o)
    zero = torch.zeros_like(o)
    within(got.masked_fill(rows, 0), *(torch.where(rows, zero, t.expand_as(o)) for t in (o, a, reach)))
    return got


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_queries_over_long_contexts(dim, src, fmt, route):
    """A NaN query is a NaN row, whether its context is split or not."""
    lens = [5000, 300, 2000]
    table, pages = table_of(lens, 64, 900)
    cache = random_cache(pages, 2, dim, 64, fmt, 901)
    q = randn((3, 8, dim), 902, src)
    q[0, 3, 5] = q[1, 0, 0] = q[2, 7, dim - 1] = math.nan
    got = nan_where_it_belongs(q, cache, lens, table)
    assert got[0, 3].isnan().all() and got[1, 0].isnan().all() and got[2, 7].isnan().all()
    new = [3, 200, 1]
    starts = starts_of(new)
    q = randn((starts[-1], 8, dim), 903, src)
    q[1, 2, 9] = q[50, 4, 1] = q[203, 0, 2] = math.nan
    nan_where_it_belongs(q, cache, lens, table, starts)


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_keys_that_are_all_a_part_sees(dim, src, route):
    """The part that begins at token 5120 has three tokens; the first new row sees
    one of them, a NaN key."""
    lens, starts = [20 * 256 + 3], [0, 3]
    table, pages = table_of(lens, 64, 910)
    cache = random_cache(pages, 2, dim, 64, "fp8", 911)
    cache.k.view(torch.uint8)[table[0, 80], 1, 0, 7] = 0x7f
    got = nan_where_it_belongs(randn((3, 4, dim), 912, src), cache, lens, table, starts)
    assert got[:, 2:].isnan().all() and not got[:, :2].isnan().any()


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_nan_values_of_vanishing_probability(dim, src, route):
    """A NaN value in a part whose scores lie so far below the others that its
    factor is 0: 0 times NaN is NaN, as in a context that is not split."""
    lens = [20 * 256]
    table, pages = table_of(lens, 64, 920)
    cache = random_cache(pages, 1, dim, 64, "fp8", 921)
    first = table[0, :4].long()
    cache.k.view(torch.uint8)[:, :, :, 0] = 0
    cache.k[first, :, :, 0] = torch.full((), -64.0).to(torch.float8_e4m3fn)
    cache.k_scale.fill_(0.02)
    cache.v.view(torch.uint8)[table[0, 1], 0, 11, 3] = 0xff
    q = randn((1, 3, dim), 922, src)
    q[:, :, 0] = 64
    got = nan_where_it_belongs(q, cache, lens, table, scale=4.0)
    assert got[:, :, 11].isnan().all()


# ---------------------------------------------------------------- launches --

@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_a_workgroup_walks_several_blocks(dim, fmt, monkeypatch):
    """Prompts under a max_q_len far too small: one block's workgroups take all."""
    monkeypatch.setenv("DSL_ATTN_FEW_ROWS", "0")
    lens, starts = [420, 700, 0, 33], [0, 400, 900, 903, 910]
    table, pages = table_of(lens, 32, 970)
    cache = random_cache(pages, 2, dim, 32, fmt, 971)
    q = randn((910, 8, dim), 972, torch.bfloat16)
    for causal in (True, False):
        check_attention(q, cache, lens, table, starts, max_q_len=1, causal=causal)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_more_workgroups_than_a_launch_has(fmt):
    """8192 sequences x 16 heads without max_q_len: by all 16384 rows they would be
    2^23 workgroups of 512 threads, one more than a launch may have."""
    seqs, heads = 8192, 16
    lens = [(b * 7) % 15 + 2 for b in range(seqs)]
    table = ints([b % 61 for b in range(seqs)])[:, None].contiguous()
    cache = random_cache(61, heads, 64, 16, fmt, 980)
    q = randn((2 * seqs, heads, 64), 981, torch.bfloat16)
    check_attention(q, cache, lens, table, starts_of([2] * seqs))


def test_more_rows_than_a_join_takes():
    """2^24 rows and heads over a context that is long enough to be split, under a
    max_q_len far too small: a workgroup of 256 threads for each would be 2^32."""
    rows, hq, dim, n = 1 << 18, 64, 64, 2304
    table, pages = table_of([n], 256, 990)
    cache = random_cache(pages, 1, dim, 256, "int8", 991)
    q = torch.randn((rows, hq, dim), dtype=torch.bfloat16, device=DEV, generator=torch.Generator(DEV).manual_seed(992))
    got = A.kv8_attention(q, to(cache, DEV), ints([n]).to(DEV), table.to(DEV), q_starts=ints([0, rows]).to(DEV),
                          max_q_len=1, causal=False)
    pick = torch.tensor([0, 1, 99999, rows - 2, rows - 1])
    some = q[pick.to(DEV)].cpu()
    within(got[pick.to(DEV)], *O.attention(some, cache, ints([n]), table, ints([0, 5]), causal=False))
    assert torch.isfinite(got).all()


@pytest.mark.parametrize("seqs,heads", [(2, 8), (4, 8), (3, 8), (3, 16), (8, 8), (5, 4), (3, 2)])
def test_blocks_of_pairs_over_the_xcds(seqs, heads):
    """Every pair of sequence and cache head gets each of its blocks, however many
    pairs rotate over the XCDs."""
    new = [700 - 90 * (b % 4) for b in range(seqs)]
    table, pages = table_of([n + 8 for n in new], 64, 995)
    cache = random_cache(pages, heads, 64, 64, "int8", 996)
    starts = starts_of(new)
    check_attention(randn((starts[-1], 2 * heads, 64), 997, torch.bfloat16), cache, [n + 8 for n in new], table, starts,
                    max_q_len=700)


# ------------------------------------------------------------------- layers --

@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_layers_chain(src):
    """Two layers one behind the other, a prompt and a single token: the results
    of the first enter the second.  A projection is off by the rounding of its
    type once: fp16's are those of the fp32 product."""
    layers = [new_layer()[0] for _ in range(2)]
    lens = [9, 4]
    table, pages = table_of([n + 1 for n in lens], 16, 950)
    caches = [KV.new_kv8_cache(pages, HKV, DIM, page=16, device=DEV) for _ in layers]
    for new, have in ((lens, lens), ([1, 1], [n + 1 for n in lens])):
        starts = starts_of(new)
        x, h = randn((starts[-1], HIDDEN), 951, src).to(DEV), randn((starts[-1], HIDDEN), 952, src).to(DEV)
        args = (ints(have).to(DEV), table.to(DEV))
        for layer, cache in zip(layers, caches):
            before = KV.KV8Cache(*(t.clone() for t in cache))
            codes, s, _ = FU.add_rmsnorm_quant(x, h, layer.norm)
            qkv = G.int8_gemm_packed(codes, layer.w_qkv, s, layer.s_qkv, out_dtype=torch.float32).to(src).view(len(x), -1, DIM)
            x, h = layer(x, h, cache, *args, q_starts=ints(starts).to(DEV), max_q_len=max(new))
            assert x.dtype == h.dtype == src and x.isfinite().all()
            KV.kv8_write(before, qkv[:, HQ:HQ + HKV], qkv[:, HQ + HKV:], *args, q_starts=ints(starts).to(DEV))
            for a, b in zip(before, cache):
                assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
            o = A.kv8_attention(qkv[:, :HQ], before, *args, q_starts=ints(starts).to(DEV), max_q_len=max(new))
            codes, s = Q.quant_int8_rows(o.view(len(x), -1))
            want = G.int8_gemm_packed(codes, layer.w_out, s, layer.s_out, out_dtype=torch.float32)
            assert torch.equal(x, want.to(src))


def test_fp16_norm_weights_are_converted_once():
    """... by the constructor, not by a launch in every call; with the same results."""
    w = [randn((n, k), 980 + i).to(DEV) / math.sqrt(k) for i, (n, k) in
         enumerate((((HQ + 2 * HKV) * DIM, HIDDEN), (HIDDEN, HQ * DIM)))]
    norm = (1 + 0.1 * randn((HIDDEN,), 985)).half().to(DEV)
    x, table, outs = randn((3, HIDDEN), 986, torch.bfloat16).to(DEV), ints([[0]]).to(DEV), []
    for weight in (norm, norm.float()):
        layer = L.Int8AttentionLayer(*w, weight, q_heads=HQ, kv_heads=HKV, dim=DIM)
        assert layer.norm.dtype == torch.float32
        cache = KV.new_kv8_cache(1, HKV, DIM, page=16, device=DEV)
        outs.append(layer(x, None, cache, ints([3]).to(DEV), table, q_starts=ints([0, 3]).to(DEV))[0])
    assert torch.equal(*outs)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("width", [3, 160])
def test_lengths_next_to_the_largest_int(width, causal, route):
    """A length far past the table's row: the row's tokens are seen."""
    lens = [2 ** 31 - 1, 2 ** 31 - 40, 150]
    table, pages = table_of([width * 16, width * 16, 40], 16, 940)
    cache = random_cache(pages, 2, 64, 16, "int8", 941)
    check_attention(randn((3, 4, 64), 942, torch.bfloat16), cache, lens, table, causal=causal)
    check_attention(randn((7, 4, 64), 943, torch.bfloat16), cache, lens, table, [0, 2, 6, 7], max_q_len=4, causal=causal)

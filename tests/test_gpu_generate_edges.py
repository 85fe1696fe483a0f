"""Several continuations of a prompt at their edges on the GPU: pages that are missing before
others and scores that overflow, with every number of query rows a wave; logits of any size;
steps that lacked pages and are made again; several new tokens by the kernels that the sizes
choose, and NaN among tokens that only some rows see."""
import math
import random

import pytest
import torch

from dsl_tool_amd import _native as N
from dsl_tool_amd import attention as A
from dsl_tool_amd import kvcache as KV
from dsl_tool_amd import logprobs as LP
from oracle import generating as GO
from oracle import serving as O
from tests.test_gpu_generate import PLAN, SHARED, check_fork, check_shared, equal, forked, ints, pool, spoil
from tests.test_gpu_generate_steps import wide  # noqa: F401
from tests.test_gpu_serving import DEV, randn, random_cache, same_cache, to, within

pytestmark = pytest.mark.gpu


# --------------------------------------------- rows that begin with nothing seen --

def holes(table, page, prefix, kind, seed):
    """The table without some of its pages, those of the prefix in every row."""
    rng, t, shared = random.Random(seed), table.clone(), prefix // page
    if kind == "first":
        t[:, :1] = -1
    elif kind == "tiles":                        # the first four tiles of 64 tokens, one for each wave
        t[:, :max(256 // page, 1)] = -1
    elif kind == "prefix":
        t[:, :shared] = -1
    elif kind == "own":
        t[:, shared:shared + 1] = -1
    else:                                        # 64 tokens and more here and there: at the beginnings of rounds too
        step = max(64 // page, 1)
        for i in range(0, t.shape[1], step):
            if i < shared:
                if rng.random() < 0.4:
                    t[:, i:min(i + step, shared)] = -1
            else:
                for row in t:
                    if rng.random() < 0.4:
                        row[i:i + step] = -1
    return t


@pytest.mark.parametrize("kind", ["first", "tiles", "prefix", "own", "some"])
@pytest.mark.parametrize("page,dim,fmt,src", [(16, 64, "int8", torch.float16), (64, 128, "fp8", torch.bfloat16),
                                              (256, 64, "fp8", torch.bfloat16), (64, 256, "int8", torch.float16),
                                              (32, 64, "fp8", torch.float16), (256, 128, "int8", torch.bfloat16)])
def test_tokens_behind_pages_that_are_none(page, dim, fmt, src, kind, wide):
    """Valid tokens behind missing ones are not lost: the first page, four tiles, the whole
    prefix, the first own page, here and there.  16 cache heads of 50 rounds and more: a
    workgroup's waves walk several tiles.  (Small scores: no sum grows.)"""
    lens, table, groups, shared, pages = forked([(12800, [3, 70, 2500, 5, 300, 1])], page, 500)
    cache = random_cache(pages, 16, dim, page, fmt, 501)
    spoil(cache, lens, table)
    table = holes(table, page, 12800, kind, 502)
    check_shared(randn((6, 64, dim), 503, src) / 4, cache, lens, table, groups, shared)
    new = [1, 3, 2, 4, 1, 1]
    check_shared(randn((12, 64, dim), 504, src) / 4, cache, lens, table, groups, shared, new, max_q_len=4)


@pytest.mark.parametrize("rows", ["16", "32", "64", None])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_holes_of_long_runs(fmt, rows, monkeypatch):
    """The rows a wave that the sizes choose too: 96 rows of a prefix of 30000 tokens a fifth
    of which is missing."""
    if rows:
        monkeypatch.setenv("DSL_ATTN_SHARED_ROWS", rows)
    lens, table, groups, shared, pages = forked([(30000, [300 + b for b in range(6)])], 64, 510)
    cache = random_cache(pages, 8, 64, 64, fmt, 511)
    spoil(cache, lens, table)
    rng = random.Random(512)
    for i in range(30000 // 64):
        if i < 9 or rng.random() < 0.2:
            table[:, i] = -1
    check_shared(randn((6, 128, 64), 513, torch.bfloat16), cache, lens, table, groups, shared)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_shared_scores_that_overflow_below(dim, fmt, wide):
    """Tokens whose scores fall below the least fp32 number, in whole tiles: probability 0, as
    in 64 bits."""
    lens, table, groups, shared, pages = forked([(12800, [3, 70, 2500, 5])], 64, 520)
    cache = random_cache(pages, 16, dim, 64, fmt, 521)
    early = table[0, 0:200:3].long()             # every third page of the prefix: some of each wave's
    cache.k.view(torch.uint8)[:, :, :, 0] = 0
    cache.k[early] = 0
    cache.k[early, :, :, 0] = torch.full((), -100.0).to(cache.k.dtype)
    cache.k_scale[early] = 3e38
    q = randn((4, 64, dim), 522, torch.bfloat16) / 4
    q[:, :, 0] = 4.0
    others = table.clone()
    others[:, 0:200:3] = -1
    args = [ints(lens).to(DEV), table.to(DEV), ints(groups).to(DEV), ints(shared).to(DEV)]
    got = A.kv8_shared_attention(q.to(DEV), to(cache, DEV), *args)
    within(got, *O.attention(q, cache, ints(lens), others))


# -------------------------------------------------------------- logits of any size --

@pytest.mark.parametrize("scale", [1.0, 0.5, 1.25, 2.0 ** -120, 2.0 ** -140, 2.0 ** 100])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [9, 1003, 40000])
def test_logprobs_of_logits_of_any_size(vocab, src, scale):
    """Rows that are masked by the type's lowest value, in part or all of them, of very low and
    very high ones, and from one end of the type to the other.  The tolerance: the result's rounding
    and that of its terms, 2^-22; 2^-19 for the sums."""
    least, most = torch.finfo(src).min, torch.finfo(src).max
    i = torch.arange(vocab, dtype=torch.float64)
    rows = [torch.full((vocab,), v, dtype=torch.float64) for v in (least, most, least / 2, -1e10, 1e10, -1e30, 1e30, -2e4)]
    rows += [torch.where(i % 5 == 2, i % 3, least), torch.where(i == vocab - 2, most, least), torch.where(i % 2 == 0, least, -math.inf),
             least + (most / vocab * 2) * i, least * (1 - (i % 7) / 64), most * (1 - (i % 7) / 64)]
    x = torch.stack(rows).clamp(least, most).where(torch.stack(rows) != -math.inf, -math.inf).to(src)
    ids = torch.tensor([[0, 1, vocab // 2, vocab - 2, vocab - 1]] * len(rows), dtype=torch.int32)
    top = min(7, vocab)
    got = LP.token_logprobs(x.to(DEV), ids.to(DEV), top=top, scale=scale)
    want = GO.logprobs(x, ids, top, scale)
    assert torch.equal(got.top_ids.cpu(), want[3])
    for g, w in ((got.logp, want[0]), (got.entropy, want[1]), (got.top_logp, want[2])):
        g, none = g.cpu(), w.float().isneginf()
        assert torch.equal(g.isneginf(), none)
        assert ((g.double() - w)[~none].abs() <= w[~none].abs() * 2.0 ** -22 + 2.0 ** -19).all()


# ------------------------------------------------------ steps that are made again --

def test_fork_made_again():
    """A step that lacked pages changes no page of a sequence that it continued, nor one that
    the caller keeps; fewer children of the same parents then come out as if it had not been
    made, tokens included.  What it dropped is free: its copies may lie there."""
    page, lens = 16, [40, 20, 25, 55]
    table, refs = pool(lens, page, 1, 600, width=5)
    mine = [table[b, :-(-n // page)].tolist() for b, n in enumerate(lens)]
    for kept in (False, True):
        counts = refs.clone()
        if kept:
            counts[mine[1]] += 1                 # the sequence that the step drops
        clean = random_cache(len(refs), 2, 64, page, "int8", 601)
        cache = to(clean, DEV)
        given = [t.to(DEV) for t in (ints(lens), table)]
        first = KV.kv8_fork(cache, *given, ints([0, 0, 2, 3, 3, 0, 2]).to(DEV), counts.to(DEV), new=30)
        assert first.lacking.item() > 0
        whole = mine[0] + mine[2] + mine[3] + (mine[1] if kept else [])
        now = to(cache, "cpu")
        for a, b in zip(now, clean):
            assert torch.equal(a.view(torch.uint8)[whole], b.view(torch.uint8)[whole])
        changed = [p for p in mine[1] if not torch.equal(now.k[p], clean.k[p])]
        assert bool(changed) != kept
        again = ints([3, 0, 0])
        want_cache = KV.KV8Cache(*(t.clone() for t in now))
        want = GO.fork(want_cache, ints(lens), table, again, counts, 1)
        got = KV.kv8_fork(cache, *given, again.to(DEV), counts.to(DEV), new=1)
        equal(got, want)
        same_cache(cache, want_cache)
        assert want[3].item() == 0
        other = KV.KV8Cache(*(t.clone() for t in clean))
        GO.fork(other, ints(lens), table, again, counts, 1)
        for row, n in zip(want[1], (55, 40, 40)):
            a, b = (O.tokens(c, n, row.tolist()) for c in (want_cache, other))
            assert all(torch.equal(x, y) for x, y in zip(a, b))


# ---------------------------------------------------------- several new tokens --

@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads,group", SHARED)
@pytest.mark.parametrize("causal", [True, False])
def test_several_tokens_that_share(page, dim, heads, group, src, fmt, causal):
    """As many new tokens as share a prefix still (96 rows of a cache head, 64 of 64 columns)
    and fewer, by the kernels that the sizes choose: none at all, more rows than tokens, new
    ones that reach into the prefix."""
    most = (64 if dim == 64 else 96) // group
    lens, table, groups, shared, pages = forked(PLAN, page, 610)
    assert lens[4] == 5 and lens[11] == 0
    cache = random_cache(pages, heads, dim, page, fmt, 611)
    spoil(cache, lens, table)
    for bound in sorted({most, min(most, 7), min(most, 2)}):
        new = [min(n, 1 + 11 * b % bound) for b, n in enumerate(lens)]
        new[3], new[4], new[5], new[7], new[11] = 0, bound, min(lens[5], bound), bound, min(3, bound)
        q = randn((sum(new), heads * group, dim), 612, src)
        for kw in ({"max_group": 7}, {}):
            check_shared(q, cache, lens, table, groups, shared, new, causal=causal, max_q_len=bound, **kw)


@pytest.mark.parametrize("key", [True, False])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim", [(16, 64), (64, 64), (64, 128), (128, 256), (32, 128)])
def test_nan_that_some_rows_see(page, dim, src, key, wide):
    """A NaN code among new tokens is one in the rows that see it, by whole rows (a key's) or in
    its column (a value's), and in no other: in a sequence's own tokens, in a prefix that a short
    sequence sees in part, at a tile's first and last token."""
    lens, table, groups, shared, pages = forked([(384, [70, 200, -230, 40, 1])], page, 620)
    clean = random_cache(pages, 2, dim, page, "fp8", 621)
    spoil(clean, lens, table)
    new = [6, 7, 5, 9, 1]
    starts = [sum(new[:b]) for b in range(6)]
    q = randn((starts[5], 8, dim), 622, src)
    o, a, reach = O.attention(q, clean, ints(lens), table, ints(starts))
    for owner, pos in ((0, 450), (1, 577), (1, 583), (1, 400), (3, 419), (2, 150), (2, 153), (0, 383), (0, 448)):
        p, slot = table[owner, pos // page].item(), pos % page
        cache = KV.KV8Cache(*(t.clone() for t in clean))
        if key:
            cache.k.view(torch.uint8)[p, 1, slot, 5] = 0x7f
        else:
            cache.v.view(torch.uint8)[p, 1, 5, slot] = 0xff
        sees = torch.zeros(o.shape, dtype=torch.bool)
        for b, n in enumerate(lens):
            for i in range(new[b]):
                if pos <= n - new[b] + i and table[b, pos // page] == p:
                    sees[starts[b] + i, 4:, slice(None) if key else slice(5, 6)] = True
        assert sees.any()
        got = check_shared(q, cache, lens, table, groups, shared, new, got_only=True, max_q_len=9).cpu()
        assert torch.equal(got.isnan(), sees), (owner, pos)
        within(got.masked_fill(sees, 0), o.masked_fill(sees, 0), a, reach)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_infinite_queries(dim, src, wide):
    """Rows of infinities, and of one, whose scores have +infinity among them: NaN; the others'
    rows are their own."""
    lens, table, groups, shared, pages = forked([(700, [1, 70, 200, 9, 5, 3])], 64, 630)
    cache = random_cache(pages, 1, dim, 64, "int8", 631)
    q = randn((6, 4, dim), 632, src)
    o, a, reach = O.attention(q, cache, ints(lens), table)
    q[3], q[5, :, 0] = math.inf, -math.inf
    got = check_shared(q, cache, lens, table, groups, shared, got_only=True)
    assert got[3].isnan().all() and got[5].isnan().all()
    others = [0, 1, 2, 4]
    within(got[others], o[others], a[others], reach[others])


def test_prompts_of_very_many_rows():
    """Prompts together past the rows that share a prefix: kv8_attention's result."""
    seqs, new, hq, dim, page = 140, 500, 64, 64, 64
    assert seqs * new * hq > 1 << 22
    table = torch.arange(seqs * 8, dtype=torch.int32).view(seqs, 8)
    table[:, 0] = 0                              # a shared first page
    cache = to(random_cache(seqs * 8, 1, dim, page, "int8", 640), DEV)
    q = torch.randn((seqs * new, hq, dim), device=DEV, generator=torch.Generator(DEV).manual_seed(641)).to(torch.bfloat16)
    lens, starts = torch.full((seqs,), new, dtype=torch.int32, device=DEV), torch.arange(seqs + 1, device=DEV).int() * new
    kw = dict(q_starts=starts, max_q_len=new)
    got = A.kv8_shared_attention(q, cache, lens, table.to(DEV), ints([0, seqs]).to(DEV), ints([64]).to(DEV), **kw)
    assert torch.equal(got, A.kv8_attention(q, cache, lens, table.to(DEV), **kw))
    with pytest.raises(N.DslError, match="at most 2"):
        A.kv8_shared_attention(q, cache, lens, table.to(DEV), ints([0, seqs]).to(DEV), ints([64]).to(DEV), q_starts=starts,
                               max_q_len=1)


@pytest.mark.parametrize("more", [0, 1])
def test_fork_next_to_the_bound(more):
    """The largest table and counts that one workgroup keeps the books of, and one page more."""
    lens, width = [700, 33, 0, 1601], 120
    table, refs = pool(lens, 16, 0, 650, width=width)
    spare = 32768 + more - (4 + 7) * width - len(refs)
    refs = torch.cat([refs, torch.zeros(spare, dtype=torch.int32)])
    cache = random_cache(len(refs), 1, 64, 16, "int8", 651)
    check_fork(cache, ints(lens), table, ints([0, 0, 3, 1, 3, 0, -1]), refs, 40)

"""Several continuations of a prompt at their edges on the GPU: pages that are missing before
others and scores that overflow, with every number of query rows a wave."""
import random

import pytest
import torch

from dsl_tool_amd import attention as A
from oracle import serving as O
from tests.test_gpu_generate import check_shared, forked, ints, spoil
from tests.test_gpu_generate_steps import wide  # noqa: F401
from tests.test_gpu_serving import DEV, randn, random_cache, to, within

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

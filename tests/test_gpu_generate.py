"""What generates several continuations of a prompt, on the GPU against plain
forms: forked and compacted pages, attention over shared prefixes, rotary
positions, log probabilities, and a run of them together."""
import math
import random

import pytest
import torch

from dsl_tool_amd import attention as A
from dsl_tool_amd import kvcache as KV
from dsl_tool_amd import logprobs as LP
from dsl_tool_amd import rotary as R
from oracle import generating as GO
from oracle import serving as O
from tests.test_gpu_serving import DEV, HALF, gen, random_cache, randn, same_cache, to, within
from tests.test_gpu_serving import spoil as spoil_all

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32)


def equal(got, want):
    for a, b, name in zip(got, want, got._fields):
        assert a.dtype == torch.int32 and torch.equal(a.cpu(), b), name


# ------------------------------------------------------------------ pages --

def pool(lens, page, spare, seed, shared=0, width=None):
    """(table, refs) of sequences that share their first pages by pairs."""
    rng, rows, at = random.Random(seed), [], 0
    for b, n in enumerate(lens):
        mine = -(-max(n, 0) // page)
        same = min(shared, len(rows[-1]), max(n, 0) // page) if b % 2 else 0
        rows.append((rows[-1][:same] if same else []) + list(range(at, at + mine - same)))
        at += mine - same
    pages = at + spare
    order = list(range(pages))
    rng.shuffle(order)
    width = width or max([len(r) for r in rows] + [1])
    table = ints([[order[p] for p in r][:width] + [-1] * (width - len(r)) for r in rows]).view(len(lens), width)
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in table[table >= 0].tolist():
        refs[p] += 1
    return table, refs


def check_fork(cache, lens, table, parents, refs, new, got_cache=None):
    """Every result and byte of the cache against the oracle's; the inputs as they were."""
    want_cache = to(cache, "cpu")
    dev = to(cache, DEV) if got_cache is None else got_cache
    given = [t.to(DEV) for t in (lens, table, parents, refs)]
    before = [t.clone() for t in given]
    more = new.to(DEV) if isinstance(new, torch.Tensor) else new
    got = KV.kv8_fork(dev, *given, new=more)
    want = GO.fork(want_cache, lens, table, parents, refs, new)
    equal(got, want)
    same_cache(dev, want_cache)
    assert all(torch.equal(a, b) for a, b in zip(given, before))
    # every count is that of the table's entries, and of what the caller kept beside them
    held = torch.zeros_like(refs)
    for p in want[1][want[1] >= 0].tolist():
        held[p] += 1
    kept = refs.clone()
    for p in table[(table >= 0) & (table < len(refs))].tolist():
        kept[p] -= 1
    assert torch.equal(want[2], held + kept)
    return got, dev


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 3), (32, 256, 1), (64, 128, 2), (128, 64, 1), (256, 128, 2)])
def test_fork(page, dim, heads, fmt):
    """Children of none, of one and of several parents; full and partly filled last
    pages; lengths of zero and one."""
    lens = [3 * page, 0, 1, 2 * page + 5, page - 1, 4 * page + 1]
    table, refs = pool(lens, page, 9, 1, shared=2, width=8)
    cache = random_cache(len(refs), heads, dim, page, fmt, 2)
    for parents in ([0, 1, 2, 3, 4, 5], [3, 3, 3, 0, 0, 5, -1, 2], [5], [], [9, -7, 6], [4, 2, 4, 2]):
        for new in (0, 1, page, 2 * page + 1):
            check_fork(cache, ints(lens), table, ints(parents), refs, new)
    check_fork(cache, ints(lens), table, ints([0, 3, 3, 1]), refs, ints([0, 7, -3, 3 * page]))


def test_fork_lacks_pages():
    """Fewer free pages than are asked for, none, and rows with no room: the rest is
    right, and what lacked can be seen."""
    lens = [20, 33, 7]
    for spare in (0, 1, 3):
        table, refs = pool(lens, 16, spare, 3, width=3)
        cache = random_cache(len(refs), 2, 64, 16, "int8", 4)
        got, _ = check_fork(cache, ints(lens), table, ints([1, 1, 1, 0, 0, 2]), refs, 40)
        assert got.lacking.item() > 0
    got, _ = check_fork(cache, ints(lens), table, ints([0, 1, 2]), refs, 2 ** 31 - 1)
    assert got.seq_lens.tolist() == [2 ** 31 - 1] * 3


def test_fork_of_odd_tables():
    """Lengths past the row, negative ones, entries that are no page, entries behind a
    sequence's last, a row inside a wider table, pages that the caller keeps."""
    lens = [100, -5, 40, 16, 10]
    wide = ints([[3, 99, 5, 1], [7, 7, -1, 0], [2, -4, 10, 11], [4, 6, 8, 9], [2 ** 31 - 1, 12, 12, 13]])
    refs = torch.zeros(20, dtype=torch.int32)
    for p in wide[(wide >= 0) & (wide < 20)].tolist():
        refs[p] += 1
    refs[[14, 15]] += 1                          # kept by the caller
    refs[16] = -1                                # never free
    cache = random_cache(20, 1, 64, 16, "fp8", 5)
    check_fork(cache, ints(lens), wide, ints([0, 0, 1, 2, 2, 3, 4, 4]), refs, 5)
    held = torch.zeros(20, dtype=torch.int32)
    view = torch.zeros((5, 9), dtype=torch.int32)
    view[:, 2:6] = wide
    part = view.to(DEV)[:, 2:5]
    for p in wide[:, :3][(wide[:, :3] >= 0) & (wide[:, :3] < 20)].tolist():
        held[p] += 1
    got = KV.kv8_fork(to(cache, DEV), ints(lens).to(DEV), part, ints([0, 2, 4]).to(DEV), held.to(DEV), new=1)
    equal(got, GO.fork(to(cache, "cpu"), ints(lens), wide[:, :3], ints([0, 2, 4]), held, 1))


@pytest.mark.parametrize("seqs,children,ctx,spare", [(700, 1500, 300, 3000), (3, 5000, 900, 70000), (1100, 1, 1500, 0),
                                                     (1, 1, 300000, 40000)])
def test_fork_large(seqs, children, ctx, spare):
    """Tables and counts past what one workgroup keeps together, free pages past
    its reach in one step."""
    rng = random.Random(seqs)
    lens = [rng.randint(0, ctx) for _ in range(seqs)]
    table, refs = pool(lens, 16, spare, 6, shared=9)
    cache = random_cache(len(refs), 1, 64, 16, "int8", 7)
    parents = [rng.randint(-1, seqs) for _ in range(children)]
    check_fork(cache, ints(lens), table, ints(parents), refs, ints([rng.choice([0, 1, 40]) for _ in parents]))


def test_fork_steps():
    """A prompt, samples of it, beams over many steps: the pages never leak, and the last
    step frees all of them."""
    rng, page = random.Random(8), 16
    cache = to(random_cache(64, 1, 64, page, "int8", 9), DEV)
    lens, table, refs = ints([]), torch.zeros((0, 12), dtype=torch.int32), torch.zeros(64, dtype=torch.int32)
    lens, table, refs = ints([0]), torch.full((1, 12), -1, dtype=torch.int32), refs
    for parents, new in [([-1], 37), ([0] * 6, 1)] + [([rng.randrange(6) for _ in range(6)], rng.choice([1, 1, 3, 16]))
                                                      for _ in range(12)] + [([-1], 0)]:
        got, _ = check_fork(to(cache, "cpu"), lens, table, ints(parents), refs, new, got_cache=cache)
        lens, table, refs = (t.cpu() for t in got[:3])
    assert (refs == 0).all() and lens.tolist() == [0]


def test_fork_in_a_graph():
    """Captured, and replayed over changed parents with eager work between; each replay
    as the eager call."""
    page, lens = 16, [50, 33, 16, 7]
    table, refs = pool(lens, page, 12, 10, width=8)
    clean = random_cache(len(refs), 2, 64, page, "int8", 11)
    cache, given = to(clean, DEV), [t.to(DEV) for t in (ints(lens), table, ints([0, 1, 2, 3]), refs)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        KV.kv8_fork(cache, *given, new=1)
        KV.kv8_compact(cache, given[1], given[3])
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step = KV.kv8_fork(cache, *given, new=1)
        packed = KV.kv8_compact(cache, step.page_table, step.refs)
    for parents in ([0, 0, 0, 1], [3, 2, 1, 0], [-1, 1, 1, 1], [2, 2, 0, 0]):
        given[2].copy_(ints(parents))
        for a, b in zip(cache, clean):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want_cache = to(clean, "cpu")
        want = GO.fork(want_cache, ints(lens), table, ints(parents), refs, 1)
        equal(step, want)
        equal(packed, GO.compact(want_cache, want[1], want[2]))
        same_cache(cache, want_cache)
        eager = to(clean, DEV)
        torch.cuda.synchronize()
        equal(KV.kv8_fork(eager, *given, new=1), want)


def check_compact(cache, table, refs):
    want_cache, dev = to(cache, "cpu"), to(cache, DEV)
    given = [table.to(DEV), refs.to(DEV)]
    before = [t.clone() for t in given]
    got = KV.kv8_compact(dev, *given)
    equal(got, GO.compact(want_cache, table, refs))
    same_cache(dev, want_cache)
    assert all(torch.equal(a, b) for a, b in zip(given, before))


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("page,dim,heads", [(16, 64, 3), (32, 256, 1), (64, 128, 2), (256, 128, 1)])
def test_compact(page, dim, heads, fmt):
    rng = random.Random(20)
    for pages, share in ((1, 1.0), (2, 0.5), (37, 0.5), (40, 0.0), (40, 1.0), (64, 0.1), (51, 0.9)):
        refs = ints([rng.choice([1, 2, 7]) if rng.random() < share else rng.choice([0, 0, -2]) for _ in range(pages)])
        live = [p for p in range(pages) if refs[p] > 0] or [0]
        table = ints([[rng.choice(live + [-1, pages, rng.randrange(pages)]) for _ in range(5)] for _ in range(3)])
        check_compact(random_cache(pages, heads, dim, page, fmt, 21), table, refs)


def test_compact_many_pages():
    rng = random.Random(22)
    refs = ints([rng.choice([0, 0, 1]) for _ in range(30011)])
    table = torch.randint(-1, 30011, (257, 70), generator=gen(23), dtype=torch.int32)
    check_compact(random_cache(30011, 1, 64, 16, "int8", 24), table, refs)


def test_compact_of_nothing():
    c = KV.new_kv8_cache(0, 2, 64, page=16, device=DEV)
    none = torch.zeros((0,), dtype=torch.int32, device=DEV)
    got = KV.kv8_compact(c, torch.full((2, 3), 5, dtype=torch.int32, device=DEV), none)
    assert got.live.item() == 0 and (got.page_table == -1).all() and got.moved.numel() == 0
    got = KV.kv8_fork(c, ints([5, 16]).to(DEV), torch.full((2, 3), -1, dtype=torch.int32, device=DEV),
                      ints([1, 0, -1]).to(DEV), none, new=20)
    assert got.seq_lens.tolist() == [36, 25, 20] and (got.page_table == -1).all() and got.lacking.item() == 2 + 1 + 2
    c = KV.new_kv8_cache(4, 2, 64, page=16, device=DEV)
    got = KV.kv8_fork(c, none, torch.zeros((0, 3), dtype=torch.int32, device=DEV), ints([0, -1]).to(DEV),
                      ints([0, 2, 0, 0]).to(DEV), new=17)
    assert got.page_table.tolist() == [[0, 2, -1], [3, -1, -1]] and got.refs.tolist() == [1, 2, 1, 1]
    assert got.lacking.item() == 1


# -------------------------------------------------------------- attention --

def forked(plan, page, seed, width=None, spare=2):
    """Groups of (prefix, [tokens behind it]): (lens, table, group starts, shared
    lens, pages), every sequence's row whole."""
    rows, lens, starts, at = [], [], [0], 0
    for prefix, behind in plan:
        whole = prefix // page
        first = list(range(at, at + whole))
        at += whole
        for t in behind:
            n = max(prefix + t, 0)
            mine = max(-(-n // page) - whole, 0)
            rows.append((first + list(range(at, at + mine)))[:-(-n // page)])
            at += mine
            lens.append(n)
        starts.append(len(lens))
    order = list(range(at + spare))
    random.Random(seed).shuffle(order)
    width = width or max([len(r) for r in rows] + [1])
    table = ints([[order[p] for p in r] + [-1] * (width - len(r)) for r in rows])
    return lens, table, starts, [p for p, _ in plan], at + spare


def spoil(cache, lens, table):
    """NaN codes behind the last tokens that end in a page of their own: those of a
    shared one are other sequences' tokens."""
    page = cache.page
    own = [n > 0 and (table == table[b, (n - 1) // page]).sum() == 1 for b, n in enumerate(lens)]
    spoil_all(cache, [n if o else 0 for n, o in zip(lens, own)], table)


def check_shared(q, cache, lens, table, groups, shared, new=None, got_only=False, **kw):
    starts = None if new is None else ints([sum(new[:i]) for i in range(len(new) + 1)])
    lt = ints(lens)
    got = A.kv8_shared_attention(q.to(DEV), to(cache, DEV), lt.to(DEV), table.to(DEV), ints(groups).to(DEV),
                                 ints(shared).to(DEV), q_starts=None if starts is None else starts.to(DEV), **kw)
    assert got.shape == q.shape and got.dtype == q.dtype
    if not got_only:
        within(got, *O.attention(q, cache, lt, table, starts, **{k: v for k, v in kw.items() if k in ("scale", "causal")}))
    return got


SHARED = [(16, 64, 2, 1), (32, 128, 1, 7), (64, 128, 2, 4), (128, 256, 1, 2), (256, 64, 1, 16), (64, 256, 2, 8)]
PLAN = [(300, [1, 40, 7, 260]), (0, [5, 90]), (15, [3]), (1025, [1, -900, 2, 63, -1100]), (512, [1, 1, 1, 1, 1, 1, 1])]


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads,group", SHARED)
def test_shared_single_tokens(page, dim, heads, group, src, fmt):
    """Groups of one and several, prefixes of no whole page, sequences shorter
    than their group's prefix and empty ones."""
    lens, table, groups, shared, pages = forked(PLAN, page, 30)
    cache = random_cache(pages, heads, dim, page, fmt, 31)
    spoil(cache, lens, table)
    q = randn((len(lens), heads * group, dim), 32, src) * 1.5
    got = check_shared(q, cache, lens, table, groups, shared)
    assert (got[lens.index(0)] == 0).all()                     # a row that sees nothing
    for kw in ({"max_group": 7}, {"max_group": 0}, {"max_q_len": 1000}, {"causal": False}, {"scale": 0.3}):
        check_shared(q, cache, lens, table, groups, shared, **kw)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,heads,group", SHARED)
@pytest.mark.parametrize("causal", [True, False])
def test_shared_several_tokens(page, dim, heads, group, src, fmt, causal):
    """New tokens behind the prefix and reaching into it, none at all, more rows
    than tokens."""
    lens, table, groups, shared, pages = forked(PLAN, page, 40)
    new = [min(n, 1 + 11 * b % 60) for b, n in enumerate(lens)]
    new[3], new[5], new[9] = 0, lens[5], 200                    # none; a whole sequence; past a short one's start
    cache = random_cache(pages, heads, dim, page, fmt, 41)
    spoil(cache, lens, table)
    q = randn((sum(new), heads * group, dim), 42, src)
    check_shared(q, cache, lens, table, groups, shared, new, causal=causal, max_q_len=max(new), max_group=7)
    check_shared(q, cache, lens, table, groups, shared, new, causal=causal)


@pytest.mark.parametrize("seqs,group", [(1, 1), (3, 4), (16, 4), (33, 4), (64, 8), (300, 1)])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_shared_sizes_of_groups(seqs, group, fmt):
    """From a few rows of a prefix to many blocks of them, over a long prefix and a table
    far wider than it."""
    lens, table, groups, shared, pages = forked([(3000, [1 + 7 * b % 90 for b in range(seqs)])], 64, 50, width=200)
    for dim in (64, 128, 256):
        cache = random_cache(pages, 2, dim, 64, fmt, 51)
        spoil(cache, lens, table)
        for src in (torch.bfloat16, torch.float16):
            check_shared(randn((seqs, 2 * group, dim), 52, src) * 2, cache, lens, table, groups, shared, max_group=seqs)


def test_shared_outside_groups():
    """No groups, sequences before, between and behind them, groups of none, shared lengths
    past the row, negative, and of sequences that all are shorter."""
    lens, table, groups, shared, pages = forked([(100, [9]), (200, [3, 30, 1]), (70, [5, 5])], 16, 60)
    for fmt in ("int8", "fp8"):
        cache = random_cache(pages, 2, 64, 16, fmt, 61)
        spoil(cache, lens, table)
        q = randn((6, 4, 64), 62, torch.bfloat16)
        for g, s in (([0], []), ([1, 4], [200]), ([1, 1, 4, 4], [77, 200, 3]), ([4, 6], [70]), ([0, 1], [2 ** 31 - 1]),
                     ([1, 4, 6], [-5, 70]), ([1, 4, 6], [199, 69]), ([1, 4], [16]), ([-3, 1, 4, 99], [100, 200, 70])):
            check_shared(q, cache, lens, table, g, s)
    short, table2, g, s, pages = forked([(320, [-200, -100, -319, -320])], 16, 63, width=24)
    cache = random_cache(pages, 2, 64, 16, "int8", 64)
    check_shared(randn((4, 4, 64), 65, torch.bfloat16), cache, short, table2, g, s)


def test_shared_pages_that_are_none():
    """Entries of the prefix and behind it that name no page."""
    lens, table, groups, shared, pages = forked([(400, [30, 90, 200])], 16, 70)
    table[:, 3], table[:, 20], table[1, 26], table[2, 30:33] = -1, pages, 2 ** 31 - 1, -9
    for fmt in ("int8", "fp8"):
        cache = random_cache(pages, 1, 128, 16, fmt, 71)
        check_shared(randn((3, 4, 128), 72, torch.bfloat16), cache, lens, table, groups, shared)
        table[:, :25] = -1                                      # a prefix of nothing
        check_shared(randn((3, 4, 128), 72, torch.bfloat16), cache, lens, table, groups, shared)
        lens, table, groups, shared, pages = forked([(400, [30, 90, 200])], 16, 70)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_shared_nan(dim, src):
    """NaN in the prefix is one in every row that sees it; in a sequence's own tokens,
    in that one's; hidden ones and masked infinities leave no trace."""
    lens, table, groups, shared, pages = forked([(256, [1, 9, -100, 40])], 16, 80)
    clean = random_cache(pages, 2, dim, 16, "fp8", 81)
    q = randn((4, 8, dim), 82, src)
    o, a, reach = O.attention(q, clean, ints(lens), table)
    for pos, rows in ((200, (0, 1, 3)), (100, (0, 1, 2, 3)), (260, (1,))):
        owner = 1 if pos >= 256 else 0
        p, slot = table[owner, pos // 16].item(), pos % 16
        if pos < 256:
            assert (table[[0, 1, 3], pos // 16] == p).all()
        for key in (True, False):
            cache = to(clean, "cpu")
            cache = KV.KV8Cache(*(t.clone() for t in cache))
            if key:
                cache.k.view(torch.uint8)[p, 1, slot, 5] = 0x7f
            else:
                cache.v.view(torch.uint8)[p, 1, 5, slot] = 0xff
            got = check_shared(q, cache, lens, table, groups, shared, got_only=True).cpu()
            sees = torch.zeros((4, 8, dim), dtype=torch.bool)
            for r in rows:
                if lens[r] > pos:
                    sees[r, 4:, slice(None) if key else slice(5, 6)] = True
            assert torch.equal(got.isnan(), sees)
            fine = torch.where(sees, torch.zeros_like(got), got)
            within(fine, o.masked_fill(sees, 0), a, reach)
    # behind the last token: NaN codes and infinite scales of pages that no row sees
    cache = KV.KV8Cache(*(t.clone() for t in clean))
    spoil(cache, lens, table)
    unused = [p for p in range(pages) if not (table == p).any()]
    cache.k_scale[unused], cache.v_scale[unused] = math.inf, math.nan
    check_shared(q, cache, lens, table, groups, shared)


def test_shared_layouts_streams_and_repeats():
    """Queries inside a projection, a result inside a wider tensor, 64-bit
    tables, another stream, several times: bit for bit."""
    lens, table, groups, shared, pages = forked([(900, [3, 60, 9]), (40, [1, 2])], 32, 90)
    cache = to(random_cache(pages, 2, 128, 32, "int8", 91), DEV)
    qkv = randn((5, 12, 128), 92, torch.bfloat16).to(DEV)
    args = [cache, ints(lens).to(DEV), table.to(DEV), ints(groups).to(DEV), ints(shared).to(DEV)]
    want = A.kv8_shared_attention(qkv[:, :8].contiguous(), *args)
    wide = torch.zeros((5, 10, 136), dtype=torch.bfloat16, device=DEV)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = [A.kv8_shared_attention(qkv[:, :8], *args) for _ in range(4)]
        long = [args[0]] + [t.long() for t in args[1:]]
        got.append(A.kv8_shared_attention(qkv[:, :8], *long, out=wide[:, 1:9, :128]))
        odd = torch.zeros((5, 8, 129), dtype=torch.bfloat16, device=DEV)[:, :, 1:].copy_(qkv[:, :8])
        got.append(A.kv8_shared_attention(odd, *args))
    side.synchronize()
    assert all(torch.equal(g, want) for g in got)
    assert (wide[:, 0] == 0).all() and (wide[:, 9] == 0).all() and (wide[:, :, 128:] == 0).all()
    empty = A.kv8_shared_attention(qkv[:0, :8], cache, ints([]).to(DEV), table[:0].to(DEV), ints([0]).to(DEV), ints([]).to(DEV))
    assert empty.shape == (0, 8, 128)


def test_shared_graphs_with_one_pool():
    """Two captured graphs whose workspaces share memory, replayed in turn, each
    replay as the eager call."""
    lens, table, groups, shared, pages = forked([(700, [1, 50]), (90, [4, 4, 4])], 16, 95)
    cache = to(random_cache(pages, 2, 64, 16, "int8", 96), DEV)
    args = [ints(lens).to(DEV), table.to(DEV), ints(groups).to(DEV), ints(shared).to(DEV)]
    q = randn((5, 8, 64), 97, torch.bfloat16).to(DEV)
    x = randn((5, 3001), 98).to(DEV)
    ids = ints([1, 2, 3, 4, 5]).to(DEV)
    graphs, outs = [torch.cuda.CUDAGraph() for _ in range(2)], []
    A.kv8_shared_attention(q, cache, *args)
    LP.token_logprobs(x, ids, top=4)
    torch.cuda.synchronize()
    with torch.cuda.graph(graphs[0]):
        outs.append(A.kv8_shared_attention(q, cache, *args))
    with torch.cuda.graph(graphs[1], pool=graphs[0].pool()):
        outs.append(LP.token_logprobs(x, ids, top=4))
    for step in range(4):
        q.copy_(randn((5, 8, 64), 200 + step, torch.bfloat16))
        x.copy_(randn((5, 3001), 300 + step))
        args[0].copy_(ints([n - step for n in lens]))
        graphs[step % 2].replay()
        graphs[1 - step % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], A.kv8_shared_attention(q, cache, *args))
        assert all(torch.equal(a, b) for a, b in zip(outs[1], LP.token_logprobs(x, ids, top=4)))


# ----------------------------------------------------------------- rotary --

def check_turned(got, want, x, magnitude=1.0, half=None):
    """Half a step of the result; and of each of its two terms the cosine's and the
    product's error: 2^-21 of the head's largest value."""
    top = x.double().abs().amax(-1, keepdim=True) * abs(magnitude) + x.double().abs().amax(-1, keepdim=True)
    tol = want.abs() * HALF[got.dtype] + top * 2.0 ** -21 + 2.0 ** -25
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("adjacent", [False, True])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,hq,hk,dim,half", [(1, 4, 1, 128, 64), (7, 3, 3, 64, 32), (33, 8, 2, 128, 16), (5, 2, 1, 256, 120),
                                                 (3, 2, 2, 80, 17), (2, 1, 1, 6, 3), (4, 2, 1, 64, 0), (9, 1, 1, 1024, 512),
                                                 (700, 5, 1, 128, 64), (3, 2, 1, 7, 2)])
def test_rotary(rows, hq, hk, dim, half, src, adjacent):
    q, k = randn((rows, hq, dim), 1, src), randn((rows, hk, dim), 2, src) * 3
    freqs = R.rotary_freqs(2 * half, device="cpu")
    pos = torch.randint(0, 5000, (rows,), generator=gen(3))
    for p in (pos, pos.to(torch.int32)):
        a, b = R.rotary(q.to(DEV), k.to(DEV), p.to(DEV), freqs.to(DEV), adjacent=adjacent)
        assert a.dtype == src and a.is_contiguous()
        check_turned(a, GO.rotary(q, pos, freqs, adjacent=adjacent), q)
        check_turned(b, GO.rotary(k, pos, freqs, adjacent=adjacent), k)
        if 2 * half < dim:
            assert torch.equal(a[..., 2 * half:].cpu(), q[..., 2 * half:])
    a, none = R.rotary(q.to(DEV), None, pos.to(DEV), freqs.to(DEV), adjacent=adjacent, magnitude=1.25)
    assert none is None
    turned = GO.rotary(q, pos, freqs, adjacent=adjacent, magnitude=1.25)
    check_turned(a, turned, q, 1.25)


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_axes(interleaved):
    """Several axes, each with its own positions; axes of no pairs; axes that are none."""
    q, k = randn((50, 4, 128), 4, torch.bfloat16), randn((50, 2, 128), 5, torch.bfloat16)
    freqs = R.rotary_freqs(128, 1e6, device="cpu")
    for sections in ([16, 24, 24], [64], [0, 32, 32], [1, 2, 3, 58]):
        axes = R.rotary_axes(sections, interleaved=interleaved, device="cpu")
        assert axes.shape == (64,) and [int((axes == a).sum()) for a in range(len(sections))] == sections
        pos = torch.randint(0, 1 << 20, (len(sections), 50), generator=gen(6))
        a, b = R.rotary(q.to(DEV), k.to(DEV), pos.to(DEV), freqs.to(DEV), axis_of=axes.to(DEV))
        check_turned(a, GO.rotary(q, pos, freqs, axes), q)
        check_turned(b, GO.rotary(k, pos, freqs, axes), k)
    axes[::7] = -1
    axes[1::7] = 99
    a, _ = R.rotary(q.to(DEV), None, pos.to(DEV), freqs.to(DEV), axis_of=axes.to(DEV))
    check_turned(a, GO.rotary(q, pos, freqs, axes), q)
    assert R.rotary_axes([2, 1, 1], interleaved=True, device="cpu").tolist() == [0, 1, 2, 0]


def test_rotary_far_positions():
    """Positions with more digits than fp32 has, negative ones, zero."""
    pos = torch.tensor([0, 1, 2 ** 24 + 1, 2 ** 31 - 1, 10 ** 12 + 7, -5, -2 ** 31])
    q = randn((7, 2, 64), 7, torch.float16)
    freqs = R.rotary_freqs(64, 500000.0, device="cpu")
    a, _ = R.rotary(q.to(DEV), None, pos.to(DEV), freqs.to(DEV))
    check_turned(a, GO.rotary(q, pos, freqs), q)
    assert torch.equal(a[0].cpu(), q[0])
    small = pos.clamp(-2 ** 31, 2 ** 31 - 1)
    b, _ = R.rotary(q.to(DEV), None, small.to(torch.int32).to(DEV), freqs.to(DEV))
    check_turned(b, GO.rotary(q, small, freqs), q)


def test_rotary_views_in_place_and_streams():
    """Heads inside a projection, odd offsets, broadcast rows, strided positions, in
    place: as from contiguous tensors, bit for bit, and nothing beside them."""
    qkv = randn((21, 9, 64), 8, torch.bfloat16).to(DEV)
    before = qkv.clone()
    freqs = R.rotary_freqs(48, device=DEV)
    pos = torch.randint(0, 9000, (21, 2), generator=gen(9)).to(DEV)
    a, b = R.rotary(qkv[:, :4].contiguous(), qkv[:, 4:6].contiguous(), pos[:, 1].contiguous(), freqs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        x, y = R.rotary(qkv[:, :4], qkv[:, 4:6], pos[:, 1], freqs)
        odd = torch.zeros((21, 4, 65), dtype=torch.bfloat16, device=DEV)[:, :, 1:].copy_(qkv[:, :4])
        z, _ = R.rotary(odd, None, pos.t()[1:], freqs)
        w, _ = R.rotary(qkv[:1, :4].expand(21, 4, 64), None, pos[:, 1], freqs)
        v, _ = R.rotary(qkv[:1, :4].repeat(21, 1, 1), None, pos[:, 1], freqs)
        r = R.rotary(qkv[:, :4], qkv[:, 4:6], pos[:, 1], freqs, inplace=True)
        s, _ = R.rotary(odd, None, pos[:, 1], freqs.float(), inplace=True)
    side.synchronize()
    assert torch.equal(x, a) and torch.equal(y, b) and torch.equal(z, a) and torch.equal(w, v)
    assert r[0].data_ptr() == qkv.data_ptr() and torch.equal(qkv[:, :4], a) and torch.equal(qkv[:, 4:6], b)
    assert torch.equal(qkv[:, 6:], before[:, 6:])
    check_turned(s, GO.rotary(before[:, :4].cpu(), pos[:, 1].cpu(), freqs.float().cpu()), before[:, :4].cpu())
    e = R.rotary(qkv[:0, :4], qkv[:0, 4:6], pos[:0, 1], freqs)
    assert e[0].shape == (0, 4, 64) and e[1].shape == (0, 2, 64)


# ----------------------------------------------------------- log probabilities --

def check_logprobs(x, ids, top, scale=1.0, got=None):
    """fp32 throughout: the result's rounding, 2^-23 of the scores' range, and
    2^-19 for the sums."""
    r = LP.token_logprobs(x.to(DEV), ids.to(DEV), top=top, scale=scale) if got is None else got
    want = GO.logprobs(x, ids.view(len(x), -1), top, scale)
    assert r.logp.shape == ids.shape and r.top_ids.dtype == torch.int32
    assert torch.equal(r.top_ids.cpu(), want[3])
    for g, w in ((r.logp.view(len(x), -1), want[0]), (r.entropy, want[1]), (r.top_logp, want[2])):
        g = g.cpu().double()
        assert torch.equal(g.isneginf(), w.isneginf())
        fine = ~w.isneginf()
        assert ((g - w)[fine].abs() <= w[fine].abs() * 2.0 ** -22 + 2.0 ** -19).all()
    return r


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 5, 5), (2, 40, 32), (7, 1000, 0), (5, 4099, 20), (2, 33000, 32),
                                            (1, 100003, 7), (600, 77, 3)])
def test_logprobs(rows, vocab, top, src):
    x = (randn((rows, vocab), 1) * 3).to(src)
    for n in ((), (4,)):
        ids = torch.randint(0, vocab, (rows,) + n, generator=gen(2), dtype=torch.int32)
        for scale in (1.0, 0.4, 2.5):
            check_logprobs(x, ids, top, scale)


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("vocab", [9, 700, 9001, 40000])
def test_logprobs_ties_and_masks(vocab, src):
    """Rows of one value, of zeros of both signs, of few values, rising and falling;
    mostly, all and all but one masked; values that pass the exponent's range."""
    i = torch.arange(vocab, dtype=torch.float32)
    rows = [torch.full((vocab,), 2.5), torch.where(i % 3 == 0, -0.0, 0.0), i % 4, (i / 64).floor(), -i / 32, i % 7 - 3,
            torch.where(i % 11 == 5, i / vocab, -math.inf), torch.full((vocab,), -math.inf),
            torch.where(i == vocab - 2, 1.0, -math.inf), torch.where(i == 3, 60000.0, -60000.0),
            torch.full((vocab,), -60000.0)]
    x = torch.stack(rows).to(src)
    ids = torch.tensor([[0, vocab - 1, vocab - 2, -1, vocab, 2 ** 31 - 1, -2 ** 31]] * len(rows), dtype=torch.int32)
    r = check_logprobs(x, ids, min(32, vocab))
    assert r.top_ids[7].tolist() == list(range(min(32, vocab))) and r.entropy[7] == 0
    assert r.logp[8].tolist()[2] == 0 and r.entropy[8] == 0


def test_logprobs_not_numbers():
    """NaN or +inf make a row's results NaN, and no other row's; the best ones' numbers
    are those of the other logits, in the vocabulary."""
    x = randn((5, 20000), 5)
    clean = x.clone()
    x[1, 777], x[2, 0], x[3, 19999] = math.nan, math.inf, math.nan
    x[4] = math.nan
    ids = ints([5, 777, 5, 6, 7])
    r = LP.token_logprobs(x.to(DEV), ids.to(DEV), top=4)
    for t in (r.logp, r.entropy, r.top_logp):
        assert not t[0].isnan().any() and t[1:].isnan().all()
    best = GO.logprobs(clean, ids[:, None], 4)[3]
    assert r.top_ids[1].tolist() == best[1].tolist() and r.top_ids[2, 0] == 0 and r.top_ids[3].tolist() == best[3].tolist()
    assert r.top_ids[4].tolist() == [0, 1, 2, 3]


def test_logprobs_layouts():
    """Rows at any address, padded rows, 64-bit numbers, no ids, no rows, the same
    every time and on another stream."""
    base = randn((40, 5003), 6).to(torch.bfloat16).to(DEV)
    ids = torch.randint(0, 4000, (40,), generator=gen(7), dtype=torch.int32).to(DEV)
    for at in range(0, 9):
        view = base[:, at:at + 4001 + at]
        a = LP.token_logprobs(view, ids, top=5)
        check_logprobs(view.cpu(), ids.cpu(), 5, got=a)
        b = LP.token_logprobs(view.t().contiguous().t(), ids.long(), top=5)
        assert torch.equal(a.top_ids, b.top_ids)
        check_logprobs(view.cpu(), ids.cpu(), 5, got=b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = [LP.token_logprobs(view, ids, top=5) for _ in range(4)]
        long = LP.token_logprobs(view, (ids.long() + (1 << 32)), top=0)
        none = LP.token_logprobs(view, None, top=5)
        one = LP.token_logprobs(view[:1].expand(3, -1), ids[:3], top=2)
    side.synchronize()
    assert all(torch.equal(x, y) for r in again for x, y in zip(r, a))
    assert long.logp.isneginf().all() and none.logp.shape == (40, 0) and torch.equal(none.top_logp, a.top_logp)
    assert torch.equal(one.entropy, a.entropy[:1].expand(3))
    e = LP.token_logprobs(view[:0], ids[:0], top=2)
    assert e.logp.shape == (0,) and e.top_ids.shape == (0, 2)

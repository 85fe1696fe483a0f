"""Generating several continuations, the operators together as a program runs them: a
prompt, its samples, beams; eager and captured.  And attention over shared
prefixes with every number of query rows a wave, scales and sizes out of the ordinary."""
import math

import pytest
import torch

from dsl_tool_amd import attention as A
from dsl_tool_amd import fused as FU
from dsl_tool_amd import gemm as G
from dsl_tool_amd import kvcache as KV
from dsl_tool_amd import layer8 as L
from dsl_tool_amd import logprobs as LP
from dsl_tool_amd import quant as Q
from dsl_tool_amd import rotary as R
from oracle import generating as GO
from oracle import serving as O
from tests.test_gpu_generate import PLAN, check_logprobs, check_shared, equal, forked, ints, spoil
from tests.test_gpu_serving import DEV, randn, random_cache, same_cache, to, within

pytestmark = pytest.mark.gpu
HQ, HKV, DIM, HIDDEN, VOCAB, PAGE = 8, 2, 64, 512, 1001, 16


def new_layer(**kw):
    w = [(randn((n, k), 800 + i) / math.sqrt(k)).to(DEV, torch.bfloat16) for i, (n, k) in
         enumerate((((HQ + 2 * HKV) * DIM, HIDDEN), (HIDDEN, HQ * DIM)))]
    return L.Int8AttentionLayer(*w, (1 + 0.1 * randn((HIDDEN,), 802)).to(DEV), q_heads=HQ, kv_heads=HKV, dim=DIM, **kw)


class Model:
    """A layer with an embedding and an output product, its cache and its sequences."""

    def __init__(self, sections, width=12, pages=64):
        self.axis_of = R.rotary_axes(sections) if sections else None
        self.layer = new_layer(freqs=R.rotary_freqs(DIM), axis_of=self.axis_of)
        self.embed = randn((VOCAB, HIDDEN), 803, torch.bfloat16).to(DEV)
        self.head = (randn((VOCAB, HIDDEN), 804) / 10).to(DEV, torch.bfloat16)
        self.axes = len(sections) if sections else 1
        self.cache = KV.new_kv8_cache(pages, HKV, DIM, page=PAGE, device=DEV)
        self.lens = torch.zeros(1, dtype=torch.int32, device=DEV)
        self.table = torch.full((1, width), -1, dtype=torch.int32, device=DEV)
        self.refs = torch.zeros(pages, dtype=torch.int32, device=DEV)

    def positions(self, at):
        return at if self.axis_of is None else torch.stack([at // (a + 1) for a in range(self.axes)])

    def run(self, tokens, at, **kw):
        """(layer output, logits) of new tokens at their positions."""
        x = self.embed[tokens]
        out, h = self.layer(x, None, self.cache, self.lens, self.table, positions=self.positions(at), **kw)
        return out, (out + h) @ self.head.T

    def by_operators(self, tokens, at, cache, shared=None, **kw):
        """The same, operator by operator, over a cache of its own."""
        layer = self.layer
        codes, s, h = FU.add_rmsnorm_quant(self.embed[tokens], None, layer.norm)
        qkv = G.int8_gemm_packed(codes, layer.w_qkv, s, layer.s_qkv).view(len(tokens), -1, DIM)
        q, k = R.rotary(qkv[:, :HQ], qkv[:, HQ:HQ + HKV], self.positions(at), layer.freqs, axis_of=self.axis_of)
        KV.kv8_write(cache, k, qkv[:, HQ + HKV:], self.lens, self.table, **kw)
        if shared:
            o = A.kv8_shared_attention(q, cache, self.lens, self.table, *shared, **kw)
        else:
            o = A.kv8_attention(q, cache, self.lens, self.table, **kw)
        codes, s = Q.quant_int8_rows(o.view(len(tokens), -1))
        return G.int8_gemm_packed(codes, layer.w_out, s, layer.s_out)

    def fork(self, parents, new):
        step = KV.kv8_fork(self.cache, self.lens, self.table, parents, self.refs, new=new)
        self.lens, self.table, self.refs = step[:3]
        return step


@pytest.mark.parametrize("sections", [None, [8, 12, 12]])
def test_steps_together(sections):
    """A prompt of 37 tokens, five samples of it, beams over eight steps.  Each step: the
    layer is bit for bit its operators; over the shared prefix it is near what
    it is over unshared attention; log probabilities and pages are the oracle's.

    Near: a row of the attention quantized to int8 is off by at most 1.1% of its norm (a
    step of amax / 127 over sqrt(12), amax up to 4.8 deviations), its own rounding and
    that of the probabilities add 0.8% (two of bf16's 2^-8), on either side: 3.8%; the result's
    rounding, 2^-8 on either side: 4.6% of the norm.  The product with the weights, normal
    and 512 wide, stretches a difference by at most 1.3 more than the row (4 deviations of 1 / sqrt(2 x 512),
    both ways): 6% is allowed."""
    m = Model(sections)
    cpu = [t.cpu() for t in (m.lens, m.table, m.refs)]
    tokens = torch.arange(37, device=DEV) * 7 % VOCAB

    def fork(parents, new):
        cache = to(m.cache, "cpu")
        want = GO.fork(cache, *cpu[:2], parents.cpu(), cpu[2], new)
        step = m.fork(parents, new)
        equal(step, want)
        same_cache(m.cache, cache)
        assert step.lacking.item() == 0
        cpu[:] = want[:3]

    fork(ints([-1]).to(DEV), 37)
    twin = KV.KV8Cache(*(t.clone() for t in m.cache))
    kw = dict(q_starts=ints([0, 37]).to(DEV), max_q_len=37)
    out, logits = m.run(tokens, torch.arange(37, device=DEV), **kw)
    assert torch.equal(out, m.by_operators(tokens, torch.arange(37, device=DEV), twin, **kw))
    same_cache(m.cache, to(twin, "cpu"))
    check_logprobs(logits[:-1].cpu(), tokens[1:].cpu().int(), 3)
    best = LP.token_logprobs(logits[-1:], None, top=5)
    parents, tokens, scores = ints([0] * 5).to(DEV), best.top_ids[0].long(), best.top_logp[0].clone()
    groups, shared = ints([0, 5]).to(DEV), ints([37]).to(DEV)
    for _ in range(8):
        fork(parents, 1)
        at = (m.lens - 1).long()
        apart = KV.KV8Cache(*(t.clone() for t in m.cache))
        alone = KV.KV8Cache(*(t.clone() for t in m.cache))
        out, logits = m.run(tokens, at, group_starts=groups, shared_lens=shared, max_group=5)
        assert torch.equal(out, m.by_operators(tokens, at, apart, (groups, shared), ))
        same_cache(m.cache, to(apart, "cpu"))
        other = m.by_operators(tokens, at, alone).double()
        assert ((out.double() - other).norm(dim=-1) <= 0.06 * other.norm(dim=-1)).all()
        best = LP.token_logprobs(logits, None, top=5)
        check_logprobs(logits.cpu(), best.top_ids[:, 2].cpu().contiguous(), 5)
        total = (scores[:, None] + best.top_logp).flatten()
        scores, order = total.topk(5)
        parents, tokens = (order // 5).int(), best.top_ids.flatten()[order].long()
    fork(ints([-1]).to(DEV), 0)
    assert (m.refs == 0).all()


def test_steps_in_a_graph():
    """A step of four samples (layer, log probabilities, the next step's pages) captured,
    and replayed over changed tokens, lengths, tables and counts with eager work between: each replay
    bit for bit the eager step."""
    m = Model(None)
    m.fork(ints([-1]).to(DEV), 40)
    m.run(torch.arange(40, device=DEV), torch.arange(40, device=DEV), q_starts=ints([0, 40]).to(DEV), max_q_len=40)
    m.fork(ints([0] * 4).to(DEV), 1)
    groups, shared = ints([0, 4]).to(DEV), ints([40]).to(DEV)
    state = [m.lens, m.table, m.refs, torch.tensor([5, 6, 7, 8], device=DEV)]

    column = torch.tensor([0, 1, 2, 0], device=DEV)

    def step(cache, lens, table, refs, tokens):
        m.cache, m.lens, m.table, m.refs = cache, lens, table, refs
        _, logits = m.run(tokens, (lens - 1).long(), group_starts=groups, shared_lens=shared, max_group=4)
        best = LP.token_logprobs(logits, None, top=3)
        parents = best.top_ids[:, 0] % 4
        fork = KV.kv8_fork(cache, lens, table, parents, refs, new=1)
        return [*best, *fork, best.top_ids[parents.long(), column].long()]

    cache = m.cache
    still = [t.clone() for t in state]
    spare = KV.KV8Cache(*(t.clone() for t in cache))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(spare, *still)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(spare, *still)
    for _ in range(5):
        for a, b in zip(still, state):
            a.copy_(b)
        for a, b in zip(spare, cache):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        want = step(cache, *state)
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert a is None and b is None or torch.equal(a, b)
        same_cache(spare, to(cache, "cpu"))
        state = [want[-5], want[-4], want[-3], want[-1]]


def test_layer_refuses():
    with pytest.raises(ValueError, match="not by both"):
        new_layer(rotate=lambda q, k: (q, k), freqs=R.rotary_freqs(DIM))
    m = Model(None)
    x = m.embed[:1]
    with pytest.raises(ValueError, match="positions"):
        m.layer(x, None, m.cache, m.lens, m.table)
    with pytest.raises(ValueError, match="positions"):
        new_layer()(x, None, m.cache, m.lens, m.table, positions=ints([0]).to(DEV))
    with pytest.raises(ValueError, match="together"):
        m.layer(x, None, m.cache, m.lens, m.table, positions=ints([0]).to(DEV), group_starts=ints([0, 1]).to(DEV))
    with pytest.raises(ValueError, match="together"):
        m.layer(x, None, m.cache, m.lens, m.table, positions=ints([0]).to(DEV), max_group=1)


# ----------------------------------------------- attention over shared prefixes --

@pytest.fixture(params=["16", "32", "64"])
def wide(request, monkeypatch):
    """That many query rows a wave (64 of 256 columns do not exist: the rule's)."""
    monkeypatch.setenv("DSL_ATTN_SHARED_ROWS", request.param)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("page,dim,group", [(16, 64, 3), (64, 128, 4), (128, 128, 1), (32, 256, 4), (128, 256, 2)])
def test_rows_a_wave(page, dim, group, src, fmt, wide):
    """Single tokens and several, sequences' own tokens in blocks of any kind."""
    lens, table, groups, shared, pages = forked(PLAN, page, 400)
    cache = random_cache(pages, 2, dim, page, fmt, 401)
    spoil(cache, lens, table)
    check_shared(randn((len(lens), 2 * group, dim), 402, src) * 1.5, cache, lens, table, groups, shared)
    new = [min(n, 1 + 5 * b % 9) for b, n in enumerate(lens)]
    check_shared(randn((sum(new), 2 * group, dim), 403, src), cache, lens, table, groups, shared, new, max_q_len=9)


@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_many_sequences_and_groups(fmt, wide):
    """More units than are looked at at a time: 150 groups of one and two, 200 sequences, and own
    tokens of as many heads as launch by themselves."""
    plan = [(16 * (b % 7) + b % 3, [1 + b % 5] + [30] * (b % 3 == 0)) for b in range(150)]
    lens, table, groups, shared, pages = forked(plan, 16, 410)
    cache = random_cache(pages, 2, 64, 16, fmt, 411)
    spoil(cache, lens, table)
    for max_group in (2, 200):
        check_shared(randn((len(lens), 8, 64), 412, torch.bfloat16), cache, lens, table, groups, shared, max_group=max_group)


@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("fmt", ["int8", "fp8"])
def test_odd_scales(fmt, dim, src, wide):
    """Page scales of 0, below 0 and far apart; a scale of 0, below 0 and large of the
    scores."""
    lens, table, groups, shared, pages = forked([(900, [1, 70, 200, 9, 5])], 64, 420)
    cache = random_cache(pages, 1, dim, 64, fmt, 421)
    for i, page in enumerate(table[1].tolist()):
        if page >= 0:
            cache.k_scale[page] *= (1.0, 0.0, -1.0, 1e-3, 1e-30)[i % 5]
            cache.v_scale[page] *= (1.0, -1.0, 0.0, 100.0, 1e-6)[i % 5]
    q = randn((5, 4, dim), 422, src)
    for scale in (None, 0.0, -0.1, 0.7):
        check_shared(q, cache, lens, table, groups, shared, scale=scale)


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("src", [torch.bfloat16, torch.float16])
def test_large_and_odd_queries(dim, src, wide):
    """Queries of very different sizes to a row; and a row of infinities and one of NaN,
    which are their own rows' alone."""
    lens, table, groups, shared, pages = forked([(700, [1, 70, 200, 9, 5, 3])], 64, 430)
    cache = random_cache(pages, 1, dim, 64, "int8", 431)
    q = randn((6, 4, dim), 432, src)
    q[1] *= 2.0 ** -12
    q[2] = q[2] * 16
    check_shared(q, cache, lens, table, groups, shared)
    o, a, reach = O.attention(q, cache, ints(lens), table)
    bad = q.clone()
    bad[3], bad[5] = math.inf, math.nan
    got = check_shared(bad, cache, lens, table, groups, shared, got_only=True)
    others = [0, 1, 2, 4]
    within(got[others], o[others], a[others], reach[others])
    assert got[5].isnan().all()


def test_rows_behind_the_last_sequence(wide):
    """Rows that no sequence has stay in bounds and leave the others' results alone."""
    lens, table, groups, shared, pages = forked([(300, [4, 9, 30])], 16, 440)
    cache = random_cache(pages, 2, 128, 16, "fp8", 441)
    q = randn((9, 8, 128), 442, torch.bfloat16)
    args = [to(cache, DEV), *(t.to(DEV) for t in (ints(lens), table, ints(groups), ints(shared)))]
    some = A.kv8_shared_attention(q[:6].to(DEV), *args, q_starts=ints([0, 1, 4, 6]).to(DEV), max_q_len=3)
    got = A.kv8_shared_attention(q.to(DEV), *args, q_starts=ints([0, 1, 4, 6]).to(DEV), max_q_len=3)
    assert torch.equal(got[:6], some)


def test_calls_at_once(wide):
    """Two streams at once, each with its own sequences of one cache: as one after the other."""
    lens, table, groups, shared, pages = forked([(2000, [4] * 20), (500, [9] * 12)], 64, 450)
    cache = to(random_cache(pages, 2, 128, 64, "int8", 451), DEV)
    q = randn((32, 8, 128), 452, torch.bfloat16).to(DEV)
    parts = [(q[:20], ints(lens[:20]).to(DEV), table[:20].to(DEV), ints([0, 20]).to(DEV), ints(shared[:1]).to(DEV)),
             (q[20:], ints(lens[20:]).to(DEV), table[20:].to(DEV), ints([0, 12]).to(DEV), ints(shared[1:]).to(DEV))]
    want = [A.kv8_shared_attention(x, cache, *rest) for x, *rest in parts]
    streams = [torch.cuda.Stream() for _ in parts]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(6):
        for i, (s, (x, *rest)) in enumerate(zip(streams, parts)):
            with torch.cuda.stream(s):
                got[i].append(A.kv8_shared_attention(x, cache, *rest))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(x, b) for x in a)


def test_long_cache():
    """Pages whose bytes lie past 2^32 of the cache (a table that skips the ones before)."""
    pages, page, heads, dim = 33000, 256, 4, 128
    cache = KV.new_kv8_cache(pages, heads, dim, page=page, device=DEV)          # 4.3 GB of keys
    small = random_cache(12, heads, dim, page, "int8", 460)
    lens, table, groups, shared, count = forked([(1500, [3, 260, 40])], page, 461, spare=0)
    assert count <= 12
    far = torch.arange(pages - 12, pages)
    for a, b in zip(cache, small):
        a[pages - 12:] = b.to(DEV)
    moved = torch.where(table >= 0, far[table.clamp_min(0).long()].int(), table)
    q = randn((3, 16, dim), 462, torch.bfloat16)
    want = check_shared(q, small, lens, table, groups, shared)
    args = [moved.to(DEV), ints(groups).to(DEV), ints(shared).to(DEV)]
    assert torch.equal(A.kv8_shared_attention(q.to(DEV), cache, ints(lens).to(DEV), *args), want)
    refs = torch.zeros(pages, dtype=torch.int32)
    for p in moved[moved >= 0].tolist():
        refs[p] += 1
    fork = KV.kv8_fork(cache, ints(lens).to(DEV), moved.to(DEV), ints([1, 0, 1, 2]).to(DEV), refs.to(DEV), new=1)
    assert fork.lacking.item() == 0
    packed = KV.kv8_compact(cache, fork.page_table, fork.refs)
    front = KV.KV8Cache(*(t[:packed.live.item()].cpu() for t in cache))
    new_lens = fork.seq_lens.cpu() - 1
    q4 = torch.stack([q[1], q[0], q[1], q[2]])
    got = A.kv8_attention(q4.to(DEV), KV.KV8Cache(*(t[:packed.live.item()] for t in cache)), new_lens.to(DEV),
                          packed.page_table)
    o, a, reach = O.attention(q4, front, new_lens, packed.page_table.cpu())
    within(got, o, a, reach)
    first = O.attention(q, small, ints(lens), table)[0]
    for child, parent in enumerate((1, 0, 1, 2)):
        assert torch.allclose(o[child], first[parent], rtol=1e-10, atol=1e-12)


def test_long_groups_of_short_sequences(wide):
    """100 sequences that all are shorter than their group's prefix, the longest among the last:
    it is the one whose row has the prefix."""
    lens, table, groups, shared, pages = forked([(640, [-640 + 3 * b for b in range(90)] + [-70, -1, -300] + [-640] * 7)],
                                                16, 470)
    cache = random_cache(pages, 1, 64, 16, "int8", 471)
    check_shared(randn((100, 2, 64), 472, torch.bfloat16), cache, lens, table, groups, shared)


def test_wide_table(wide):
    """A table far wider than any sequence, whose rounds would pass an int in steps of four tiles."""
    lens, table, groups, shared, pages = forked([(900, [1 + 5 * b for b in range(64)])], 256, 480)
    cache = random_cache(pages, 8, 64, 256, "int8", 481)
    q = randn((64, 8, 64), 482, torch.float16)
    far = torch.full((64, 1 << 22), -1, dtype=torch.int32, device=DEV)
    far[:, :table.shape[1]] = table.to(DEV)
    got = A.kv8_shared_attention(q.to(DEV), to(cache, DEV), ints(lens).to(DEV), far, ints(groups).to(DEV),
                                 ints(shared).to(DEV), max_group=64)
    within(got, *O.attention(q, cache, ints(lens), table))

"""CPU: what the entry points of several continuations refuse, at the C ABI and
in Python; nothing here reaches a GPU."""
import os

import pytest
import torch

from dsl_tool_amd import _native as N
from dsl_tool_amd import attention as A
from dsl_tool_amd import kvcache as KV
from dsl_tool_amd import logprobs as LP
from dsl_tool_amd import rotary as R
from tests.test_serving_host import CACHE, P, cache_cases, refused

Q = P + (1 << 20)     # another aligned pointer that is never read


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} is not built; run `python -m dsl_tool_amd.build`")
    return N.lib()


def refuse_each(lib, fn, good, cases):
    for at, value, status, word in cases:
        args = list(good)
        args[at] = value
        refused(lib, fn, args, status, word)


def test_shared_attention(lib):
    good = [P, 512, 128, 4] + CACHE + [P, P, 2, 2, P, 512, 128, 7, 4, 0.1, 1, 0, P, 1 << 30, None]
    for at, value, st, word in cache_cases(True):
        args = list(good)
        args[4 + at] = value
        if at == 11 and value > 5:
            args[4 + 10] = value
        refused(lib, "dsl_kv8_shared_attention", args, st, word)
    refuse_each(lib, "dsl_kv8_shared_attention", good, [
        (3, 5, -1, "q_heads"), (0, P + 4, -1, "q must"), (19, None, -1, "group_starts"), (20, P + 2, -1, "shared_lens"),
        (21, -1, -1, "groups"), (21, 65536, -2, "groups"), (22, -1, -1, "max_group"), (25, 64, -1, "strides of out"),
        (26, (1 << 20) + 1, -2, "at most 2^22"), (28, float("nan"), -1, "scale"), (30, 7, -1, "x_dtype"),
        (31, None, -3, "workspace"), (32, 16, -3, "workspace"), (31, P + 8, -3, "workspace")])
    for at in (18, 26):                          # no sequences, no rows
        args = list(good)
        args[18] = args[26] = 0
        assert lib.dsl_kv8_shared_attention(*args) == 0
    assert lib.dsl_kv8_shared_attention_workspace_bytes(2, 64, 128, 5, 3, 0, 4, 1, 1, 3) == 0
    assert lib.dsl_kv8_shared_attention_workspace_bytes(2, 64, 128, 5, 3, 7, 4, 4, -1, 3) == 0
    assert lib.dsl_kv8_shared_attention_workspace_bytes(2, 64, 128, 5, 3, 7, 4, 4, 2, 2) > 0


FORK = [P, P, P, P, 10, 2, 64, 128, P, 5, 5, P, 3, P, P, 0, 4, P, P, Q, Q, P, P, 1 << 20, None]


def test_fork(lib):
    refuse_each(lib, "dsl_kv8_fork", FORK, [
        (0, P + 8, -1, "k_cache"), (1, None, -1, "v_cache"), (2, None, -1, "scales"), (4, -1, -1, "pages"), (5, 0, -1, "heads"),
        (6, 48, -2, "page size"), (7, 96, -2, "head dim"), (8, None, -1, "page table"), (9, 4, -1, "table_ld"),
        (10, 1 << 30, -1, "table"), (11, None, -1, "seq_lens"), (12, 70000, -2, "sequences"), (13, P + 1, -1, "parents"),
        (14, P + 2, -1, "new tokens"), (15, -1, -1, "new tokens"), (15, 1 << 31, -1, "new tokens"), (16, -1, -1, "children"),
        (16, 65536, -2, "children"), (17, None, -1, "refs"), (18, None, -1, "out_lens"), (19, None, -1, "out_table"),
        (20, P + 2, -1, "out_refs"), (21, None, -1, "lacking"), (19, P, -1, "old ones"), (20, P, -1, "old ones"),
        (22, None, -3, "workspace"), (23, 8, -3, "workspace")])
    assert lib.dsl_kv8_fork_workspace_bytes(-1, 5, 4, 10) == 0
    assert lib.dsl_kv8_fork_workspace_bytes(3, 5, 4, 10) > 0


def test_fork_in_place(lib):
    args = list(FORK)
    refused(lib, "dsl_kv8_fork", args, -1, "new lengths")      # seq_lens are out_lens


def test_compact(lib):
    good = [P, P, P, P, 10, 2, 64, 128, P, 5, 5, 3, P, Q, Q, P, P, P, 1 << 20, None]
    refuse_each(lib, "dsl_kv8_compact", good, [
        (0, None, -1, "k_cache"), (6, 20, -2, "page size"), (9, 4, -1, "table_ld"), (12, None, -1, "refs"),
        (13, None, -1, "out_table"), (14, P, -1, "old ones"), (15, None, -1, "moved"), (16, None, -1, "live"),
        (17, None, -3, "workspace"), (18, 4, -3, "workspace")])
    args = list(good)
    args[9], args[13] = 6, P
    refused(lib, "dsl_kv8_compact", args, -1, "table in place")


def test_rotary(lib):
    good = [P, 512, 128, 4, P, 256, 128, 2, 7, 128, 64, P, 0, 7, 1, None, P, 1.0, 0, 0, Q, 512, 128, Q, 256, 128, None]
    refuse_each(lib, "dsl_rotary", good, [
        (0, None, -1, "q or its result"), (20, P + 1, -1, "q or its result"), (4, None, -1, "k or its result"),
        (2, 64, -1, "strides of q"), (25, 64, -1, "strides of k"), (3, 0, -1, "q_heads"), (8, -1, -1, "rows"),
        (8, 1 << 24, -2, "rows"), (9, 2048, -2, "dim"), (10, 65, -1, "pairs"), (10, -1, -1, "pairs"), (11, None, -1, "positions"),
        (11, P + 2, -1, "positions"), (13, 6, -1, "positions"), (14, 0, -1, "axes"),
        (14, 2, -1, "axis_of"), (15, P + 1, -1, "axis_of"), (16, P + 4, -1, "freqs"), (17, float("inf"), -1, "magnitude"),
        (19, 1, -1, "x_dtype")])
    args = list(good)
    args[20], args[21] = P, 640
    refused(lib, "dsl_rotary", args, -1, "in place")
    args = list(good)
    args[8] = args[13] = 0
    assert lib.dsl_rotary(*args) == 0


def test_logprobs(lib):
    good = [P, 7, 1000, 1000, 0, P, 2, 2, 1.0, 5, P, P, P, P, P, 1 << 30, None]
    refuse_each(lib, "dsl_token_logprobs", good, [
        (0, None, -1, "logits"), (0, P + 1, -1, "logits"), (1, -1, -1, "rows"), (1, 1 << 22, -2, "rows"), (2, 0, -1, "vocab"),
        (3, 999, -1, "ld"), (4, 9, -1, "x_dtype"), (5, None, -1, "ids"), (6, 1, -1, "ids"), (7, -1, -1, "ids"),
        (8, 0.0, -1, "scale"), (8, float("inf"), -1, "scale"), (8, float("nan"), -1, "scale"), (9, -1, -1, "top"),
        (9, 33, -2, "top"), (10, None, -1, "logp"), (11, P + 2, -1, "entropy"), (12, None, -1, "top_logp"),
        (13, None, -1, "top_ids")])
    args = list(good)
    args[2], args[9] = 4, 5
    refused(lib, "dsl_token_logprobs", args, -1, "top")
    args = list(good)
    args[1], args[2], args[3], args[15] = 1, 200000, 200000, 16       # split over workgroups
    refused(lib, "dsl_token_logprobs", args, -3, "workspace")
    args = list(good)
    args[1] = 0
    assert lib.dsl_token_logprobs(*args) == 0
    assert lib.dsl_token_logprobs_workspace_bytes(1, 200000, 40, 0) == 0


def test_python_refusals():
    c = KV.new_kv8_cache(4, 2, 128, device="cpu")
    lens, table, refs = (torch.zeros(s, dtype=torch.int32) for s in ((3,), (3, 1), (4,)))
    q = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    for new in (-1, 1.5, True, 1 << 31, None):
        with pytest.raises(ValueError, match="new"):
            KV.kv8_fork(c, lens, table, lens, refs, new=new)
    with pytest.raises(ValueError, match="GPU"):
        KV.kv8_fork(c, lens, table, lens, refs)
    with pytest.raises(ValueError, match="GPU"):
        KV.kv8_compact(c, table, refs)
    with pytest.raises(ValueError, match="page_table"):
        KV.kv8_compact(c, refs, refs)
    with pytest.raises(ValueError, match="GPU"):
        A.kv8_shared_attention(q, c, lens, table, torch.tensor([0, 3]), torch.tensor([16]))
    with pytest.raises(ValueError, match="GPU"):
        R.rotary(q, q, lens, R.rotary_freqs(128, device="cpu"))
    with pytest.raises(ValueError, match="q must be"):
        R.rotary(q[0], None, lens, R.rotary_freqs(128, device="cpu"))
    for bad in (3, -2, 2.0):
        with pytest.raises(ValueError, match="rotary_dim"):
            R.rotary_freqs(bad, device="cpu")
    for bad in ([], [1, -1], [1.5]):
        with pytest.raises(ValueError, match="sections"):
            R.rotary_axes(bad, device="cpu")
    x = torch.zeros((3, 10))
    with pytest.raises(ValueError, match="GPU"):
        LP.token_logprobs(x, lens)
    with pytest.raises(ValueError, match="rows, vocab"):
        LP.token_logprobs(x[0], lens)

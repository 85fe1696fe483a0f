"""CPU: what the 8-bit attention layer's entry points refuse, at the C ABI and
in Python; nothing here reaches a GPU."""
import os

import pytest
import torch

from dsl_tool_amd import _native as N
from dsl_tool_amd import attention as A
from dsl_tool_amd import fused as FU
from dsl_tool_amd import kvcache as KV
from dsl_tool_amd import quant as Q

P = 1 << 20           # an aligned pointer that is never read


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} is not built; run `python -m dsl_tool_amd.build`")
    return N.lib()


def refused(lib, fn, args, status, word):
    assert getattr(lib, fn)(*args) == status, fn
    assert word in lib.dsl_last_error().decode(), lib.dsl_last_error()


def test_row_quantizers(lib):
    for args, st, word in [((P, 4, 12, 16, 0, P, P, None), -1, "multiple of 8"),
                           ((P, 4, 16, 8, 0, P, P, None), -1, "ldx"),
                           ((P, 4, 16, 20, 0, P, P, None), -1, "ldx"),
                           ((P, 4, 40000, 40000, 0, P, P, None), -2, "32768"),
                           ((P, 4, 16, 16, 9, P, P, None), -1, "x_dtype"),
                           ((P + 2, 4, 16, 16, 0, P, P, None), -1, "aligned"),
                           ((P, 4, 16, 16, 0, None, P, None), -1, "q is NULL"),
                           ((P, 4, 16, 16, 0, P, None, None), -1, "scales"),
                           ((P, -1, 16, 16, 0, P, P, None), -1, "rows")]:
        refused(lib, "dsl_quant_int8_rows", args, st, word)
    assert lib.dsl_quant_int8_rows(None, 0, 16, 16, 0, None, None, None) == 0
    good = [P, 4, 16, 16, P, 16, P, 0, 1e-6, 0, 0, P, P, P, None]
    for at, value, st, word in [(9, 1, -1, "x_dtype"), (10, 5, -1, "qfmt"), (7, 3, -1, "weight dtype"),
                                (8, -1.0, -1, "eps"), (8, float("nan"), -1, "eps"), (5, 8, -1, "ldr"),
                                (4, P + 8, -1, "residual"), (6, None, -1, "weight"), (11, P + 2, -1, "h must"),
                                (2, 20, -1, "multiple of 8")]:
        args = list(good)
        args[at] = value
        refused(lib, "dsl_add_rmsnorm_quant", args, st, word)


# k, v, scales, pages, heads, page, dim, fmt, table, ld, width, lens, starts, seqs
CACHE = [P, P, P, P, 10, 2, 64, 128, 0, P, 5, 5, P, P, 3]


def cache_cases(rows_at):
    return [(7, 96, -2, "head dim"), (6, 48, -2, "page size"), (6, 8, -2, "page size"), (8, 2, -1, "fmt"),
            (10, 4, -1, "table_ld"), (0, P + 8, -1, "k_cache"), (1, None, -1, "v_cache"), (2, None, -1, "scales"),
            (12, None, -1, "seq_lens"), (9, None, -1, "page table"), (5, 0, -1, "heads"), (14, 70000, -2, "sequences"),
            (11, 1 << 30, -1, "table")] + ([(13, None, -1, "starts")] if rows_at else [])


def test_cache_entry_points(lib):
    write = CACHE + [P, 256, 128, P, 256, 128, 7, 4, 0, None]
    read = CACHE + [P, P, 7, 0, None]
    attn = [P, 512, 128, 4] + CACHE + [P, 512, 128, 7, 4, 0.1, 1, 0, P, 1 << 30, None]
    for fn, good, off in (("dsl_kv8_write", write, 0), ("dsl_kv8_read", read, 0), ("dsl_kv8_attention", attn, 4)):
        for at, value, st, word in cache_cases(True):
            args = list(good)
            args[off + at] = value
            if at == 11 and value > 5:
                args[off + 10] = value
            refused(lib, fn, args, st, word)
    for at, value, word in [(15, P + 2, "k must"), (16, 12, "strides of k"), (17, 64, "strides of k"), (20, 130, "strides of v"),
                            (22, -1, "max_q"), (23, 1, "x_dtype")]:
        args = list(write)
        args[at] = value
        refused(lib, "dsl_kv8_write", args, -1, word)
    for at, value, st, word in [(3, 5, -1, "q_heads"), (0, P + 4, -1, "q must"), (1, 10, -1, "strides of q"),
                                (21, 64, -1, "strides of out"), (24, float("inf"), -1, "scale"), (26, 7, -1, "x_dtype")]:
        args = list(attn)
        args[at] = value
        refused(lib, "dsl_kv8_attention", args, st, word)
    for at, value, st, word in [(27, None, -3, "workspace"), (28, 16, -3, "workspace")]:
        args = list(attn)
        args[14] = args[15] = 64                 # contexts long enough to be split
        args[at] = value
        refused(lib, "dsl_kv8_attention", args, st, word)
    # nothing to do is no error
    for fn, good, at in (("dsl_kv8_write", write, 21), ("dsl_kv8_read", read, 17), ("dsl_kv8_attention", attn, 22)):
        args = list(good)
        args[at] = 0
        assert getattr(lib, fn)(*args) == 0
    assert lib.dsl_kv8_attention_workspace_bytes(2, 64, 128, 5, 3, 0, 4, 1) == 0


def test_python_refusals():
    x = torch.zeros((4, 64), dtype=torch.bfloat16)
    w = torch.ones(64)
    with pytest.raises(ValueError, match="fmt"):
        FU.add_rmsnorm_quant(x, x, w, fmt="mxfp4")
    with pytest.raises(ValueError, match="GPU"):
        FU.add_rmsnorm_quant(x, x, w)
    with pytest.raises(ValueError, match="GPU"):
        Q.quant_int8_rows(x)
    with pytest.raises(ValueError, match="page"):
        KV.new_kv8_cache(4, 2, 128, page=48, device="cpu")
    with pytest.raises(ValueError, match="fmt"):
        KV.new_kv8_cache(4, 2, 128, fmt="int4", device="cpu")
    c = KV.new_kv8_cache(4, 2, 128, device="cpu")
    assert c.page == 64 and c.k.shape == (4, 2, 64, 128) and c.v.shape == (4, 2, 128, 64)
    lens, table = torch.zeros(3, dtype=torch.int32), torch.zeros((3, 1), dtype=torch.int32)
    k = torch.zeros((3, 2, 128), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="GPU"):
        KV.kv8_write(c, k, k, lens, table)
    with pytest.raises(ValueError, match="GPU"):
        A.kv8_attention(k, c, lens, table)
    with pytest.raises(TypeError, match="dtype"):
        KV.kv8_read(c, lens, table, lens, 3, dtype=torch.float32)
    with pytest.raises(ValueError, match="total"):
        KV.kv8_read(c, lens, table, lens, -1)


def test_attention_counts_rows_in_ints(lib):
    attn = [P, 512, 128, 4] + CACHE + [P, 512, 128, 7, 4, 0.1, 1, 0, P, 1 << 30, None]
    attn[22] = (1 << 28) + 1
    refused(lib, "dsl_kv8_attention", attn, -1, "query heads")

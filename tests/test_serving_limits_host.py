"""CPU: the attention's workspace query at sizes that the call refuses."""
import os

import pytest

from dsl_tool_amd import _native as N


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} is not built; run `python -m dsl_tool_amd.build`")
    return N.lib()


# heads, page, dim, width, seqs, rows, q_heads, max_q
GOOD = [2, 64, 128, 64, 3, 7, 4, 4]


@pytest.mark.parametrize("change,word", [
    ({0: 1 << 32, 6: 1 << 32}, "heads"), ({0: 0}, "heads"), ({4: 1 << 32, 5: 64, 7: 64}, "sequences"),
    ({4: 1 << 32, 5: 10 ** 6, 6: 1 << 20, 7: 10 ** 6}, "sequences"), ({5: 1 << 31}, "rows"), ({5: 1 << 29}, "2^30"),
    ({1: 48}, "page size"), ({2: 1 << 32}, "head dim"), ({3: 1 << 40}, "2^31"), ({6: 5}, "multiple"), ({7: -1}, "max_q"),
    ({5: -1}, "rows")])
def test_workspace_query_refuses_what_the_call_refuses(lib, change, word):
    assert lib.dsl_kv8_attention_workspace_bytes(*GOOD) > 0
    args = list(GOOD)
    for at, value in change.items():
        args[at] = value
    assert lib.dsl_kv8_attention_workspace_bytes(*args) == 0
    assert word in lib.dsl_last_error().decode()


def test_nothing_to_do_needs_no_workspace(lib):
    for at in (4, 5):
        args = list(GOOD)
        args[at] = 0
        assert lib.dsl_kv8_attention_workspace_bytes(*args) == 0

"""CPU: further refusals of several continuations' entry points; nothing here reaches a GPU."""
import os

import pytest
import torch

from dsl_tool_amd import _native as N
from dsl_tool_amd import layer8 as L
from tests.test_generate_host import refuse_each
from tests.test_serving_host import CACHE, P, refused


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} is not built; run `python -m dsl_tool_amd.build`")
    return N.lib()


def test_logprobs_scale(lib):
    good = [P, 7, 1000, 1000, 0, P, 2, 2, 1.0, 5, P, P, P, P, P, 1 << 30, None]
    refuse_each(lib, "dsl_token_logprobs", good, [(8, 2.0 ** 126, -1, "scale"), (8, 3e38, -1, "scale"), (8, -1.0, -1, "scale"),
                                                  (8, 1e-60, -1, "scale")])


def test_layer_axes_without_freqs():
    """What says how freqs turn the heads does not go by without a word where there are none."""
    w = torch.zeros(512, 128), torch.zeros(128, 256), torch.ones(128)
    for kw in ({"adjacent": True}, {"axis_of": torch.zeros(32, dtype=torch.int32)},
               {"adjacent": True, "rotate": lambda q, k: (q, k)}):
        with pytest.raises(ValueError, match="freqs"):
            L.Int8AttentionLayer(*w, q_heads=4, kv_heads=2, dim=64, **kw)


def test_shared_attention_of_many_rows(lib):
    """More rows than prefixes are read once for: refused by their number where they are, and
    not where each sequence is computed by itself."""
    rows = (1 << 20) + 1
    args = [P, 512, 128, 4] + CACHE + [P, P, 2, 2, P, 512, 128, rows, 48, 0.1, 1, 0, None, 0, None]
    refused(lib, "dsl_kv8_shared_attention", args, -2, "at most 2^22")
    args[27] = 500                               # max_q: 1000 rows to a cache head
    refused(lib, "dsl_kv8_shared_attention", args, -3, "workspace")
    sizes = [2, 64, 128, 5, 3, rows, 4]
    assert lib.dsl_kv8_shared_attention_workspace_bytes(*sizes, 48, 2, 2) == 0
    assert lib.dsl_kv8_shared_attention_workspace_bytes(*sizes, 49, 2, 2) > 0

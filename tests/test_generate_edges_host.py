"""CPU: further refusals of several continuations' entry points; nothing here reaches a GPU."""
import os

import pytest

from dsl_tool_amd import _native as N
from tests.test_generate_host import refuse_each
from tests.test_serving_host import P


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} is not built; run `python -m dsl_tool_amd.build`")
    return N.lib()


def test_logprobs_scale(lib):
    good = [P, 7, 1000, 1000, 0, P, 2, 2, 1.0, 5, P, P, P, P, P, 1 << 30, None]
    refuse_each(lib, "dsl_token_logprobs", good, [(8, 2.0 ** 126, -1, "scale"), (8, 3e38, -1, "scale"), (8, -1.0, -1, "scale"),
                                                  (8, 1e-60, -1, "scale")])

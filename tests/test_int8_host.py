"""CPU: what the int8 GEMM refuses at the C ABI, and which kernel a shape takes."""
import os

import pytest

from dsl_tool_amd import _native as N
from tests import test_routes as R

P = 1 << 20           # an aligned pointer that is never read


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(N.LIB_PATH):
        pytest.fail(f"{N.LIB_PATH} is not built; run `python -m dsl_tool_amd.build`")
    return N.lib()


def test_refusals(lib):
    good = [P, P, P, 4, 32, 64, 32, 0, P, P, None]
    for at, value, st, word in [(5, 24, -1, "multiple of 16"), (5, 1 << 17, -2, "131072"), (6, 31, -1, "ldc"),
                                (7, 9, -1, "out_dtype"), (0, P + 8, -1, "a must"), (1, None, -1, "b is NULL"),
                                (2, P + 1, -1, "c is"), (2, None, -1, "c is"), (8, P + 2, -1, "scales"),
                                (9, None, -1, "scales"), (3, -1, -1, "m >= 0")]:
        args = list(good)
        args[at] = value
        assert lib.dsl_int8_gemm(*args) == st, args
        assert word in lib.dsl_last_error().decode(), lib.dsl_last_error()
    for at in (3, 4):
        args = [None, None, None, 4, 32, 64, 32, 0, None, None, None]
        args[at] = 0
        assert lib.dsl_int8_gemm(*args) == 0


@pytest.mark.parametrize("m,n,k,want", [
    (1, 8, 16, "stream tail 16x16"), (16, 7168, 4096, "stream 16x32"), (300, 777, 656, "stream tail 64x16"),
    (3000, 24, 80, "stream tail 32x16"), (1500, 1300, 144, "pipe 128x128"), (700, 1000, 64, "pipe 64x128 deep"),
    (1024, 4096, 4096, "pipe 128x128 deep"), (2100, 2056, 272, "persist 256x128"), (4001, 7168, 4096, "persist 256x256"),
    (4300, 4300, 144, "persist 256x256 + pipe 128x128")])
def test_routes(monkeypatch, m, n, k, want):
    monkeypatch.setitem(R.MODES, "int8", 6)
    assert R.route("int8", m, n, k) == want

"""int8 GEMM with a scale per token and per output channel: the sums are exact
integers, so the result is off by the fp32 conversion, two products and the
output type's rounding only."""
import pytest
import torch

from dsl_tool_amd import gemm as G
from dsl_tool_amd import quant as Q

pytestmark = pytest.mark.gpu
DEV = "cuda"
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}
FP32 = 4 * 2.0 ** -24            # sum to fp32, two products (the last one is a float32 result's own rounding)

# m, n, k: every kernel that the router picks, at sizes that are no whole tiles
SIZES = [(1, 8, 16), (1, 1, 16), (3, 7, 48), (16, 130, 256), (16, 2056, 4096), (17, 130, 272), (33, 1001, 512),
         (64, 4096, 1024), (100, 129, 1040), (300, 777, 656), (257, 264, 2048), (1100, 40, 512), (3000, 24, 80),
         (1500, 1300, 144), (1500, 1300, 64), (700, 1000, 64), (500, 2048, 2048), (700, 1301, 1664),
         (1024, 2049, 1536), (2100, 2056, 272), (2048, 2055, 400), (4352, 3840, 256), (4100, 4001, 272),
         (4300, 4300, 144)]


def codes(shape, seed, most=127):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-most - 1, most + 1, shape, generator=g, dtype=torch.int8)


def scales(n, seed):
    return torch.rand(n, generator=torch.Generator().manual_seed(seed)) * 0.05 + 0.001


def within(c, qa, qw, sa, sw):
    ref = (qa.double() @ qw.double().t()) * sa.double()[:, None] * sw.double()
    assert c.shape == ref.shape
    err = (c.cpu().double() - ref).abs()
    tol = ref.abs() * (HALF[c.dtype] + FP32)
    assert (err <= tol).all(), (err / tol.clamp_min(1e-30)).max()


@pytest.mark.parametrize("out", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_int8_gemm(m, n, k, out):
    qa, qw, sa, sw = codes((m, k), 1), codes((n, k), 2), scales(m, 3), scales(n, 4)
    c = G.int8_gemm_packed(qa.to(DEV), qw.to(DEV), sa.to(DEV), sw.to(DEV), out_dtype=out)
    assert c.dtype == out
    within(c, qa, qw, sa, sw)


@pytest.mark.parametrize("m,n", [(1, 64), (40, 64), (130, 2000), (2048, 2055)])
def test_sums_past_24_bits(m, n):
    """Codes that all agree: sums of 2^14 k, which fp32 accumulation would round."""
    k = 16384 + 16
    qa = torch.full((m, k), -128, dtype=torch.int8)
    qa[:, ::7] = 127
    qw = codes((n, k), 5, 3)
    qw[: n // 2] = -128
    sa, sw = torch.ones(m), torch.ones(n)
    c = G.int8_gemm_packed(qa.to(DEV), qw.to(DEV), sa.to(DEV), sw.to(DEV), out_dtype=torch.float32)
    within(c, qa, qw, sa, sw)


@pytest.mark.parametrize("m,n,k", [(5, 300, 512), (200, 257, 272), (1500, 1300, 144), (2100, 2056, 272), (4352, 3840, 256)])
def test_out_views_streams_and_repeats(m, n, k):
    """A result inside a wider tensor whose other elements stay, unaligned
    operands, a stream of its own; the same bytes every time."""
    qa, qw, sa, sw = codes((m, k), 6), codes((n, k), 7), scales(m, 8), scales(n, 9)
    a, w, s, t = (x.to(DEV) for x in (qa, qw, sa, sw))
    want = G.int8_gemm_packed(a, w, s, t)
    wide = torch.zeros((m, n + 5), dtype=torch.bfloat16, device=DEV)
    odd = torch.empty(m * k + 1, dtype=torch.int8, device=DEV)[1:].view(m, k).copy_(a)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c = G.int8_gemm_packed(a, w, s, t, out=wide[:, 3:n + 3])
        d = G.int8_gemm_packed(odd, w, s, t)
    side.synchronize()
    assert c.data_ptr() == wide[:, 3:].data_ptr()
    assert torch.equal(c, want) and torch.equal(d, want)
    assert (wide[:, :3] == 0).all() and (wide[:, n + 3:] == 0).all()
    for _ in range(3):
        assert torch.equal(G.int8_gemm_packed(a, w, s, t), want)


def test_quantized_product():
    """Rows quantized by the library: within the codes' half steps of the product
    of the unquantized rows."""
    g = torch.Generator().manual_seed(10)
    x, w = torch.randn((37, 1024), generator=g).bfloat16(), (torch.randn((200, 1024), generator=g) * 0.03).bfloat16()
    (qx, sx), (qw, sw) = Q.quant_int8_rows(x.to(DEV)), Q.quant_int8_rows(w.to(DEV))
    c = G.int8_gemm_packed(qx, qw, sx, sw, out_dtype=torch.float32).cpu().double()
    x, w, sx, sw = x.double(), w.double(), sx.cpu().double(), sw.cpu().double()
    tol = (x.abs().sum(1)[:, None] * sw / 2 + w.abs().sum(1) * sx[:, None] / 2 + 1024 * sx[:, None] * sw / 4) * (1 + 2.0 ** -20)
    assert ((c - x @ w.t()).abs() <= tol).all()


def test_empty_and_refused():
    e = torch.zeros((0, 64), dtype=torch.int8, device=DEV)
    w = torch.zeros((5, 64), dtype=torch.int8, device=DEV)
    s0, s5 = torch.ones(0, device=DEV), torch.ones(5, device=DEV)
    assert G.int8_gemm_packed(e, w, s0, s5).shape == (0, 5)
    assert G.int8_gemm_packed(w, e, s5, s0).shape == (5, 0)
    with pytest.raises(TypeError, match="int8"):
        G.int8_gemm_packed(w.view(torch.uint8), w, s5, s5)
    with pytest.raises(ValueError, match="K mismatch"):
        G.int8_gemm_packed(w, w[:, :32].contiguous(), s5, s5)
    with pytest.raises(ValueError, match="scales"):
        G.int8_gemm_packed(w, w, s5[:4], s5)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        G.int8_gemm_packed(w[:, :24].contiguous(), w[:, :24].contiguous(), s5, s5)

"""The int8 Linear (ress_int8_linear) and the row quantiser against their
formula: codes by the same fp32 steps (exact), sums in 64 bits.  The scales
and the bias take four fp32 roundings: 2^-22 of |product| + |bias|; the GELU a
few more (2^-20 of |y|, and as much of an absolute 1 in erf's tail times |y|);
a bf16 output 2^-8 of the value."""

import pytest
import torch

from ress_b200 import kernels as K
from ress_b200._lib import RessError

from streaming_ref import quant_rows

pytestmark = pytest.mark.gpu


def _inputs(m, k, n, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(m, k, device="cuda", generator=g) * (0.2 + torch.rand(k, device="cuda", generator=g) * 3)
    w = torch.randn(n, k, device="cuda", generator=g) * 0.05
    bias = torch.randn(n, device="cuda", generator=g)
    return x.to(dtype), w, bias


def _check(out, x8, sx, w8, sw, bias, act):
    prod = (x8 @ w8.double().t()) * sx.double()[:, None] * sw.double()
    y = prod + bias.double() if bias is not None else prod
    tol = 2.0 ** -22 * (prod.abs() + (bias.double().abs() if bias is not None else 0))
    if act:
        y = 0.5 * y * (1 + torch.erf(y / 2 ** 0.5))
        tol = 2 * tol + 2.0 ** -20 * y.abs() + 2.0 ** -22 * prod.abs()
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * y.abs()
    err = (out.double() - y).abs()
    assert bool((err <= tol + 1e-30).all()), float((err - tol).max())


SHAPES = [(1, 16, 1), (1, 64, 8), (1, 1024, 512), (3, 80, 33), (16, 128, 72), (17, 256, 100), (37, 1536, 250),
          (64, 64, 64), (65, 208, 129), (128, 1024, 256), (129, 1040, 257), (300, 512, 1000), (700, 4096, 136),
          (1374, 1024, 320)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", SHAPES)
def test_linear(m, k, n, dtype):
    x, w, bias = _inputs(m, k, n, dtype, seed=m + k + n)
    w8, sw = K.int8_quant_rows(w)
    x8, sx = quant_rows(x)
    for b, act, od in ((bias, None, None), (None, "gelu", torch.float32), (bias, "gelu", torch.bfloat16)):
        out = K.int8_linear(x, w8, sw, b, act=act, out_dtype=od)
        again = K.int8_linear(x, w8, sw, b, act=act, out_dtype=od)
        torch.cuda.synchronize()
        assert K.check_status() == 0
        assert out.shape == (m, n) and out.dtype == (od or dtype)
        _check(out, x8, sx, w8, sw, b, act)
        assert torch.equal(out, again)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n", [(20, 400, 2048), (20, 528, 2049), (256, 2064, 1000), (257, 1024, 1001), (128, 144, 4000),
                                   (30, 4112, 64), (4, 8192, 40), (5, 6560, 24)])
def test_linear_few_tiles(m, k, n, dtype):
    """Tiles few enough for their K to be shared by several CTAs, at the sizes
    where their number changes; rows and channels past the tiles' last."""
    x, w, bias = _inputs(m, k, n, dtype, seed=m + k + n)
    x[m // 2] = 0
    w8, sw = K.int8_quant_rows(w)
    x8, sx = quant_rows(x)
    for act in (None, "gelu"):
        out = K.int8_linear(x, w8, sw, bias, act=act)
        torch.cuda.synchronize()
        assert K.check_status() == 0
        _check(out, x8, sx, w8, sw, bias, act)
        # the same bits on the paths of a single token and of the others
        assert torch.equal(K.int8_linear(x[1:2], w8, sw, bias, act=act), out[1:2])
        assert torch.equal(K.int8_linear(x[2:], w8, sw, bias, act=act), out[2:])


@pytest.mark.parametrize("m,k,n", [(12001, 1008, 1024), (9999, 1024, 1000), (8200, 2064, 1024), (5000, 4096, 1016)])
def test_linear_over_several_waves(m, k, n):
    """Tiles for several waves of the GPU; rows of a
    wider tensor, a zero row and one that is not finite among them."""
    x, w, bias = _inputs(m, k + 16, n, torch.bfloat16, seed=m)
    x, w = x[:, 8:k + 8], w[:, :k].contiguous()
    x[m // 2] = 0
    x[m - 1, 3] = torch.inf
    w8, sw = K.int8_quant_rows(w)
    out = K.int8_linear(x, w8, sw, bias, act="gelu")
    torch.cuda.synchronize()
    assert K.check_status() == 0
    x8, sx = quant_rows(x)
    _check(out[:-1], x8[:-1], sx[:-1], w8, sw, bias, "gelu")
    assert bool(out[-1].isnan().all())
    for _ in range(3):
        assert torch.equal(K.int8_linear(x, w8, sw, bias, act="gelu")[:-1], out[:-1])
    # the same bits as among few tokens
    assert torch.equal(K.int8_linear(x[77:177], w8, sw, bias, act="gelu"), out[77:177])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k", [(1, 16), (7, 80), (1000, 1040), (33, 4096)])
def test_quant_rows(m, k, dtype):
    x, _, _ = _inputs(m, k, 1, dtype, seed=m + k)
    x[0] = 0
    if m > 5:
        x[3] *= 1e-30
        x[4] *= 1e30
    x8, s = K.int8_quant_rows(x)
    r8, rs = quant_rows(x)
    assert torch.equal(s, rs) and torch.equal(x8.double(), r8)


def test_extremes():
    """Codes of +-127 throughout at a long K (sums beyond 2^24), zero rows, rows that are not finite."""
    m, k, n = 130, 8192, 64
    x = torch.ones(m, k, device="cuda")
    x[1] = -1
    x[2] = 0
    x[3, 5] = torch.nan
    x[4, 6] = torch.inf
    w8 = torch.full((n, k), 127, dtype=torch.int8, device="cuda")
    w8[1] = -127
    sw = torch.full((n,), 1 / 127, device="cuda")
    for rows in (slice(0, 8), slice(0, m)):
        out = K.int8_linear(x[rows], w8, sw)
        x8, sx = quant_rows(x[rows])
        fine = [i for i in range(out.shape[0]) if i not in (3, 4)]
        _check(out[fine], x8[fine], sx[fine], w8, sw, None, None)
        assert not out[2].any() and bool(out[3:5].isnan().all())
    K.check_status()


def test_strided_rows_and_batches():
    x, w, bias = _inputs(150, 3 * 256, 96, torch.bfloat16, seed=1)
    w8, sw = K.int8_quant_rows(w[:, :256].contiguous())
    part = x[:, 256:512]  # rows 768 apart
    for rows in (part, part[:9], part[:1]):
        assert torch.equal(K.int8_linear(rows, w8, sw, bias), K.int8_linear(rows.contiguous(), w8, sw, bias))
    y = K.int8_linear(part.reshape(3, 50, 256), w8, sw, bias)
    assert y.shape == (3, 50, 96) and torch.equal(y.view(150, 96), K.int8_linear(part, w8, sw, bias))
    assert K.int8_linear(part[:0], w8, sw).shape == (0, 96)


def test_rows_do_not_depend_on_their_company():
    """A token's output is the same bits alone, among a few and among many."""
    x, w, bias = _inputs(400, 1024, 200, torch.bfloat16, seed=2)
    w8, sw = K.int8_quant_rows(w)
    many = K.int8_linear(x, w8, sw, bias, act="gelu")
    for rows in (slice(5, 6), slice(0, 16), slice(30, 90)):
        assert torch.equal(K.int8_linear(x[rows], w8, sw, bias, act="gelu"), many[rows])


def test_refusals():
    x, w, bias = _inputs(4, 64, 8, torch.bfloat16, seed=3)
    w8, sw = K.int8_quant_rows(w)
    for args, kw in [((x.half(), w8, sw), {}), ((x.cpu(), w8, sw), {}), ((x, w8.float(), sw), {}),
                     ((x, w8.t(), sw), {}), ((x[:, :48], w8, sw), {}), ((x, w8, sw.double()), {}),
                     ((x, w8, sw[:4]), {}), ((x, w8, sw, bias.bfloat16()), {}), ((x, w8, sw, bias.cpu()), {}),
                     ((x, w8, sw), dict(act="relu")), ((x, w8, sw), dict(out_dtype=torch.float16)),
                     ((x[:, :24], w8[:, :24].contiguous(), sw), {})]:  # K not a multiple of 16
        with pytest.raises(RessError):
            K.int8_linear(*args, **kw)
    with pytest.raises(RessError):
        K.int8_quant_rows(x[:, :24])


def test_rows_that_no_copy_engine_takes():
    """Rows off a 16-byte boundary, at an odd distance, or all the same one (expanded)."""
    x, w, bias = _inputs(130, 270, 96, torch.bfloat16, seed=4)
    w8, sw = K.int8_quant_rows(w[:, :256].contiguous())
    flat = x.reshape(-1)
    for rows in (x[:, 3:259], x[:, 8:264], flat[1:1 + 100 * 256].view(100, 256), x[:1, :256].expand(70, 256),
                 x[None, :1, :256].expand(3, 50, 256), x.t()[:256].t(), x.float()[:, 1:257], x.float()[:5, 1:257]):
        plain = rows.clone(memory_format=torch.contiguous_format)
        assert torch.equal(K.int8_linear(rows, w8, sw, bias), K.int8_linear(plain, w8, sw, bias))
        for a, b in zip(K.int8_quant_rows(rows), K.int8_quant_rows(plain)):
            assert a.shape == b.shape and torch.equal(a, b)


# The tile that each size takes, without and with GELU (a pair's 256 x 256, one
# CTA's 128 x 128 or 128 x 64), and the passes of its busiest CTA.  Odd widths
# are stored by plain instructions, the others by TMA.
TILES = [
    (1374, 4096, 1024, "128: one pass of 32 slices"),
    (300, 1024, 4096, "128: one pass"),
    (257, 1024, 4097, "128: one pass, plain stores"),
    (3000, 256, 1500, "128: two passes of 2 slices; 64 with GELU: four"),
    (3000, 256, 1501, "the same, plain stores"),
    (2200, 2064, 1022, "pair: one pass of 17 slices, plain bf16 stores; 128 with GELU"),
    (700, 1024, 1024, "64: one pass"),
    (165, 1536, 3001, "64: one pass of 12 slices, plain stores"),
    (2100, 144, 2000, "128: two passes of 2 slices; 64 with GELU: four"),
    (5000, 1040, 1001, "pair: two passes, plain stores"),
    (9999, 1024, 1001, "pair: three passes, plain stores"),
    (12001, 1008, 1024, "pair: three passes"),
]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m,k,n,tile", TILES)
def test_linear_tiles(m, k, n, tile, dtype):
    """Every tile in both output types: remainders of rows, channels and K, one pass and several, both ways of storing."""
    x, w, bias = _inputs(m, k, n, dtype, seed=m + k + n)
    w8, sw = K.int8_quant_rows(w)
    x8, sx = quant_rows(x)
    for b, act in ((bias, None), (None, "gelu")):
        out = K.int8_linear(x, w8, sw, b, act=act)
        torch.cuda.synchronize()
        assert K.check_status() == 0
        _check(out, x8, sx, w8, sw, b, act)
        # the same bits in another tile
        assert torch.equal(K.int8_linear(x[-20:], w8, sw, b, act=act), out[-20:])


def test_a_graph_of_linears():
    """Captured and replayed on new tokens: the quantiser and the product of both, back to back."""
    for m in (1, 64, 1500):
        x, w, bias = _inputs(m, 512, 512, torch.bfloat16, seed=m)
        w8, sw = K.int8_quant_rows(w)
        want = K.int8_linear(K.int8_linear(x, w8, sw, bias, act="gelu"), w8, sw)
        held, graph = torch.zeros_like(x), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = K.int8_linear(K.int8_linear(held, w8, sw, bias, act="gelu"), w8, sw)
        for _ in range(3):
            held.copy_(x)
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)

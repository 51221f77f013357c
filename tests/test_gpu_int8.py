"""Rows in 8 bits (FGMS.nn.quantize_rows, add_norm_int8) and their products (int8_linear), against the plain formulas in 64 bits."""
import pytest
import torch

from tests import block_util as B

pytestmark = pytest.mark.gpu

SHAPES = [(1, 8), (1, 1), (3, 5), (257, 8), (1000, 16), (301, 40), (77, 63), (130, 64), (129, 128), (50, 512), (33, 520), (37, 1096), (19, 2048),
          (9, 4096), (5, 8200), (3, 12001), (4, 16384)]


def features(n, c, dtype, gen, by=1.0):
    return (by * torch.randn(n, c, generator=gen)).to(B.DTYPES[dtype]).cuda()


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rows_in_eight_bits(shape, dtype):
    from FGMS import nn
    gen = torch.Generator().manual_seed(shape[0] + shape[1])
    n, c = shape
    x, residual = features(n, c, dtype, gen), features(n, c, dtype, gen, 3.0)
    q, scales = nn.quantize_rows(x)
    assert q.shape == (n, c) and q.dtype == torch.int8 and scales.dtype == torch.float32 and (n == 1 or q.stride(0) % 16 == 0)
    B.check_eighths(q, scales, B.cpu(x), torch.zeros(n, c, dtype=torch.float64), "rows")
    scale = (1 + 0.2 * torch.randn(c, generator=gen)).to(B.DTYPES[dtype]).cuda()
    for r, w in ((residual, scale), (None, None)):
        q, scales, h = nn.add_norm_int8(x, r, w, 1e-3)
        if r is None:
            assert h is x
        else:
            B.within(h, *B.total(x, r, torch.ones(n, c, dtype=torch.float64)), "sum")
        B.check_eighths(q, scales, *B.normed(h, w, 1e-3, unit=0.0), "norm")
        assert torch.equal(h, nn.add_norm(x, r, w, 1e-3)[1])
    wide = features(n, 2 * c, dtype, gen, 2.0)
    q, scales = nn.quantize_rows(wide, gated=True)
    a, b = B.cpu(wide).chunk(2, 1)
    v = a * torch.sigmoid(a) * b
    # (the exponential's argument is rounded at up to 8 |a| / ln 2 halves of a step, itself and the quotient at a few)
    B.check_eighths(q, scales, v, B.SUM * (2 * a.abs() + 16) * v.abs() + 1e-37, "gated")


def test_halves_go_to_even_numbers():
    from FGMS import nn
    x = torch.tensor([[127.0, 0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 63.5, -126.5, 0.0, -127.0, 3.0, 0.25, -0.75, 100.5, 99.5]], device="cuda")
    q, scales = nn.quantize_rows(x)
    assert scales.tolist() == [1.0]
    assert q.tolist() == [[127, 0, 2, 2, 0, -2, -2, 64, -126, 0, -127, 3, 0, -1, 100, 100]]


def test_quotients_are_those_of_a_division():
    """Of 16-bit values, half of a row's largest and its odd multiples of 1/254 among them, and of 32-bit ones."""
    from FGMS import nn
    for t in B.DTYPES.values():
        gen = torch.Generator().manual_seed(4)
        x = torch.randn(2000, 2072, generator=gen).to(t)
        x[:, :64] = (x.abs().amax(1, keepdim=True).double() * (2 * torch.arange(64) + 1) / 254).to(t)
        x = x.cuda()
        q, scales = nn.quantize_rows(x)
        want = x.cpu().float().abs().amax(1) / 127      # (on the CPU, whose divisions are rounded as they should be)
        assert torch.equal(scales.cpu(), want)
        assert torch.equal(q.cpu(), torch.round(x.cpu().float() / want[:, None]).to(torch.int8))


@pytest.mark.parametrize("channels", [24, 72, 1096, 4100])
def test_rows_without_values(channels):
    """Zeros, numbers too small for a scale, infinities and NaN."""
    from FGMS import nn
    inf = float("inf")
    x = torch.randn(8, channels, device="cuda")
    want = nn.quantize_rows(x)
    x[1], x[3, channels - 1], x[4, 0], x[6, 3] = 0, inf, -inf, float("nan")
    x[5] = 1e-38
    q, scales = nn.quantize_rows(x)
    assert scales[3].isnan() and scales[4].isnan() and scales[6].isnan() and scales[1] == 0 and scales[5] == 0
    assert not q[[1, 3, 4, 5, 6]].any()
    rest = [0, 2, 7]
    assert torch.equal(q[rest], want[0][rest]) and torch.equal(scales[rest], want[1][rest])
    w = torch.ones(3, channels, dtype=torch.int8, device="cuda")
    y = nn.int8_linear(q, scales, w, torch.ones(3, device="cuda"), dtype=torch.float32)
    assert y[[3, 4, 6]].isnan().all() and (y[[1, 5]] == 0).all() and y[rest].isfinite().all()
    big = torch.full((2, channels), 6e4, dtype=torch.float16, device="cuda")
    q, scales, h = nn.add_norm_int8(big, big)
    assert (h == inf).all() and scales.isnan().all()


# rows, outputs, channels
PRODUCTS = [(1, 1, 1), (1, 16, 16), (1, 7, 24), (5, 33, 63), (8, 64, 64), (16, 100, 128), (17, 130, 129), (33, 64, 200), (64, 257, 512), (65, 31, 1096),
            (100, 96, 40), (128, 128, 256), (129, 192, 64), (300, 260, 1000), (1000, 65, 72), (257, 513, 2048), (2, 4096, 300), (16, 300, 8200),
            (1, 1000, 4096), (2100, 520, 136), (700, 2000, 384), (3, 10, 100000)]


def eighths(n, c, gen, behind):
    """int8 rows on 16 bytes with something behind their channels, and scales."""
    padded = (c + 15) // 16 * 16
    held = torch.full((n, padded), behind, dtype=torch.int8)
    held[:, :c] = torch.randint(-128, 128, (n, c), generator=gen).to(torch.int8)
    return held.cuda()[:, :c], (torch.rand(n, generator=gen) + 0.1).cuda() / 127


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("shape", PRODUCTS, ids=str)
def test_products(shape, dtype):
    from FGMS import nn
    n, outputs, c = shape
    gen = torch.Generator().manual_seed(n + outputs + c)
    x, sx = eighths(n, c, gen, 77)
    w, sw = eighths(outputs, c, gen, -99)
    sw = sw / c
    bias = torch.randn(outputs, generator=gen).to(B.DTYPES[dtype]).cuda()
    for b in (None, bias):
        y = nn.int8_linear(x, sx, w, sw, b, B.DTYPES[dtype])
        assert y.dtype == B.DTYPES[dtype]
        B.within(y, *B.product(x, sx, w, sw, b, B.DTYPES[dtype]), "product")
    # rows that do not begin on 16 bytes, or end with their storage
    if n * outputs * c <= 1 << 26:
        bare = [t.contiguous() for t in (x, w)]
        shifted = [torch.cat([t.new_zeros(t.shape[0], 3), t], 1)[:, 3:] for t in (x, w)]
        for u, v in (bare, shifted, [x, bare[1]], [t.t().contiguous().t() for t in (x, w)]):
            assert torch.equal(nn.int8_linear(u, sx, v, sw, bias, B.DTYPES[dtype]), y)


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("shape", [(4200, 4100, 1111), (4097, 4352, 2048), (9000, 1025, 130), (20000, 200, 72), (8300, 64, 40)], ids=str)
def test_wide_products(shape, dtype):
    """The widest tiles, and rows behind their last; sums of whole numbers in 64 bits on the card, where they are exact too."""
    from FGMS import nn
    n, outputs, c = shape
    gen = torch.Generator().manual_seed(n)
    x, sx = eighths(n, c, gen, 55)
    w, sw = eighths(outputs, c, gen, 66)
    bias = torch.randn(outputs, generator=gen).to(B.DTYPES[dtype]).cuda()
    y = nn.int8_linear(x, sx, w, sw / c, bias, B.DTYPES[dtype]).double()
    want = x.double() @ w.double().t().contiguous() * sx.double()[:, None] * (sw / c).double()
    off = 4 * B.SUM * want.abs()
    want += bias.double()
    off += (B.SUM + B.UNIT[B.DTYPES[dtype]]) * want.abs() + B.TINY[B.DTYPES[dtype]]
    assert ((y - want).abs() <= off).all()


def test_far_rows():
    """Rows behind 2^32 bytes of x, and results behind 2^32 elements."""
    from FGMS import nn
    gen = torch.Generator().manual_seed(2)
    w, sw = eighths(24, 16000, gen, 1)
    x = torch.zeros(270000, 16000, dtype=torch.int8, device="cuda")
    at = torch.tensor([0, 1, 134217, 134218, 268435, 268436, 269998, 269999], device="cuda")
    few, _ = eighths(8, 16000, gen, 0)
    x[at] = few
    scales = torch.ones(270000, device="cuda") / 16000
    y = nn.int8_linear(x, scales, w, sw, None, torch.float32)
    B.within(y[at], *B.product(few, scales[:8], w, sw, None, torch.float32), "far rows")
    y[at] = 0
    assert not y.any()
    del x, y
    w, sw = eighths(8000, 24, gen, 1)
    x = torch.zeros(600000, 32, dtype=torch.int8, device="cuda")[:, :24]
    few, _ = eighths(3, 24, gen, 0)
    x[[7, 536870, 599999]] = few
    y = nn.int8_linear(x, torch.ones(600000, device="cuda"), w, sw, None, torch.float16)
    B.within(y[[7, 536870, 599999]], *B.product(few, torch.ones(3), w, sw, None, torch.float16), "far results")
    assert not y[536871:599999].any()


def test_largest_sums():
    """Sums at the ends of 32 bits."""
    from FGMS import nn
    c = 131071
    x = torch.full((2, c + 1), -128, dtype=torch.int8, device="cuda")[:, :c]
    w = torch.full((3, c + 1), -128, dtype=torch.int8, device="cuda")[:, :c].clone()
    w[1] = 127
    one = torch.ones(3, device="cuda")
    y = nn.int8_linear(x, one[:2], w, one, dtype=torch.float32)
    want = torch.tensor([128 * 128 * c, -128 * 127 * c, 128 * 128 * c], dtype=torch.float32, device="cuda")
    assert torch.equal(y, want.expand(2, 3))
    with pytest.raises(ValueError, match="131071"):
        nn.int8_linear(x.new_zeros(2, c + 1), one[:2], x.new_zeros(3, c + 1), one)


def test_refusals():
    from FGMS import nn
    q, s = torch.zeros(4, 32, dtype=torch.int8, device="cuda"), torch.ones(4, device="cuda")
    for bad in ((q.float(), s, q, s), (q, s, q.int(), s), (q, s[:3], q, s), (q, s, q, s.half()), (q, s[:, None], q, s), (q, s, q[:, :16], s),
                (q, s, q.cpu(), s), (q, s.cpu(), q, s), (q, s, q, s, s), (q, s, q, s, s[:2].half()), (q, s, q, s, None, torch.float64),
                (q[:, :0], s, q[:, :0], s), (q, s, q[:0], s[:0])):
        with pytest.raises(ValueError):
            nn.int8_linear(*bad)
    with pytest.raises(ValueError, match="no gradients"):
        nn.int8_linear(q, s.requires_grad_(), q, s)
    with pytest.raises(ValueError, match="halves"):
        nn.quantize_rows(torch.zeros(2, 7, device="cuda"), gated=True)

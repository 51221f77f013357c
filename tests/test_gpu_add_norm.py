"""Sums with dropout and their norms (FGMS.nn.add_norm, dropout_add), and their gradients, against the plain formulas in 64 bits."""
import pytest
import torch

from tests import block_util as B

pytestmark = pytest.mark.gpu

# rows, channels
SHAPES = [(1, 8), (1, 1), (3, 5), (257, 8), (1000, 16), (301, 40), (77, 63), (130, 64), (129, 128), (61, 200), (50, 512), (33, 520), (40, 1024),
          (37, 1096), (19, 2048), (18, 2056), (9, 4096), (7, 4104), (6, 8192), (5, 8200), (3, 12001), (4, 16384), (20000, 32), (4100, 256)]


def features(n, c, dtype, gen, by=1.0):
    return (by * torch.randn(n, c, generator=gen)).to(B.DTYPES[dtype]).cuda()


def seed_of(gen):
    return torch.randint(-1 << 63, (1 << 63) - 1, (2,), generator=gen).cuda()


def check_norm(x, residual, scale, p, seed, gy, gh, eps=1e-6):
    from FGMS import nn
    leaves = [t for t in (x, residual, scale) if t is not None]
    factor = B.factors(*x.shape, p, seed) if p else torch.ones(x.shape, dtype=torch.float64)
    out = nn.add_norm(x, residual, scale, eps, p, seed)
    both = residual is not None or p > 0
    if both:
        B.within(out[1], *B.total(x, residual, factor), "sum")
    else:
        assert out[1] is x
    y, off = B.normed(out[1], scale, eps)
    B.within(out[0], y, off, "norm")
    used = (out, (gy, gh)) if both else (out[:1], (gy,))
    got = dict(zip((n for n, t in (("x", x), ("residual", residual), ("scale", scale)) if t is not None),
                   torch.autograd.grad(used[0], leaves, used[1], retain_graph=True)))
    gs, gs_off, gx, gx_off, gw, gw_off = B.norm_grads(out[1], scale, eps, gy, gh if both else None, factor)
    B.within(got["x"], gx, gx_off, "gradient of x")
    if residual is not None:
        B.within(got["residual"], gs, gs_off, "gradient of the residual")
    if scale is not None:
        B.within(got["scale"], gw, gw_off, "gradient of the scale")
    again = torch.autograd.grad(used[0], leaves, used[1], retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got.values(), again))
    # each gradient on its own, and of one output alone
    for leaf, g in zip(leaves, got.values()):
        assert torch.equal(torch.autograd.grad(used[0], leaf, used[1], retain_graph=True)[0], g)
    if both:
        alone = torch.autograd.grad(out[1], x, gh, retain_graph=True)[0]
        B.within(alone, B.cpu(gh) * factor, (B.UNIT[x.dtype] + 4 * B.SUM) * (B.cpu(gh) * factor).abs() + B.TINY[x.dtype], "gradient by the sum")
    return out


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_both_passes(shape, dtype):
    gen = torch.Generator().manual_seed(shape[0] * 31 + shape[1])
    x, residual, gy, gh = (features(*shape, dtype, gen) for _ in range(4))
    scale = (1 + 0.2 * torch.randn(shape[1], generator=gen)).to(B.DTYPES[dtype]).cuda().requires_grad_()
    x.requires_grad_(), residual.requires_grad_()
    check_norm(x, residual, scale, 0.0, None, gy, gh)
    check_norm(x, residual, scale, 0.25, seed_of(gen), gy, gh)


@pytest.mark.parametrize("dtype", list(B.DTYPES))
def test_inputs_that_are_not_there(dtype):
    gen = torch.Generator().manual_seed(5)
    x, residual, gy, gh = (features(211, 96, dtype, gen) for _ in range(4))
    x.requires_grad_(), residual.requires_grad_()
    scale = torch.full((96,), 0.5, dtype=B.DTYPES[dtype], device="cuda", requires_grad=True)
    check_norm(x, None, scale, 0.0, None, gy, gh)
    check_norm(x, None, None, 0.0, None, gy, gh)
    check_norm(x, residual, None, 0.0, None, gy, gh)
    check_norm(x, None, scale, 0.1, seed_of(gen), gy, gh)
    check_norm(x, residual, scale, 0.1, seed_of(gen), gy, gh, eps=0.5)


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("shape", [(40, 64), (9, 1096), (5, 4096)], ids=str)
def test_slices_and_orders(shape, dtype):
    """Rows of a wider tensor, on 16 bytes and not, broadcast rows, columns first: as the same values laid out row by row."""
    from FGMS import nn
    gen = torch.Generator().manual_seed(3)
    n, c = shape
    wide = features(n, 3 * c + 24, dtype, gen)
    seed = seed_of(gen)
    columns = features(c, n, dtype, gen)
    for x in (wide[:, 8:8 + c], wide[:, 16 + c:16 + 2 * c], wide[:, 3:3 + c], wide[:1, :c].expand(n, c), columns.t()):
        for residual in (wide[:, c + 8:2 * c + 8], wide[:, c + 1:2 * c + 1], None):
            plain = [t.contiguous() if t is not None else None for t in (x, residual)]
            for a, b in zip(nn.add_norm(x, residual, None, p=0.3, seed=seed), nn.add_norm(*plain, None, p=0.3, seed=seed)):
                assert torch.equal(a, b)
            assert torch.equal(nn.dropout_add(x, residual, 0.3, seed), nn.dropout_add(*plain, 0.3, seed))
            for a, b in zip(nn.add_norm_int8(x, residual), nn.add_norm_int8(*plain)):
                assert torch.equal(a, b)
    # gradients by way of a slice and of a transposed output gradient
    leaf = wide.clone().requires_grad_()
    y, h = nn.add_norm(leaf[:, 3:3 + c], None, None)
    g = columns.t()
    got = torch.autograd.grad(y, leaf, g)[0]
    part = wide[:, 3:3 + c].clone().requires_grad_()
    want = torch.autograd.grad(nn.add_norm(part, None, None)[0], part, g.contiguous())[0]
    assert torch.equal(got[:, 3:3 + c], want) and not got[:, 3 + c:].any() and not got[:, :3].any()


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("shape", [(1, 1), (7, 3), (1000, 8), (300, 72), (65, 1096), (31, 4096), (5, 16384)], ids=str)
def test_dropout(shape, dtype):
    from FGMS import nn
    gen = torch.Generator().manual_seed(shape[1])
    x, residual, g = (features(*shape, dtype, gen) for _ in range(3))
    x.requires_grad_(), residual.requires_grad_()
    for p in (0.0, 0.1, 0.5, 0.999):
        seed = seed_of(gen)
        factor = B.factors(*shape, p, seed)
        out = nn.dropout_add(x, residual, p, seed)
        B.within(out, *B.total(x, residual, factor), "sum")
        gx, gr = torch.autograd.grad(out, (x, residual), g)
        B.within(gx, B.cpu(g) * factor, (B.UNIT[x.dtype] + 4 * B.SUM) * (B.cpu(g) * factor).abs() + B.TINY[x.dtype], "gradient of x")
        assert torch.equal(gr, g)
        bare = nn.dropout_add(x, None, p, seed)
        B.within(bare, *B.total(x, None, factor), "without a residual")
        assert torch.equal(torch.autograd.grad(bare, x, g)[0], gx)


def test_seeds():
    """Every seed and stream number has words of its own; without one, torch's generator says which."""
    from FGMS import nn
    x = torch.ones(200, 64, device="cuda")
    seen = set()
    for seed in ((0, 0), (1, 0), (0, 1), (1 << 32, 0), (0, 1 << 32), (-1, 0), (0, -1), (-1 << 63, (1 << 63) - 1)):
        t = torch.tensor(seed, device="cuda")
        y = nn.dropout_add(x, None, 0.5, t)
        assert torch.equal(y.cpu().double(), B.factors(200, 64, 0.5, t))
        seen.add(tuple(y.flatten().tolist()))
    assert len(seen) == 8
    torch.manual_seed(7)
    a, b = nn.dropout_add(x, None, 0.5), nn.dropout_add(x, None, 0.5)
    torch.manual_seed(7)
    assert torch.equal(a, nn.dropout_add(x, None, 0.5)) and not torch.equal(a, b)
    # shares that no step of 2^-16 is nearer to than zero drop nothing
    assert torch.equal(nn.dropout_add(x, None, 2.0 ** -18, t), x)
    assert nn.add_norm(x, None, None, p=2.0 ** -18, seed=t)[1] is x


def test_differences():
    """Gradients of both operators against differences, in fp32 over a function that is smooth at a fixed seed."""
    from FGMS import nn
    gen = torch.Generator().manual_seed(11)
    x, residual, gy, gh = (features(6, 24, "fp32", gen) for _ in range(4))
    scale = (1 + 0.2 * torch.randn(24, generator=gen)).cuda()
    seed = torch.tensor([5, 9], device="cuda")
    factor = B.factors(6, 24, 0.25, seed)
    leaves = [t.requires_grad_() for t in (x, residual, scale)]

    def value(x, residual, scale):      # the same function in 64 bits
        h = x * factor + residual
        return ((h * scale / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-6)) * B.cpu(gy)).sum() + (h * B.cpu(gh)).sum()

    got = torch.autograd.grad(nn.add_norm(x, residual, scale, p=0.25, seed=seed), leaves, (gy, gh))
    at = [B.cpu(t) for t in leaves]
    for i, g in enumerate(got):
        for place in range(0, at[i].numel(), 7):
            step = 1e-5
            ends = []
            for d in (step, -step):
                moved = [t.clone() for t in at]
                moved[i].view(-1)[place] += d
                ends.append(value(*moved))
            want = float(ends[0] - ends[1]) / (2 * step)
            assert abs(float(g.view(-1)[place]) - want) < 1e-4 * max(1.0, abs(want))


def test_values_that_are_no_numbers():
    """An infinity or NaN stays in its row; one that is dropped is gone."""
    from FGMS import nn
    for dtype in B.DTYPES.values():
        x = torch.ones(9, 72, dtype=dtype, device="cuda")
        clean = nn.add_norm(x, x, None)
        x[2, 5], x[6, 70] = float("inf"), float("nan")
        y, h = nn.add_norm(x, torch.ones_like(x), None)
        rest = [i for i in range(9) if i not in (2, 6)]
        assert torch.equal(y[rest], clean[0][rest]) and torch.equal(h[rest], clean[1][rest])
        assert h[2, 5] == float("inf") and y[6].isnan().all()
        assert y[2, 5].isnan()
        seed = torch.tensor([3, 4], device="cuda")
        factor = B.factors(9, 72, 0.5, seed).cuda()
        y = nn.dropout_add(x, None, 0.5, seed)
        assert not (factor == 0)[~y.isfinite()].any() and (y[factor == 0] == 0).all()
        zero = torch.zeros(3, 72, dtype=dtype, device="cuda", requires_grad=True)
        y = nn.add_norm(zero, None, None)[0]
        assert (y == 0).all() and torch.autograd.grad(y, zero, torch.ones_like(y))[0].isfinite().all()


def test_far_rows():
    """Rows behind 2^32 bytes and 2^31 elements, and their words."""
    from FGMS import nn
    n, c = 140000, 16384
    seed = torch.tensor([11, 12], device="cuda")
    x = torch.zeros(n, c, dtype=torch.float16, device="cuda")
    x[-1] = 1
    y, h = nn.add_norm(x, None, None, p=0.5, seed=seed)
    per = c // 8
    words = B.philox([torch.arange((n - 1) * per, n * per), torch.zeros(per, dtype=torch.int64), torch.full((per,), 12), torch.zeros(per, dtype=torch.int64)], [11, 0])
    words = torch.stack([w >> shift & 0xFFFF for w in words for shift in (0, 16)], 1).reshape(1, c)
    want = 2.0 * (words >= 32768)
    assert torch.equal(h[-1:].cpu().double(), want.double()) and not h[:-1].any() and not y[:-1].any()
    B.within(y[-1:], *B.normed(h[-1:], None, 1e-6), "norm")
    assert torch.equal(nn.dropout_add(x, None, 0.5, seed)[-1], h[-1])
    del y, h
    q, scales, _ = nn.add_norm_int8(x)
    assert (q[-1] == 127).all() and not q[-2].any() and not scales[:-1].any()
    g = torch.ones(n, c, dtype=torch.float16, device="cuda")
    x[-1, ::2] = 3
    leaf = x.requires_grad_()
    got = torch.autograd.grad(nn.add_norm(leaf, None, None)[0], leaf, g)[0]
    row = x[-1:].detach()
    gs, off, *_ = B.norm_grads(row, None, 1e-6, g[-1:], None, torch.ones(1, c, dtype=torch.float64))
    B.within(got[-1:], gs, off, "gradient")


def test_more_rows_than_a_launch_takes():
    """Both sides of the row that the second launch begins with."""
    from FGMS import nn
    if torch.cuda.mem_get_info()[0] < 150 << 30:
        pytest.skip("needs 150 GB")
    n, c = (1 << 25) + 5, 512
    at = torch.tensor([0, (1 << 25) - 1, 1 << 25, n - 1])
    gen = torch.Generator().manual_seed(1)
    rows = features(4, c, "fp16", gen)
    x = torch.zeros(n, c, dtype=torch.float16, device="cuda")
    x[at] = rows
    per = c // 8
    chunk = (at[:, None] * per + torch.arange(per)).flatten()
    words = B.philox([chunk & B.MASK, chunk >> 32, torch.full_like(chunk, 12), torch.zeros_like(chunk)], [11, 0])
    words = torch.stack([w >> shift & 0xFFFF for w in words for shift in (0, 16)], 1).reshape(4, c)
    factor = 2.0 * (words >= 32768).double()
    seed = torch.tensor([11, 12], device="cuda")
    y, h = nn.add_norm(x, None, None, p=0.5, seed=seed)
    B.within(h[at], *B.total(rows, None, factor), "sum")
    B.within(y[at], *B.normed(h[at], None, 1e-6), "norm")
    kept = h[at]
    del y, h
    out = nn.dropout_add(x, None, 0.5, seed)
    assert torch.equal(out[at], kept)
    out[at] = 0
    assert not out.any()
    del out
    q, scales = nn.quantize_rows(x)
    few = nn.quantize_rows(rows)
    assert torch.equal(q[at], few[0]) and torch.equal(scales[at], few[1])
    q[at] = 0
    assert not q.any()


def test_captured_seeds():
    """Seeds that a captured call draws are new ones at every replay."""
    from FGMS import nn
    x = torch.ones(100, 64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    nn.dropout_add(x, None, 0.5)
    with torch.cuda.graph(graph):
        y = nn.dropout_add(x, None, 0.5)
    seen = []
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(y.clone())
        assert ((y == 0) | (y == 2)).all() and abs(float(y.mean()) - 1) < 0.2
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_no_rows():
    from FGMS import nn
    x = torch.zeros(0, 24, device="cuda", requires_grad=True)
    scale = torch.ones(24, device="cuda", requires_grad=True)
    y, h = nn.add_norm(x, x, scale, p=0.1)
    assert y.shape == h.shape == (0, 24)
    gx, gw = torch.autograd.grad(y, (x, scale), torch.zeros_like(y))
    assert gx.shape == (0, 24) and torch.equal(gw, torch.zeros_like(scale))
    assert nn.dropout_add(x, None, 0.1).shape == (0, 24)
    q, scales, _ = nn.add_norm_int8(x.detach())
    assert q.shape == (0, 24) and scales.shape == (0,)
    assert nn.int8_linear(q, scales, torch.zeros(5, 24, dtype=torch.int8, device="cuda"), torch.ones(5, device="cuda")).shape == (0, 5)


def test_gpu_refusals():
    from FGMS import nn
    x = torch.zeros(4, 24, device="cuda")
    for bad in (x[:3], x[:, :16], x.half(), x.cpu(), x[0]):
        with pytest.raises(ValueError):
            nn.add_norm(x, bad)
        with pytest.raises(ValueError):
            nn.dropout_add(x, bad)
    for bad in (x, x[0, :16], x[0].half(), x[0].cpu()):
        with pytest.raises(ValueError):
            nn.add_norm(x, None, bad)
    for bad in (torch.zeros(2, device="cuda"), torch.zeros(3, dtype=torch.int64, device="cuda"), torch.zeros(2, dtype=torch.int64)):
        with pytest.raises(ValueError, match="seed"):
            nn.dropout_add(x, None, 0.5, bad)
    for p in (1.0, -0.5, float("nan")):
        with pytest.raises(ValueError):
            nn.dropout_add(x, None, p, torch.zeros(2, dtype=torch.int64, device="cuda"))
    for bad in (x.double(), x.int()):
        with pytest.raises(ValueError, match="float32, float16 and bfloat16"):
            nn.add_norm(bad)
    with pytest.raises(ValueError, match="16384"):
        nn.add_norm(torch.zeros(1, 16385, device="cuda"))
    with pytest.raises(ValueError):
        nn.add_norm(x, eps=-1.0)
    seed = torch.tensor([1, 2], device="cuda")
    leaf = x.clone().requires_grad_()
    y = nn.add_norm(leaf, None, None, p=0.5, seed=seed)[0]
    seed += 1
    with pytest.raises(RuntimeError, match="seed has been modified"):
        y.sum().backward()
    y, h = nn.add_norm(leaf, x, None)
    h.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    with pytest.raises(ValueError, match="no gradients"):
        nn.add_norm_int8(leaf)
    with pytest.raises(ValueError, match="no gradients"):
        nn.quantize_rows(leaf)

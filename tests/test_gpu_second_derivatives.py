"""Gradients of gradients (create_graph=True): those of dropout_add against the formula, and where there are none a refusal in place
of a part that is left out."""
import pytest
import torch

from tests import block_util as B

pytestmark = pytest.mark.gpu


def features(n, c, seed, dtype=torch.float32):
    return torch.randn(n, c, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()


@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("shape", [(40, 64), (7, 13)], ids=str)
def test_dropout_add(shape, p):
    """A gradient penalty over y = f x^3 + x, f what dropout multiplies with: g = v (3 f x^2 + 1); d(g^2)/dx = 12 g v f x, d(g^2)/dv = 2 g
    (3 f x^2 + 1).  Each of some ten operations rounds at 2^-24 of terms that are no larger than those with their signs taken away."""
    from FGMS import nn
    x, v = features(*shape, 1).requires_grad_(), features(*shape, 2).requires_grad_()
    seed = torch.tensor([3, 8], device="cuda")
    f = B.factors(*shape, p, seed)
    g, = torch.autograd.grad(nn.dropout_add(x ** 3, x, p, seed), x, v, create_graph=True)
    gx, gv = torch.autograd.grad((g * g).sum(), (x, v))
    a, b = B.cpu(x), B.cpu(v)
    slope = 3 * f * a ** 2 + 1
    step = 32 * 2.0 ** -24
    B.within(g, b * slope, step * b.abs() * slope + 1e-30, "gradient")
    B.within(gx, 12 * b ** 2 * slope * f * a, step * 12 * b ** 2 * slope * f * a.abs() + 1e-30, "by x")
    B.within(gv, 2 * b * slope ** 2, step * 2 * b.abs() * slope ** 2 + 1e-30, "by the output gradient")


def test_dropout_add_third_derivatives_and_changed_seeds():
    from FGMS import nn
    x, v = features(9, 24, 3).requires_grad_(), features(9, 24, 4).requires_grad_()
    seed = torch.tensor([1, 2], device="cuda")
    f = B.factors(9, 24, 0.5, seed).float().cuda()
    g, = torch.autograd.grad(nn.dropout_add(x, None, 0.5, seed), x, v, create_graph=True)
    gg, = torch.autograd.grad(g, v, x, create_graph=True)
    assert torch.equal(g, f * v) and torch.equal(gg, f * x) and torch.equal(torch.autograd.grad(gg.sum(), x)[0], f)
    g, = torch.autograd.grad(nn.dropout_add(x, None, 0.5, seed), x, v, create_graph=True)
    seed += 1
    with pytest.raises(RuntimeError, match="seed has been modified"):
        torch.autograd.grad(g, v, x)


@pytest.mark.parametrize("p", [0.0, 0.25])
def test_add_norm_refuses(p):
    """First derivatives are the same with and without a graph of them; to pass through one that depends on what is asked for is refused,
    also beside a path of torch's own."""
    from FGMS import nn
    x, w = features(20, 64, 5).requires_grad_(), features(1, 64, 6)[0].requires_grad_()
    r, gy, gh = features(20, 64, 7).requires_grad_(), features(20, 64, 8).requires_grad_(), features(20, 64, 9)
    seed = torch.tensor([3, 8], device="cuda")
    leaves = (x, r, w)
    out = nn.add_norm(x, r, w, p=p, seed=seed)
    want = torch.autograd.grad(out, leaves, (gy, gh), retain_graph=True)
    got = torch.autograd.grad(out, leaves, (gy, gh), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    for g in got:
        for by in (x, r, gy):
            with pytest.raises(NotImplementedError, match="add_norm has no second derivatives"):
                torch.autograd.grad(g.sum() + (by ** 2).sum(), by, retain_graph=True)
    for g in got[:2]:
        with pytest.raises(NotImplementedError, match="second derivatives"):
            torch.autograd.grad(g.sum(), w, retain_graph=True)
    # x as the branch and as the residual: the path through the square has a second derivative, the norm's has none
    y, h = nn.add_norm(x ** 2, x, w, p=p, seed=seed)
    g, = torch.autograd.grad((y * h).sum(), x, create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        g.square().sum().backward()
    # what depends on no leaf is a constant, as it always was
    g, = torch.autograd.grad(nn.add_norm(x.detach(), None, w)[0], w, gh, create_graph=True)
    assert not g.requires_grad
    # a norm of the features themselves
    g, = torch.autograd.grad(nn.add_norm(x, None, None)[0], x, gh, create_graph=True)
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad(g.sum(), x)


def test_blocks_still_train_with_a_graph_of_their_gradients():
    """The same gradients but for silu's, which torch forms by another formula where a graph of it is asked for, s (1 + a (1 - s)) in separate
    operations: five roundings at 2^-24 of terms no larger than 1.3 times the result's largest, on their way through the block's products; twenty
    operations with their sums of 64 to 128 products differ by less than 4096 such steps (as in test_block_is_its_formula), these by a part of that."""
    from FGMS import nn
    from tests import attention_util as U
    torch.manual_seed(1)
    block = nn.VoxelBlock(32, 4, sections=(2, 1, 1), device="cuda")
    feats, coords = features(40, 32, 10), torch.zeros(40, 3, dtype=torch.int32, device="cuda")
    loss = block(feats, coords, U.offsets([40])).square().mean()
    want = torch.autograd.grad(loss, list(block.parameters()), retain_graph=True)
    got = torch.autograd.grad(loss, list(block.parameters()), create_graph=True)
    for a, b in zip(want, got):
        assert float((a - b).detach().abs().max()) < 4096 * 2.0 ** -24 * float(a.abs().max())


def refuses(grads, of):
    """The gradients that depend on `of` refuse a second pass, also beside a path of torch's own."""
    for g in grads:
        with pytest.raises(NotImplementedError, match="second derivatives"):
            torch.autograd.grad(g.sum() + (of ** 2).sum(), of, retain_graph=True)


def test_attention_refuses():
    from FGMS import nn
    from tests import attention_util as U
    gen = torch.Generator().manual_seed(4)
    q, k, v, g, gk = (torch.randn(30, 2, 16, generator=gen).cuda().requires_grad_() for _ in range(5))
    w, u = torch.randn(2, 16, generator=gen).cuda().unbind()
    w, u = w.clone().requires_grad_(), u.clone().requires_grad_()
    coords, freqs = torch.randint(0, 50, (30, 3), generator=gen, dtype=torch.int32).cuda(), nn.rotary_freqs((3, 3, 2)).cuda()
    turned = nn.norm_rotary(q, k, w, u, coords, freqs, (3, 3, 2))
    want = torch.autograd.grad(turned, (q, k, w, u), (g, gk), retain_graph=True)
    gq_, gk_, gw, gu = torch.autograd.grad(turned, (q, k, w, u), (g, gk), create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, (gq_, gk_, gw, gu)))
    refuses((gq_, gw), q), refuses((gq_,), w), refuses((gq_, gw), g)
    refuses((gk_, gu), k), refuses((gk_,), u), refuses((gk_, gu), gk)
    # (neither side's gradients have a part of the other's)
    extra = torch.autograd.grad(gq_.sum() + (k ** 2).sum(), k, retain_graph=True)[0]
    assert torch.equal(extra, 2 * k)
    out = nn.segment_attention(q, k, v, U.offsets([10, 20]))
    want = torch.autograd.grad(out, (q, k, v), g, retain_graph=True)
    got = torch.autograd.grad(out, (q, k, v), g, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    refuses(got, q), refuses(got, k), refuses(got, g), refuses(got[:2], v)
    # values alone: a linear map, whose gradient by constants is one
    got, = torch.autograd.grad(nn.segment_attention(q.detach(), k.detach(), v, U.offsets([10, 20])), v, g.detach(), create_graph=True)
    assert not got.requires_grad


def test_sparse_conv_refuses():
    from fgms_amd import clouds
    from FGMS import nn
    from tests.test_gpu_voxel_attention import small_cloud
    coords = small_cloud(1)
    kmap = nn.KernelMap.from_coords(coords, coords, clouds.offsets_cube(3))
    gen = torch.Generator().manual_seed(5)
    x, w = torch.randn(len(coords), 32, generator=gen).cuda().requires_grad_(), torch.randn(27, 32, 32, generator=gen).cuda().requires_grad_()
    g = torch.randn(len(coords), 32, generator=gen).cuda().requires_grad_()
    gx, gw = torch.autograd.grad(nn.sparse_conv(x, w, kmap), (x, w), g, create_graph=True)
    refuses((gx,), w), refuses((gw,), x), refuses((gx, gw), g)
    assert torch.equal(torch.autograd.grad(gx.sum() + (x ** 2).sum(), x, retain_graph=True)[0], 2 * x)
    gx, = torch.autograd.grad(nn.sparse_conv(x, w.detach(), kmap), x, g.detach(), create_graph=True)
    assert not gx.requires_grad


class Takes(torch.autograd.Function):
    """b, whatever a is: a's gradient is none."""

    @staticmethod
    def forward(ctx, a, b):
        return b.clone()

    @staticmethod
    def backward(ctx, g):
        return None, g


def test_passes_that_bring_no_gradient():
    """A gradient that a pass reaches and brings nothing to refuses nothing."""
    from FGMS import nn
    x, v, w = features(20, 64, 11).requires_grad_(), features(20, 64, 12).requires_grad_(), features(1, 64, 13)[0]
    g, = torch.autograd.grad(nn.add_norm(x, None, w)[0], x, v, create_graph=True)
    gx, gv, gg = torch.autograd.grad(Takes.apply(g, v * 2).sum(), (x, v, g), allow_unused=True, retain_graph=True)
    assert gx is None and gg is None and torch.equal(gv, torch.full_like(v, 2))
    with pytest.raises(NotImplementedError, match="second derivatives"):
        torch.autograd.grad((Takes.apply(g, v) + g).sum(), x)

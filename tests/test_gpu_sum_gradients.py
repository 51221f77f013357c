"""Gradients of add_norm's sum by itself: the sum's own, whatever its rows hold."""
import pytest
import torch

from tests import block_util as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(B.DTYPES))
def test_rows_that_have_no_norm(dtype):
    """Infinities, NaN, and zeros with eps 0, in rows whose norm nobody reads: the gradient is the one that comes in, or what dropout leaves of it."""
    from FGMS import nn
    gen = torch.Generator().manual_seed(1)
    x, r, g = (torch.randn(12, 72, generator=gen).to(B.DTYPES[dtype]).cuda() for _ in range(3))
    w = torch.randn(72, generator=gen).to(B.DTYPES[dtype]).cuda().requires_grad_()
    x[2, 5], x[6, 70], x[8] = float("inf"), float("nan"), 0
    r[8] = 0
    x.requires_grad_(), r.requires_grad_()
    seed = torch.tensor([3, 4], device="cuda")
    h = nn.add_norm(x, r, w, 0.0)[1]
    gx, gr, gw = torch.autograd.grad(h, (x, r, w), g, retain_graph=True)
    assert torch.equal(gx, g) and torch.equal(gr, g) and torch.equal(gw, torch.zeros_like(w))
    for leaf, want in ((x, g), (r, g)):
        assert torch.equal(torch.autograd.grad(h, leaf, g, retain_graph=True)[0], want)
    wide = torch.randn(12, 99, generator=gen).to(B.DTYPES[dtype]).cuda()[:, 20:92]
    for out in (g, wide, g[:1].expand(12, 72), g.sum().expand(12, 72)):
        y, h = nn.add_norm(x, r, w, 0.0, 0.5, seed)
        gx, gr, gw = torch.autograd.grad(h, (x, r, w), out)
        want = torch.autograd.grad(nn.dropout_add(x, r, 0.5, seed), (x, r), out)
        assert torch.equal(gx, want[0]) and torch.equal(gr, want[1]) and torch.equal(gw, torch.zeros_like(w))
        assert gx.isfinite().all()
    # the seed is still the forward pass's, and a gradient of this gradient is there
    y, h = nn.add_norm(x, r, None, p=0.5, seed=seed)
    v = g.clone().requires_grad_()
    gx, = torch.autograd.grad(h, x, v, create_graph=True)
    factor = B.factors(12, 72, 0.5, seed).to(B.DTYPES[dtype]).cuda()
    assert torch.equal(torch.autograd.grad(gx, v, torch.ones_like(g))[0], factor)
    h = nn.add_norm(x, r, None, p=0.5, seed=seed)[1]
    seed += 1
    with pytest.raises(RuntimeError, match="seed has been modified"):
        torch.autograd.grad(h, x, g)

"""add_norm and add_norm_int8 without a sum as operators of torch's dispatcher: their results are their own, and x goes on as itself."""
import pytest
import torch

from tests import block_util as B

pytestmark = pytest.mark.gpu


def features(n, c, seed):
    return torch.randn(n, c, generator=torch.Generator().manual_seed(seed)).cuda()


def test_results_are_their_own():
    import FGMS.backend      # noqa: F401
    x = features(20, 64, 1)
    y, h = torch.ops.fgms.add_norm(x, None, None, 1e-6, 0.0, None)
    assert torch.equal(h, x) and h.data_ptr() != x.data_ptr()
    B.within(y, *B.normed(x, None, 1e-6), "norm")
    h = torch.ops.fgms.add_norm_int8(x, None, None, 1e-6)[2]
    assert torch.equal(h, x) and h.data_ptr() != x.data_ptr()
    leaf = x.clone().requires_grad_()
    y, h = torch.ops.fgms.add_norm(leaf, None, None, 1e-6, 0.0, None)
    assert torch.equal(torch.autograd.grad(h, leaf, x)[0], x)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -18])
def test_traces_without_a_sum(p):
    from FGMS import nn
    x, w, g = features(20, 64, 2), features(1, 64, 3)[0], features(20, 64, 4)
    seed = torch.tensor([1, 2], device="cuda")

    def chain(x):
        own = x * 2
        y, h = nn.add_norm(own, None, w, p=p, seed=seed)
        h.add_(1)      # (the features themselves: what reads them next sees it)
        q, scales, k = nn.add_norm_int8(own, None, w)
        k.mul_(3)
        return y, h + own, q, scales, k

    traced = torch.jit.trace(chain, (x,), check_trace=False)
    names = [n.kind() for n in traced.graph.nodes()]
    assert "fgms::norm" in names and "fgms::norm_int8" in names and "fgms::add_norm" not in names and "fgms::add_norm_int8" not in names
    for _ in range(3):      # (a trace is optimised after its first runs)
        assert all(torch.equal(a, b) for a, b in zip(traced(g), chain(g)))
    leaf = g.clone().requires_grad_()
    traced = torch.jit.trace(lambda x: nn.add_norm(x, None, w)[0], (x,), check_trace=False)
    assert torch.equal(torch.autograd.grad(traced(leaf), leaf, x)[0], torch.autograd.grad(nn.add_norm(leaf, None, w)[0], leaf, x)[0])
    with pytest.raises(ValueError, match="p must be"):
        torch.jit.trace(lambda x: nn.add_norm(x, None, w, p=-1.0, seed=seed)[0], (x,), check_trace=False)

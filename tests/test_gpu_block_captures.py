"""Backward passes of what goes around attention, captured while eager graphs of some of their leaves live."""
import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu


def features(seed):
    return torch.randn(64, 64, generator=torch.Generator().manual_seed(seed)).half().cuda()


def test_gradients_that_nobody_asks_for():
    """Leaves whose gradient the captured pass does not form may belong to an eager graph; those whose it forms may not."""
    from FGMS import nn
    x, r, g = features(1).requires_grad_(), features(2).requires_grad_(), features(3)
    w = features(4)[0].clone().requires_grad_()
    seed = torch.tensor([1, 2], device="cuda")
    side = U.own_stream()
    for call in (lambda a, b: nn.add_norm(a, b, w)[0], lambda a, b: nn.add_norm(a, b, w, p=0.5, seed=seed)[0], lambda a, b: nn.dropout_add(a, b, 0.5, seed)):
        want = torch.autograd.grad(call(x, r), x, g)[0]
        eager = nn.add_norm(g, r, w)[0]      # (r and w are its leaves)
        assert eager.requires_grad
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(call(x, r), x, g)[0]
        for _ in range(3):
            with torch.no_grad():
                got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = call(x, r)
            with pytest.raises(RuntimeError, match="eager pass"):
                torch.autograd.grad(y, (x, r), g)
        del eager, y

"""Offsets, coordinates and frequencies written to between the forward and the backward pass: refused, as torch refuses it for
the tensors that it saves."""
import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("which", ["q_offsets", "k_offsets", "both"])
def test_offsets(which):
    from FGMS import nn
    torch.manual_seed(0)
    q, k, v, g = (torch.randn(50, 2, 16, device="cuda").half() for _ in range(4))
    leaves = [t.requires_grad_() for t in (q, k, v)]
    qo = U.offsets([20, 30])
    ko = qo if which == "both" else U.offsets([20, 30])
    out = nn.segment_attention(*leaves, qo, ko)
    first = torch.autograd.grad(out, leaves, g, retain_graph=True)
    (ko if which == "k_offsets" else qo).copy_(U.offsets([35, 15]))
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, leaves, g, retain_graph=True)
    # the next forward pass takes them as they are
    out = nn.segment_attention(*leaves, U.offsets([20, 30]))
    assert all(torch.equal(a, b) for a, b in zip(first, torch.autograd.grad(out, leaves, g)))


@pytest.mark.parametrize("which", ["coords", "freqs"])
def test_turns(which):
    from FGMS import nn
    torch.manual_seed(1)
    sections = (4, 4)
    q, k = (torch.randn(30, 2, 16, device="cuda").requires_grad_() for _ in range(2))
    coords, freqs = torch.randint(0, 50, (30, 2), dtype=torch.int32, device="cuda"), nn.rotary_freqs(sections, device="cuda")
    out = nn.norm_rotary(q, k, None, None, coords, freqs, sections)
    (coords if which == "coords" else freqs).mul_(2)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(out, (q, k), out)


def test_tensors_of_inference_mode_are_taken():
    """They count no changes, and are taken as before."""
    from FGMS import nn
    torch.manual_seed(2)
    sections = (4, 4)
    with torch.inference_mode():
        coords, at = torch.randint(0, 50, (30, 2), dtype=torch.int32, device="cuda"), torch.tensor([0, 30], dtype=torch.int32, device="cuda")
    x = torch.randn(30, 2, 16, device="cuda").requires_grad_()
    q, k = nn.norm_rotary(x, x, None, None, coords, nn.rotary_freqs(sections, device="cuda"), sections)
    out = nn.segment_attention(q, k, x, at)
    assert torch.isfinite(torch.autograd.grad(out, x, torch.ones_like(out))[0]).all()

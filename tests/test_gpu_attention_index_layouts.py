"""Coordinates, frequencies, offsets and lengths that are slices of other tensors are copied, as queries and keys are."""
import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu


def test_coordinates_of_a_batched_cloud():
    from FGMS import nn
    torch.manual_seed(0)
    sections = (3, 3, 2)
    batched = torch.randint(0, 50, (40, 4), dtype=torch.int32, device="cuda")
    freqs = nn.rotary_freqs(sections, device="cuda")
    wide = torch.zeros(8, 2, device="cuda")
    wide[:, 1] = freqs
    x = torch.randn(40, 2, 16, device="cuda").requires_grad_()

    def run(coords, freqs):
        out = nn.norm_rotary(x, x, None, None, coords, freqs, sections)
        return out, lambda: torch.autograd.grad(out, x, [torch.ones_like(t) for t in out])[0]

    plain, plain_grad = run(batched[:, 1:].contiguous(), freqs)
    got, got_grad = run(batched[:, 1:], wide[:, 1])
    assert all(torch.equal(a, b) for a, b in zip(plain, got))
    batched.zero_()      # (the copy is what the backward pass reads)
    assert torch.equal(plain_grad(), got_grad())


def test_offsets_and_lengths():
    from FGMS import nn
    torch.manual_seed(1)
    q, k, v = (torch.randn(60, 2, 16, device="cuda").half() for _ in range(3))
    table = torch.tensor([[0, 0, 7], [25, 20, 30], [60, 60, 5]], dtype=torch.int32, device="cuda")
    cols = [c.contiguous() for c in table.T]
    want = nn.segment_attention(q, k, v, cols[0], cols[1], k_lengths=cols[2][:2])
    assert torch.equal(nn.segment_attention(q, k, v, table[:, 0], table[:, 1], k_lengths=table[:2, 2]), want)


def test_other_types_are_refused():
    from FGMS import nn
    x = torch.randn(4, 2, 16, device="cuda")
    at = torch.tensor([0, 4], device="cuda")
    with pytest.raises(ValueError, match="int32"):
        nn.segment_attention(x, x, x, at)
    with pytest.raises(ValueError, match="dimension"):
        nn.segment_attention(x, x, x, at.int()[None])

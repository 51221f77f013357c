"""Infinities and NaN in one segment do not reach another's rows, in either pass; forward, keys that a row does not see may hold anything."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu
LENGTHS = {"three": [90, 70, 40], "long": [1300, 900, 700], "windows": [7, 30, 1, 12, 40, 3] * 20}


@pytest.mark.parametrize("bad", [math.nan, math.inf], ids=str)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("lengths", list(LENGTHS))
@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_gradients(dtype, lengths, causal, bad):
    from FGMS import nn
    torch.manual_seed(0)
    lengths = LENGTHS[lengths]
    n, at = sum(lengths), U.offsets(lengths)
    tensors = [torch.randn(n, h, 40, device="cuda").to(U.DTYPES[dtype]) for h in (4, 2, 2, 4)]      # q, k, v, g

    def run():
        q, k, v, g = (t.detach() for t in tensors)
        leaves = [t.requires_grad_() for t in (q, k, v)]
        out = nn.segment_attention(*leaves, at, causal=causal)
        return [out.detach(), *torch.autograd.grad(out, leaves, g)]

    plain = run()
    first = lengths[0]
    rows = torch.ones(n, dtype=torch.bool, device="cuda")
    rows[first:first + lengths[1]] = False      # the second segment's
    for t in tensors:
        kept = t.clone()
        t[first + lengths[1] // 2] = bad
        assert all(torch.equal(a[rows], b[rows]) for a, b in zip(plain, run()))
        t.copy_(kept)
    assert all(torch.equal(a, b) for a, b in zip(plain, run()))


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_keys_that_are_not_seen(dtype, bad):
    from FGMS import nn
    torch.manual_seed(1)
    q, k, v = (torch.randn(200, h, 64, device="cuda").to(U.DTYPES[dtype]) for h in (4, 2, 2))
    at = U.offsets([200])
    plain = nn.segment_attention(q, k, v, at, causal=True)
    for row in (199, 150, 64, 3):
        other = k.clone()
        other[row:] = bad
        assert torch.equal(nn.segment_attention(q, other, v, at, causal=True)[:row], plain[:row])

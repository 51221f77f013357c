"""Rows in front of the first key that causal order shows them are zeros, and so are their gradients, whatever keys and values hold."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf], ids=str)
@pytest.mark.parametrize("nq, nk", [(100, 50), (40, 39), (1300, 700)])
@pytest.mark.parametrize("d", [16, 40, 64, 128])
@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_rows_without_keys(dtype, d, nq, nk, bad):
    from FGMS import nn
    torch.manual_seed(0)
    q, g = (torch.randn(nq, 4, d, device="cuda").to(U.DTYPES[dtype]) for _ in range(2))
    k, v = (torch.randn(nk, 2, d, device="cuda").to(U.DTYPES[dtype]) for _ in range(2))
    k[0], v[1] = bad, bad
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = nn.segment_attention(*leaves, U.offsets([nq]), U.offsets([nk]), causal=True)
    gq = torch.autograd.grad(out, q, g)[0]
    none = nq - nk
    assert torch.equal(out[:none], torch.zeros_like(out[:none]))
    assert torch.equal(gq[:none], torch.zeros_like(gq[:none]))
    assert not torch.isfinite(out[none:]).all()

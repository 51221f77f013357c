"""Rows whose scores are all minus infinity come out as rows without keys do, from one launch and from one cut along the keys."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("keys", [1, 40, 300, 6000])
@pytest.mark.parametrize("d", [16, 40, 64])
@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_all_scores_minus_infinity(dtype, d, keys):
    from fgms_amd import capi
    dtype = U.DTYPES[dtype]
    torch.manual_seed(0)
    q, k, v = (torch.randn(n, 2, d, device="cuda").to(dtype) for n in (3, keys, keys))
    q[..., 0] = 1.0
    k[..., 0] = -math.inf
    out, lse = torch.full_like(q, 7.0), torch.empty(3, 2, device="cuda")
    capi.segment_attention_fwd(q, k, v, out, lse, U.offsets([3]), U.offsets([keys]), scale=0.3)
    assert torch.equal(out, torch.zeros_like(out))
    assert (lse == -math.inf).all()
    # one finite score: its value, whatever part of the keys it lies in
    for at in {0, keys // 2, keys - 1}:
        other = k.clone()
        other[at, :, 0] = 0.5
        capi.segment_attention_fwd(q, other, v, out, lse, U.offsets([3]), U.offsets([keys]), scale=0.3)
        want = U.attention(q, other[at:at + 1], v[at:at + 1], [3], [1], False, 0.3)
        U.within(out, want.out, want.out_off, "out")
        U.within(lse, want.lse, want.lse_off + 2.0 ** -22, "lse")


@pytest.mark.parametrize("keys", [40, 6000])
def test_scores_that_are_no_number_stay(keys):
    from FGMS import nn
    torch.manual_seed(1)
    q, k, v = (torch.randn(n, 1, 32, device="cuda").half() for n in (2, keys, keys))
    k[keys // 2] = math.nan
    assert torch.isnan(nn.segment_attention(q, k, v, U.offsets([2]), U.offsets([keys]))).all()

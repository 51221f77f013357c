"""Gated rows in 8 bits at the far end of silu, where its exponential leaves the normal numbers."""
import pytest
import torch

from tests import block_util as B

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", list(B.DTYPES))
def test_far_below_zero(dtype):
    """Down to -87.25 values are silu's (its argument is rounded at up to 2 |a| halves of a step, the rest at a few), from -87.5 on zeros; a row's other
    values are what they are beside them."""
    from FGMS import nn
    t = B.DTYPES[dtype]
    a = torch.tensor([-60.0, -80.0, -87.0, -87.5, -88.0, -90.0, -100.0, -1000.0, -60000.0]).to(t)
    b = torch.full_like(a, 40000.0)
    x = torch.stack([a, b], 1)
    assert (a[:3] >= -87.25).all() and (a[3:] <= -87.5).all()
    q, scales = nn.quantize_rows(x.cuda(), gated=True)
    want = (B.cpu(a) * torch.sigmoid(B.cpu(a)) * B.cpu(b)).abs() / 127
    assert ((scales.cpu().double() - want)[:3].abs() <= B.SUM * (2 * a[:3].abs().double() + 20) * want[:3]).all()
    assert q[:3, 0].tolist() == [-127] * 3 and not scales[3:].any() and not q[3:].any()
    one = torch.cat([a, torch.ones(1, dtype=t), b, torch.ones(1, dtype=t)])[None].cuda()
    q, scales = nn.quantize_rows(one, gated=True)
    assert q.tolist() == [[0] * 9 + [127]] and abs(float(scales) * 127 - 0.7310585786) < 1e-6

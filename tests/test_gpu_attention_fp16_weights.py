"""fp16 attention with weights far below a row's largest, at the lower end of the type's range."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu
UNIT = U.UNIT[torch.float16]


@pytest.mark.parametrize("d", [16, 32, 40, 128])      # with the rows' sums out of a column of ones, and without
@pytest.mark.parametrize("above", [12.0, 15.0, 18.0])
@pytest.mark.parametrize("first", [True, False])
def test_weak_keys_beside_a_sink(d, above, first):
    """One key of zero value `above` every other: what is left of a row are the others, down to 2^-26 of the largest each.
    Weights are held times 2^7 at least: half a step of fp16's smallest numbers is 2^-32 of a row's largest weight; above
    those, and of the result, a half step is 2^-11 of the number, of the sums 2^-24 a term."""
    from FGMS import nn
    n, rows, size = 480, 70, 30000.0
    q, k = torch.zeros(rows, 1, d), torch.zeros(n, 1, d)
    q[..., 0] = 8.0
    sink = 0 if first else n - 1
    k[sink, 0, 0] = above / 8
    v = torch.full((n, 1, d), size)
    v[::3] /= 4
    v[sink] = 0
    q, k, v = (t.half().cuda() for t in (q, k, v))
    out = nn.segment_attention(q, k, v, U.offsets([rows]), U.offsets([n]), scale=1.0)
    weak = math.exp(-above)
    total = 1 + (n - 1) * weak
    sizes = v.double().cpu()[:, 0, 0]
    want = float(sizes.sum()) * weak / total
    off = (float(sizes.sum()) * (2.0 ** -32 + UNIT * weak) + want * (UNIT + (n + above * 4 + 64) * U.SUM)) * 1.01 + U.TINY[torch.float16]
    assert (out.double() - want).abs().max() <= off, (out.flatten()[:4], want, off)


def test_scores_that_rise_within_the_slack():
    """Rows whose maximum rises by less than 2^8 from tile to tile keep the first one: the weights' numbers grow to 2^15."""
    from FGMS import nn
    n, d = 448, 16
    q, k = torch.zeros(40, 1, d), torch.zeros(n, 1, d)
    q[..., 0] = 1.0
    k[:, 0, 0] = torch.arange(n) // 64 * 5.4
    v = torch.randn(n, 1, d, generator=torch.Generator().manual_seed(0))
    q, k, v = (t.half().cuda() for t in (q, k, v))
    out = nn.segment_attention(q, k, v, U.offsets([40]), U.offsets([n]), scale=1.0)
    want = U.attention(q, k, v, [40], [n], False, 1.0)
    U.within(out, want.out, want.out_off, "out")

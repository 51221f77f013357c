"""One row of queries, keys or values, whatever stride it carries: a slice of a tensor expanded over rows has a row stride of 0."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu
H, HK, D = 4, 2, 32


def single(heads, row, dtype, seed):
    """[1, heads, D] with a row stride of `row` elements."""
    t = torch.randn(heads * D, generator=torch.Generator().manual_seed(seed)).to(dtype).cuda()
    return t.as_strided((1, heads, D), (row, D, 1))


@pytest.mark.parametrize("row", [0, 8, HK * D])
@pytest.mark.parametrize("which", ["k", "v", "k and v", "all"])
@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_both_passes(dtype, which, row):
    from FGMS import nn
    dtype = U.DTYPES[dtype]
    rows = 1 if which == "all" else 5
    gen = torch.Generator().manual_seed(0)
    q, g = (torch.randn(rows, H, D, generator=gen).to(dtype).cuda() for _ in range(2))
    if which == "all":
        q = single(H, row, dtype, 1)
    k = single(HK, row if which != "v" else HK * D, dtype, 2)
    v = single(HK, row if which != "k" else HK * D, dtype, 3)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    assert leaves[2].stride(0) == v.stride(0)
    out = nn.segment_attention(*leaves, U.offsets([rows]), U.offsets([1]))
    want = U.attention(q, k, v, [rows], [1], False, 1 / math.sqrt(D), g)
    U.within(out, want.out, want.out_off, "out")
    for n, t in zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, g)):
        U.within(t, getattr(want, n), getattr(want, n + "_off"), n)


@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_expanded_over_rows(dtype):
    """The ordinary way to such a tensor; torch calls it contiguous."""
    from FGMS import nn
    dtype = U.DTYPES[dtype]
    torch.manual_seed(4)
    k, v = (torch.randn(1, HK, D, device="cuda").to(dtype).expand(80, -1, -1)[:1] for _ in range(2))
    assert k.stride(0) == 0 and k.is_contiguous()
    q = torch.randn(3, H, D, device="cuda").to(dtype)
    # (the middle segment has the key)
    out = nn.segment_attention(q, k, v, U.offsets([1, 1, 1]), U.offsets([0, 1, 0]))
    assert torch.equal(out[1], v[0].repeat_interleave(H // HK, 0)) and not out[0].any() and not out[2].any()


@pytest.mark.parametrize("row", [0, 8])
def test_c_entry(row):
    from fgms_amd import capi
    q, k, v = single(H, row, torch.float16, 5), single(HK, row, torch.float16, 6), single(HK, row, torch.float16, 7)
    out, lse, at = torch.empty(1, H, D, dtype=torch.float16, device="cuda"), torch.empty(1, H, device="cuda"), U.offsets([1])
    capi.segment_attention_fwd(q, k, v, out, lse, at, at, scale=0.25)
    want = U.attention(q, k, v, [1], [1], False, 0.25)
    U.within(out, want.out, want.out_off, "out")
    U.within(lse, want.lse, want.lse_off + 2.0 ** -22, "lse")

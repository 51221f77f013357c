"""Norms and rotation of queries alone (no key heads): the keys' scale has a gradient of zeros."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows", [0, 70])
@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_scale_without_keys(dtype, rows):
    from FGMS import nn
    dtype, d, sections = U.DTYPES[dtype], 16, (4, 4)
    torch.manual_seed(0)
    q, k = torch.randn(rows, 3, d, device="cuda").to(dtype), torch.empty(rows, 0, d, device="cuda", dtype=dtype)
    scales = [(1 + torch.randn(d, device="cuda") / 4).to(dtype) for _ in range(2)]
    coords = torch.randint(-50, 50, (rows, 2), dtype=torch.int32, device="cuda")
    freqs = nn.rotary_freqs(sections, device="cuda")
    leaves = [t.requires_grad_() for t in (q, k, *scales)]
    out = nn.norm_rotary(*leaves, coords, freqs, sections)
    g = torch.randn_like(out[0])
    # memory that the results may be given holds something else
    spoiled = [torch.full((d,), math.nan, dtype=dtype, device="cuda") for _ in range(64)]
    del spoiled
    got = torch.autograd.grad(out, leaves, (g, torch.empty_like(out[1])))
    assert got[1].shape == (rows, 0, d)
    assert torch.equal(got[3], torch.zeros_like(got[3]))
    _, _, gx, gx_off, gw, gw_off = U.turned(q, scales[0], coords, freqs, sections, 1e-6, False, g)
    U.within(got[0], gx, gx_off, "gradient of q")
    U.within(got[2], gw, gw_off, "gradient of q's scale")


@pytest.mark.parametrize("rows", [0, 70])
def test_c_entry(rows):
    from fgms_amd import capi
    d, sections = 8, (2,)
    q, g = torch.ones(rows, 1, d, device="cuda"), torch.ones(rows, 1, d, device="cuda")
    none, scale = torch.empty(rows, 0, d, device="cuda"), torch.ones(d, device="cuda")
    coords, freqs = torch.zeros(rows, 1, dtype=torch.int32, device="cuda"), torch.ones(2, device="cuda")
    gq, gqs, gks = torch.empty_like(q), torch.full_like(scale, math.nan), torch.full_like(scale, math.nan)
    capi.norm_rotary_bwd(g, none, q, none, scale, scale, coords, freqs, sections, gq, none, gqs, gks)
    assert torch.equal(gks, torch.zeros_like(gks))
    assert torch.isfinite(gqs).all()

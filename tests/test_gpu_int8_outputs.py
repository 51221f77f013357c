"""Products of few rows with very many outputs (a vocabulary's): every rule that chooses tiles by their number alone, rows far from filling them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("channels", [72, 520, 1100, 4096])
def test_few_rows_of_many_outputs(channels):
    """Whole numbers under 2^24 with scales that are powers of two: exact but for the result's own rounding."""
    from FGMS import nn
    gen = torch.Generator(device="cuda").manual_seed(channels)
    padded = (channels + 15) // 16 * 16
    w = torch.randint(-9, 10, (131073, padded), generator=gen, device="cuda").to(torch.int8)[:, :channels]
    x = torch.randint(-9, 10, (70, padded), generator=gen, device="cuda").to(torch.int8)[:, :channels]
    sums = x.float() @ w.float().t() / 8
    sx, sw = torch.ones(70, device="cuda"), torch.full((131073,), 0.125, device="cuda")
    for rows in (1, 2, 16, 17, 32, 33, 40, 64, 70):
        for outputs in (8192, 8193, 32641, 65281, 65537, 128256, 131073):
            for dtype in (torch.float16, torch.bfloat16, torch.float32):
                y = nn.int8_linear(x[:rows], sx[:rows], w[:outputs], sw[:outputs], None, dtype)
                assert torch.equal(y, sums[:rows, :outputs].to(dtype)), (rows, outputs, dtype)

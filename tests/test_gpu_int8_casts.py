"""Layers in 8 bits through every way that a module is cast or moved."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("channels", [40, 48])
def test_casts(channels):
    from FGMS import nn
    torch.manual_seed(1)
    layer = nn.Int8Linear(torch.nn.Linear(channels, 7, device="cuda"))
    x = torch.randn(9, channels, device="cuda")
    weight, scales = layer.weight.clone(), layer.weight_scales.clone()
    with torch.no_grad():
        want = layer(x)
        for cast in (lambda: layer.type(torch.float16), lambda: layer.to(torch.bfloat16), lambda: layer.half(), lambda: layer.to("cpu", torch.float16), lambda: layer.cuda(),
                     lambda: layer.type(torch.float32), lambda: layer.float()):
            cast()
            assert layer.weight.dtype == torch.int8 and layer.weight_scales.dtype == torch.float32 and layer.weight.stride(0) % 16 == 0
            assert torch.equal(layer.weight.cuda(), weight) and torch.equal(layer.weight_scales.cuda(), scales)
            if layer.weight.is_cuda:
                assert layer(x.to(layer.dtype)).dtype == layer.dtype
        assert layer.dtype == torch.float32 and layer(x).shape == want.shape
        # without storage, and with some again
        state = {k: v.clone() for k, v in layer.state_dict().items()}
        layer.to("meta").to_empty(device="cuda")
        assert layer.weight.dtype == torch.int8 and layer.weight_scales.is_cuda and layer.weight.stride(0) % 16 == 0
        layer.load_state_dict(state)
        assert torch.equal(layer(x), nn.int8_linear(*nn.quantize_rows(x), weight, scales, state["bias"], torch.float32))

"""What the entry points around attention refuse, before any device work; and the generator's words."""
import ctypes
import math

import pytest
import torch

from tests import block_util as B

P = ctypes.c_void_p(4096)      # (a pointer that no kernel may see: every call below is refused)
ODD = ctypes.c_void_p(4097)
EIGHT = ctypes.c_void_p(4104)
NULL = ctypes.c_void_p()


def call(name, **given):
    from fgms_amd import capi
    return getattr(capi.lib(), name)(*given.values()), capi.lib().fgms_last_error().decode()


def norm_fwd(**change):
    a = dict(x=P, residual=P, scale=P, sum=P, out=P, n=4, channels=24, x_row=24, residual_row=24, eps=1e-6, p=0.1, seed=P, dtype=1, stream=NULL)
    return call("fgms_add_norm_fwd", **{**a, **change})


def norm_bwd(**change):
    a = dict(out=P, sum_grad=P, x=P, scale=P, x_grad=P, residual_grad=P, scale_grad=P, scale_sums=P, n=4, channels=24, x_row=24, eps=1e-6, p=0.1,
             seed=P, dtype=1, stream=NULL)
    return call("fgms_add_norm_bwd", **{**a, **change})


def drop(**change):
    a = dict(x=P, residual=P, out=P, n=4, channels=24, x_row=24, residual_row=24, p=0.1, seed=P, dtype=1, stream=NULL)
    return call("fgms_dropout_add", **{**a, **change})


def eighths(**change):
    a = dict(x=P, out=P, scales=P, n=4, channels=24, x_row=48, out_row=32, gated=1, dtype=1, stream=NULL)
    return call("fgms_quantize_rows", **{**a, **change})


def norm_eighths(**change):
    a = dict(x=P, residual=P, scale=P, sum=P, out=P, scales=P, n=4, channels=24, x_row=24, residual_row=24, out_row=32, eps=1e-6, dtype=1, stream=NULL)
    return call("fgms_add_norm_int8", **{**a, **change})


def linear(**change):
    a = dict(x=P, x_scales=P, weight=P, weight_scales=P, bias=P, out=P, n=4, outputs=8, channels=24, x_row=32, weight_row=32, dtype=1, stream=NULL)
    return call("fgms_int8_linear", **{**a, **change})


COMMON = [dict(dtype=3), dict(dtype=-1), dict(n=-1), dict(n=1 << 31), dict(channels=0), dict(channels=-8)]
ROWS = COMMON + [dict(channels=16385), dict(x=NULL), dict(x=ODD), dict(x_row=-1), dict(x_row=1 << 50)]
EPS = [dict(eps=-1.0), dict(eps=math.nan), dict(eps=math.inf)]
DROPS = [dict(p=-0.1), dict(p=1.0), dict(p=1 - 2.0 ** -20), dict(p=math.nan), dict(seed=NULL), dict(seed=ctypes.c_void_p(4100))]
REFUSED = [(norm_fwd, ROWS + EPS + DROPS + [dict(out=NULL), dict(residual=ODD), dict(residual_row=-1), dict(scale=ODD), dict(sum=ODD)]),
           (norm_bwd, ROWS + EPS + DROPS + [dict(out=NULL), dict(sum_grad=ODD), dict(x_grad=ODD), dict(scale_sums=NULL), dict(scale_sums=ODD)]),
           (drop, ROWS + DROPS + [dict(out=NULL), dict(out=ODD), dict(residual=ODD)]),
           (eighths, ROWS + [dict(out=NULL), dict(scales=NULL), dict(scales=ODD), dict(out_row=23)]),
           (norm_eighths, ROWS + EPS + [dict(out=NULL), dict(scales=NULL), dict(sum=ODD), dict(out_row=0)]),
           (linear, COMMON + [dict(channels=131072, x_row=131072, weight_row=131072), dict(outputs=0), dict(outputs=(1 << 20) + 1), dict(x=NULL),
                              dict(x=EIGHT), dict(weight=NULL), dict(weight=EIGHT), dict(x_scales=NULL), dict(weight_scales=ODD), dict(bias=ODD),
                              dict(out=NULL), dict(x_row=16), dict(weight_row=24), dict(x_row=40), dict(x_row=(4 << 20) + 16)])]


@pytest.mark.parametrize("entry, change", [(f, c) for f, cs in REFUSED for c in cs], ids=lambda v: v.__name__ if callable(v) else next(iter(v)))
def test_c_entries_refuse(entry, change):
    rc, message = entry(**change)
    assert rc == -1 and message.startswith("fgms_"), (rc, message)


def test_nothing_to_do_is_no_error():
    for entry in (norm_fwd, drop, eighths, norm_eighths, linear):
        assert entry(n=0, x=NULL, out=NULL)[0] == 0
    assert norm_bwd(n=0, x=NULL, out=NULL, scale_grad=NULL)[0] == 0
    from fgms_amd import capi
    assert capi.lib().fgms_add_norm_bwd_sums(0, 8) == 0 and capi.lib().fgms_add_norm_bwd_sums(5, 0) == 0
    assert capi.lib().fgms_add_norm_bwd_sums(1, 24) == 24


def test_python_entries_refuse():
    from FGMS import nn
    x, q = torch.zeros(4, 24), torch.zeros(4, 24, dtype=torch.int8)
    for f in (nn.add_norm, nn.dropout_add, nn.quantize_rows, nn.add_norm_int8):
        with pytest.raises(ValueError, match="GPU tensor"):
            f(x) if f is not nn.dropout_add else f(x, p=0.0)
        with pytest.raises(ValueError, match="expected x"):
            f(x[0]) if f is not nn.dropout_add else f(x[0], p=0.0)
    with pytest.raises(ValueError, match="GPU tensor"):
        nn.int8_linear(q, x[:, 0], q, x[:, 0])
    with pytest.raises(ValueError, match="expected x"):
        nn.int8_linear(q, x[:, 0], q[:, :8], x[:, 0])
    with pytest.raises(ValueError):
        nn.VoxelBlock(64, 4, hidden=0)
    with pytest.raises(ValueError):
        nn.VoxelBlock(64, 4, p=1.0)
    with pytest.raises(ValueError):
        nn.VoxelBlock(64, 5)


def test_generator():
    """The published outputs of Philox4x32-10 for a counter and key of zeros, of ones, and of digits of pi."""
    assert B.philox([0] * 4, [0] * 2) == [0x6627e8d5, 0xe169c58d, 0xbc57ac4c, 0x9b00dbd8]
    assert B.philox([B.MASK] * 4, [B.MASK] * 2) == [0x408f276d, 0x41c83b0e, 0xa20bc7c6, 0x6d5451fd]
    assert B.philox([0x243f6a88, 0x85a308d3, 0x13198a2e, 0x03707344], [0xa4093822, 0x299f31d0]) == [0xd16cfe09, 0x94fdcceb, 0x5001e420, 0x24126ea1]

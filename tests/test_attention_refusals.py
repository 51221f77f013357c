"""What the attention entry points refuse, before any device work."""
import ctypes
import math

import pytest
import torch


def test_python_entries_refuse():
    from FGMS import nn
    q, at = torch.zeros(4, 2, 16), torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU tensor"):
        nn.segment_attention(q, q, q, at)
    with pytest.raises(ValueError, match="expected q"):
        nn.segment_attention(q[0], q, q, at)
    with pytest.raises(ValueError, match="expected q"):
        nn.segment_attention(q, q, q[:3], at)
    with pytest.raises(ValueError, match="GPU tensor"):
        nn.norm_rotary(q, q, None, None, torch.zeros(4, 1, dtype=torch.int32), torch.zeros(8), (8,))
    with pytest.raises(ValueError, match="expected q"):
        nn.norm_rotary(q, q[:2], None, None, torch.zeros(4, 1, dtype=torch.int32), torch.zeros(8), (8,))
    with pytest.raises(ValueError):
        nn.VoxelAttention(64, 5)
    with pytest.raises(ValueError):
        nn.VoxelAttention(64, 4, kv_heads=3)


# (a pointer that no kernel may see: every call below is refused)
P = ctypes.c_void_p(4096)
ODD = ctypes.c_void_p(4098)
NULL = ctypes.c_void_p()


def attention(**change):
    a = dict(q=P, k=P, v=P, out=P, lse=P, q_offsets=P, k_offsets=P, k_lengths=NULL, n_q=4, n_k=4, segments=1, heads=4, kv_heads=2, dim=16,
             q_row=64, q_head=16, k_row=32, k_head=16, v_row=32, v_head=16, causal=0, scale=0.25, dtype=1, stream=NULL)
    a.update(change)
    return a


def call_forward(**change):
    from fgms_amd import capi
    return capi.lib().fgms_segment_attention_fwd(*attention(**change).values()), capi.lib().fgms_last_error().decode()


def call_backward(**change):
    from fgms_amd import capi
    grads = {n: change.pop(n, P) for n in ("g", "gq", "gk", "gv")}
    a = attention(**change)
    a.pop("k_lengths")
    head = [grads["g"]] + [a.pop(n) for n in ("q", "k", "v", "out", "lse")] + [grads[n] for n in ("gq", "gk", "gv")]
    return capi.lib().fgms_segment_attention_bwd(*head, *a.values()), capi.lib().fgms_last_error().decode()


@pytest.mark.parametrize("change", [
    dict(dtype=3), dict(dtype=-1), dict(dim=0), dict(dim=12), dict(dim=136), dict(heads=0), dict(kv_heads=0), dict(kv_heads=3), dict(n_q=-1),
    dict(n_k=1 << 31), dict(segments=-1), dict(q_offsets=NULL), dict(k_offsets=NULL), dict(scale=0.0), dict(scale=-1.0), dict(scale=math.nan),
    dict(scale=math.inf), dict(q=NULL), dict(k=ODD), dict(v=NULL), dict(q_row=4), dict(k_head=-16), dict(v_row=33), dict(out=NULL), dict(out=ODD),
], ids=str)
def test_attention_refuses(change):
    for call in (call_forward, call_backward):
        rc, message = call(**change)
        assert rc == -1 and "fgms_segment_attention" in message, (rc, message)


def test_backward_refuses():
    for change in (dict(g=NULL), dict(lse=NULL), dict(g=ODD), dict(gk=ODD)):
        assert call_backward(**change)[0] == -1


def turn(backward, **change):
    from fgms_amd import capi
    a = dict(q=P, k=P, qs=P, ks=P, coords=P, freqs=P, qo=P, ko=P, n=4, h=2, hk=1, dim=16, q_row=32, q_head=16, k_row=16, k_head=16, axes=2,
             sections=(ctypes.c_int * 4)(4, 4, 0, 0), interleaved=0, eps=1e-6, dtype=1, stream=NULL)
    a.update(change)
    if not backward:
        return capi.lib().fgms_norm_rotary_fwd(*a.values())
    qo, ko = a.pop("qo"), a.pop("ko")
    first = [a.pop(n) for n in ("q", "k", "qs", "ks", "coords", "freqs")]
    return capi.lib().fgms_norm_rotary_bwd(qo, ko, *first, P, P, P, P, *a.values())


@pytest.mark.parametrize("change", [
    dict(dtype=7), dict(dim=20), dict(dim=256), dict(h=0), dict(hk=-1), dict(n=-1), dict(axes=0), dict(axes=5), dict(eps=-1.0), dict(eps=math.nan),
    dict(sections=(ctypes.c_int * 4)(-1, 4, 0, 0)), dict(sections=(ctypes.c_int * 4)(5, 4, 0, 0)), dict(sections=None), dict(coords=NULL),
    dict(freqs=NULL), dict(q=NULL), dict(q=ODD), dict(k=NULL), dict(qs=ODD), dict(q_row=31), dict(k_head=-8), dict(qo=NULL), dict(ko=ODD),
], ids=lambda c: next(iter(c)))
def test_norm_rotary_refuses(change):
    from fgms_amd import capi
    for backward in (False, True):
        assert turn(backward, **change) == -1
        assert "fgms_norm_rotary" in capi.lib().fgms_last_error().decode()


def test_nothing_to_do_is_no_error():
    assert call_forward(n_q=0, q=NULL, out=NULL)[0] == 0
    assert turn(False, n=0, q=NULL, k=NULL, coords=NULL) == 0

"""The ctypes entries of attention check every tensor's size before a kernel can write past it."""
import pytest
import torch


class OnTheCard(torch.Tensor):
    """A tensor that says it is on the GPU (no call below reaches the library)."""

    @property
    def is_cuda(self):
        return True


def tensor(*shape, dtype=torch.float16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(OnTheCard)


@pytest.fixture(autouse=True)
def no_library(monkeypatch):
    from fgms_amd import capi

    def refuse():
        raise AssertionError("the library was called")

    monkeypatch.setattr(capi, "lib", refuse)
    monkeypatch.setattr(capi, "_stream", lambda: None)


def attend(backward, **change):
    from fgms_amd import capi
    f, i = torch.float32, torch.int32
    a = dict(q=tensor(6, 4, 16), k=tensor(5, 2, 16), v=tensor(5, 2, 16), out=tensor(6, 4, 16), lse=tensor(6, 4, dtype=f), q_offsets=tensor(3, dtype=i),
             k_offsets=tensor(3, dtype=i))
    if backward:
        a.update(out_grad=tensor(6, 4, 16), q_grad=tensor(6, 4, 16), k_grad=tensor(5, 2, 16), v_grad=tensor(5, 2, 16))
    else:
        a.update(k_lengths=tensor(2, dtype=i))
    a.update(change)
    (capi.segment_attention_bwd if backward else capi.segment_attention_fwd)(**a)


@pytest.mark.parametrize("change", [dict(out=(5, 4, 16)), dict(out=(6, 2, 16)), dict(lse=(6, 3)), dict(lse=(6,)), dict(k_offsets=(4,)), dict(v=(4, 2, 16)),
                                    dict(k=(5, 2, 8), v=(5, 2, 8)), dict(k_lengths=(1,)), dict(out_grad=(6, 4, 8)), dict(q_grad=(5, 4, 16)),
                                    dict(k_grad=(5, 1, 16)), dict(v_grad=(6, 2, 16))], ids=str)
def test_attention(change):
    types = dict(lse=torch.float32, k_offsets=torch.int32, k_lengths=torch.int32)
    change = {n: tensor(*s, dtype=types.get(n, torch.float16)) for n, s in change.items()}
    for backward in (False, True):
        if any(n.endswith("grad") for n in change) and not backward or "k_lengths" in change and backward:
            continue
        with pytest.raises(ValueError):
            attend(backward, **change)
    with pytest.raises(AssertionError, match="library"):
        attend(False)
    with pytest.raises(AssertionError, match="library"):
        attend(True)


def turn(backward, **change):
    from fgms_amd import capi
    f, i = torch.float32, torch.int32
    a = dict(q=tensor(6, 4, 16), k=tensor(6, 2, 16), q_scale=tensor(16), k_scale=tensor(16), coords=tensor(6, 2, dtype=i), freqs=tensor(6, dtype=f),
             sections=(4, 2))
    if backward:
        a.update(q_out_grad=tensor(6, 4, 16), k_out_grad=tensor(6, 2, 16), q_grad=tensor(6, 4, 16), k_grad=tensor(6, 2, 16), q_scale_grad=tensor(16),
                 k_scale_grad=tensor(16))
    else:
        a.update(q_out=tensor(6, 4, 16), k_out=tensor(6, 2, 16))
    a.update(change)
    (capi.norm_rotary_bwd if backward else capi.norm_rotary_fwd)(**a)


BOTH = [dict(q_scale=(8,)), dict(k_scale=(2, 8)), dict(coords=(5, 2)), dict(freqs=(5,))]
FORWARD = [dict(q_out=(5, 4, 16)), dict(k_out=(6, 4, 8))]
BACKWARD = [dict(q_out_grad=(6, 4, 8)), dict(k_out_grad=(5, 2, 16)), dict(q_grad=(6, 2, 16)), dict(k_grad=(6, 1, 16)), dict(q_scale_grad=(8,)),
            dict(k_scale_grad=(15,))]


@pytest.mark.parametrize("backward, change", [(False, c) for c in BOTH + FORWARD] + [(True, c) for c in BOTH + BACKWARD], ids=str)
def test_norm_rotary(backward, change):
    types = dict(coords=torch.int32, freqs=torch.float32)
    with pytest.raises(ValueError):
        turn(backward, **{n: tensor(*s, dtype=types.get(n, torch.float16)) for n, s in change.items()})
    with pytest.raises(AssertionError, match="library"):
        turn(backward)

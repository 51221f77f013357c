"""The cache of the attention layer takes rows, not their gradients, and a step that is refused leaves it as it was."""
import pytest
import torch


def test_append_keeps_the_cache_out_of_the_graph():
    from FGMS import nn
    cache = nn.VoxelCache(2, 3, 1, 8)
    k, v = torch.randn(2, 1, 8, requires_grad=True), torch.randn(2, 1, 8, requires_grad=True)
    cache.append(k * 2, v * 2)
    assert not cache.k.requires_grad and not cache.v.requires_grad
    assert cache.lengths.tolist() == [1, 1] and torch.equal(cache.k[::3], k.detach() * 2) and torch.equal(cache.v[::3], v.detach() * 2)


@pytest.mark.parametrize("what", ["layer", "feats"])
def test_refused_steps_leave_the_cache(what):
    from FGMS import nn
    layer, cache = nn.VoxelAttention(32, 2), nn.VoxelCache(2, 3, 2, 16)
    layer.requires_grad_(what != "feats")
    feats, coords = torch.randn(2, 32, requires_grad=what == "feats"), torch.zeros(2, 3, dtype=torch.int32)
    for _ in range(2):
        with pytest.raises(ValueError, match="no_grad"):
            layer.step(feats, coords, cache)
    assert cache.lengths.tolist() == [0, 0] and not cache.k.any() and not cache.v.any()
    assert not cache.k.requires_grad


@pytest.mark.gpu
def test_steps_after_a_refusal():
    from FGMS import nn
    torch.manual_seed(0)
    layer = nn.VoxelAttention(32, 2, causal=True, device="cuda")
    caches = [nn.VoxelCache(2, 4, 2, 16, device="cuda") for _ in range(2)]
    for i in range(3):
        feats, coords = torch.randn(2, 32, device="cuda"), torch.randint(0, 9, (2, 3), dtype=torch.int32, device="cuda")
        with pytest.raises(ValueError, match="no_grad"):
            layer.step(feats, coords, caches[0])
        with torch.no_grad():
            assert torch.equal(layer.step(feats, coords, caches[0]), layer.step(feats, coords, caches[1]))
        assert caches[0].lengths.tolist() == [i + 1] * 2
    # a layer without gradients needs no context
    layer.requires_grad_(False)
    assert torch.isfinite(layer.step(feats, coords, caches[0])).all()

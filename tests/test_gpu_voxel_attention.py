"""The attention layer over voxel clouds (FGMS.nn.VoxelAttention) next to sparse convolutions: training, rows one at a time over
a cache, windows, and what both operators give when a small network uses them together."""
import math

import numpy as np
import pytest
import torch

from fgms_amd import clouds
from tests import attention_util as U

pytestmark = pytest.mark.gpu


def small_cloud(seed, size=24):
    rng = np.random.default_rng(seed)
    pts = np.concatenate([clouds._patch(rng, rng.uniform(6, 18, 3), 9, 9, oblique=False),
                          clouds._sphere_shell(rng, np.array([12., 12, 12]), 7.0, 2500)])
    return torch.from_numpy(clouds.dedup(pts, size)).cuda()


@pytest.mark.parametrize("size", [4, (8, 8, 3)], ids=str)
def test_windows(size):
    from FGMS import nn
    coords = small_cloud(0) - 11      # cells on both sides of zero
    order, offsets = nn.window_segments(coords, size)
    assert sorted(order.tolist()) == list(range(len(coords)))
    cells = torch.div(coords[order].cpu(), torch.as_tensor(size), rounding_mode="floor")
    at = offsets.tolist()
    assert at[0] == 0 and at[-1] == len(coords) and offsets.dtype == torch.int32
    seen = set()
    for a, b in zip(at, at[1:]):
        assert b > a and len({tuple(c) for c in cells[a:b].tolist()}) == 1
        seen.add(tuple(cells[a].tolist()))
        assert (order[a:b][1:] > order[a:b][:-1]).all()      # rows of a window in the cloud's order
    assert len(seen) == len(at) - 1


def test_network_trains():
    """A sparse convolution, attention in windows and another convolution, as one network."""
    from FGMS import nn
    torch.manual_seed(0)
    coords = small_cloud(1)
    order, offsets = nn.window_segments(coords, 6)
    coords = coords[order].contiguous()
    kmap = nn.KernelMap.from_coords(coords, coords, clouds.offsets_cube(3))
    first = nn.SparseConv(8, 32, 27, device="cuda")
    mix = nn.VoxelAttention(32, 4, kv_heads=2, sections=(2, 1, 1), device="cuda")
    last = nn.SparseConv(32, 8, 27, device="cuda")
    params = [p for m in (first, mix, last) for p in m.parameters()]
    opt = torch.optim.Adam(params, lr=0.01)
    x, target = torch.randn(len(coords), 8, device="cuda"), torch.randn(len(coords), 8, device="cuda")
    losses = []
    for _ in range(12):
        opt.zero_grad()
        y = first(x, kmap)
        y = y + mix(y, coords, offsets)
        loss = ((last(torch.relu(y), kmap) - target) ** 2).mean()
        loss.backward()
        assert all(p.grad is not None and torch.isfinite(p.grad).all() for p in params)
        opt.step()
        losses.append(float(loss.detach()))
    assert losses[-1] < losses[0]


@pytest.mark.parametrize("dtype", list(U.DTYPES))
def test_layer_is_its_formula(dtype):
    from FGMS import nn
    torch.manual_seed(2)
    t = U.DTYPES[dtype]
    layer = nn.VoxelAttention(64, 4, kv_heads=2, sections=(3, 3, 2), causal=True, dtype=t, device="cuda")
    lengths = [33, 70, 1]
    coords = torch.randint(0, 100, (104, 3), dtype=torch.int32, device="cuda")
    feats = torch.randn(104, 64, device="cuda").to(t)
    with torch.no_grad():
        got = layer(feats, coords, U.offsets(lengths))
        qkv = layer.qkv(feats)
        q, k, v = (s.unflatten(1, (-1, 16)) for s in qkv.split((64, 32, 32), 1))
        q64, _ = U.turned(q, layer.q_scale, coords, layer._freqs, layer.sections, 1e-6, False)
        k64, _ = U.turned(k, layer.k_scale, coords, layer._freqs, layer.sections, 1e-6, False)
        want = U.attention(q64.to(t), k64.to(t), v, lengths, lengths, True, 0.25)
        # the same projection of the plain result: a product of 64 channels, its inputs off by their own bounds and by the
        # rounding of q and k, which may fall the other way (a step each of scores of order one)
        ref = want.out.flatten(1) @ layer.out.weight.cpu().double().T
        step = U.UNIT[t]
        off = (want.out_off.flatten(1) + 16 * step * want.out.flatten(1).abs() + 16 * step) @ layer.out.weight.cpu().double().abs().T + 2 * step * ref.abs() + 1e-6
    U.within(got, ref, off, "layer")


def test_row_by_row():
    """Rows one at a time over a cache are the causal layer over all of them: the same roundings of the same values, but the
    projections' sums in the order that their sizes bring, and the softmax sums in parts."""
    from FGMS import nn
    torch.manual_seed(3)
    scans, rows, channels = 3, 40, 64
    layer = nn.VoxelAttention(channels, 4, kv_heads=2, sections=(3, 3, 2), causal=True, device="cuda")
    feats = torch.randn(scans, rows, channels, device="cuda")
    coords = torch.randint(0, 50, (scans, rows, 3), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        whole = layer(feats.flatten(0, 1), coords.flatten(0, 1), U.offsets([rows] * scans)).unflatten(0, (scans, rows))
        cache = nn.VoxelCache(scans, 64, layer.kv_heads, layer.dim, device="cuda")
        for i in range(rows):
            y = layer.step(feats[:, i].contiguous(), coords[:, i].contiguous(), cache)
            # fp32 sums of 64 products, a softmax and another 64: a few hundred roundings of 2^-24 of values of order one
            assert float((y - whole[:, i]).abs().max()) < 512 * 2.0 ** -24, i
        assert cache.lengths.tolist() == [rows] * scans


def test_a_full_cache_replaces_its_last_row():
    from FGMS import nn
    cache = nn.VoxelCache(2, 3, 1, 8, device="cuda")
    for i in range(5):
        cache.append(torch.full((2, 1, 8), float(i), device="cuda"), torch.full((2, 1, 8), -float(i), device="cuda"))
    assert cache.lengths.tolist() == [3, 3]
    assert cache.k[:, 0, 0].tolist() == [0, 1, 4, 0, 1, 4] and cache.v[2, 0, 0] == -4


def test_cast_layers_keep_their_angles():
    from FGMS import nn
    layer = nn.VoxelAttention(32, 2).half().cuda()
    assert layer._freqs.dtype == torch.float32
    coords = torch.tensor([[1000, 3, 5]], dtype=torch.int32, device="cuda")
    with torch.no_grad():
        y = layer(torch.randn(1, 32, device="cuda").half(), coords, U.offsets([1]))
    assert y.dtype == torch.float16 and torch.isfinite(y).all()

"""Norms of queries and keys with their rotation by coordinates (FGMS.nn.norm_rotary), and its gradients, against the plain
formulas in 64 bits."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu

# rows, heads, key heads, channels, sections, interleaved
CASES = {
    "one": (1, 1, 1, 8, (4,), False),
    "space": (1000, 4, 4, 16, (3, 3, 2), False),
    "space-time": (257, 8, 2, 64, (8, 8, 8, 8), True),
    "some-pairs": (301, 5, 1, 72, (12, 0, 10), True),
    "halves-of-36": (301, 5, 1, 72, (20, 16), False),
    "widest": (130, 2, 1, 128, (30, 20, 14), False),
    "odd-heads": (99, 3, 3, 40, (7, 7, 6), True),
    "no-turn": (50, 2, 2, 24, (0, 0), False),
    "many-rows": (40000, 2, 1, 32, (6, 5, 5), False),
}


def inputs(case, dtype, seed=0, reach=500):
    n, h, hk, d, sections, _ = CASES[case]
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen).to(U.DTYPES[dtype])

    q, k, qs, ks = normal(n, h, d), normal(n, hk, d), 1 + normal(d) / 4, 1 + normal(d) / 4
    leaves = [t.cuda().requires_grad_() for t in (q, k, qs, ks)]
    coords = torch.randint(-reach, reach, (n, len(sections)), generator=gen, dtype=torch.int64).to(torch.int32).cuda()
    from FGMS import nn
    return leaves, coords, nn.rotary_freqs(sections, device="cuda"), normal(n, h, d).cuda(), normal(n, hk, d).cuda()


@pytest.mark.parametrize("dtype", list(U.DTYPES))
@pytest.mark.parametrize("case", list(CASES))
def test_both_passes(case, dtype):
    from FGMS import nn
    sections, interleaved = CASES[case][4:]
    (q, k, qs, ks), coords, freqs, gq, gk = inputs(case, dtype)
    out = nn.norm_rotary(q, k, qs, ks, coords, freqs, sections, interleaved=interleaved)
    got = torch.autograd.grad(out, (q, k, qs, ks), (gq, gk), retain_graph=True)
    for i, (x, w, g) in enumerate(((q, qs, gq), (k, ks, gk))):
        y, y_off, gx, gx_off, gw, gw_off = U.turned(x, w, coords, freqs, sections, 1e-6, interleaved, g)
        U.within(out[i], y, y_off, "qk"[i])
        U.within(got[i], gx, gx_off, "gradient of " + "qk"[i])
        U.within(got[2 + i], gw, gw_off, "gradient of a scale")
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(out, (q, k, qs, ks), (gq, gk), retain_graph=True)))
    # a gradient on its own, and one output's alone
    assert torch.equal(torch.autograd.grad(out, ks, (gq, gk), retain_graph=True)[0], got[3])
    assert torch.equal(torch.autograd.grad(out[0], q, gq, retain_graph=True)[0], got[0])
    # no scales: ones
    ones = torch.ones_like(qs)
    bare = nn.norm_rotary(q, k, None, None, coords, freqs, sections, interleaved=interleaved)
    assert all(torch.equal(a, b) for a, b in zip(bare, nn.norm_rotary(q, k, ones, ones, coords, freqs, sections, interleaved=interleaved)))
    assert torch.equal(torch.autograd.grad(bare, k, (gq, gk))[0],
                       torch.autograd.grad(nn.norm_rotary(q, k, ones, ones, coords, freqs, sections, interleaved=interleaved), k, (gq, gk))[0])


def test_far_coordinates():
    """Any 32-bit coordinate: the angle keeps its fraction of a turn."""
    from FGMS import nn
    (q, k, qs, ks), _, freqs, _, _ = inputs("space-time", "fp32", 1)
    sections = CASES["space-time"][4]
    for reach in (1 << 20, (1 << 31) - 1):
        coords = torch.randint(-reach, reach, (q.shape[0], 4)).to(torch.int32).cuda()
        coords[0] = -(1 << 31) if reach > 1 << 30 else reach
        out = nn.norm_rotary(q, k, qs, ks, coords, freqs, sections)
        y, y_off = U.turned(q, qs, coords, freqs, sections, 1e-6, False)
        U.within(out[0], y, y_off, "far")


def test_gradients_against_differences():
    """Central differences of the fp32 kernel in steps of 2^-7; a row of d channels of order one has third derivatives of
    order one along a direction of order one, of which a sixth of the step squared is left."""
    from FGMS import nn
    sections, interleaved = CASES["odd-heads"][4:]
    leaves, coords, freqs, gq, gk = inputs("odd-heads", "fp32", 2)
    out = nn.norm_rotary(*leaves, coords, freqs, sections, interleaved=interleaved)
    grads = torch.autograd.grad(out, leaves, (gq, gk))
    gen = torch.Generator().manual_seed(3)
    step = 2.0 ** -7
    for i, grad in enumerate(grads):
        along = torch.randn(grad.shape, generator=gen).cuda()
        value = []
        for sign in (1, -1):
            x = [t.detach() for t in leaves]
            x[i] = x[i] + sign * step * along
            a, b = nn.norm_rotary(*x, coords, freqs, sections, interleaved=interleaved)
            value.append((a.double() * gq.double()).sum() + (b.double() * gk.double()).sum())
        change, want = float((value[0] - value[1]) / (2 * step)), float((grad.double() * along.double()).sum())
        size = float((grad.double() * along.double()).norm())
        assert abs(change - want) <= 32 * step ** 2 * size + 1e-3 * size, (i, change, want, size)


def test_layouts_and_zero_rows():
    from FGMS import nn
    torch.manual_seed(4)
    n, h, hk, d, sections = 77, 4, 2, 48, (10, 10)
    coords = torch.randint(0, 100, (n, 2), dtype=torch.int32, device="cuda")
    freqs = nn.rotary_freqs(sections, device="cuda")
    for dtype in U.DTYPES.values():
        qkv = torch.randn(n, (h + 2 * hk) * d, device="cuda").to(dtype)
        qkv[5] = 0      # a row of zeros: its norm is that of eps
        q, k, _ = (t.unflatten(1, (-1, d)) for t in qkv.split((h * d, hk * d, hk * d), 1))
        scale = torch.randn(d, device="cuda").to(dtype)
        gq, gk = torch.randn_like(q.contiguous()), torch.randn_like(k.contiguous())

        def run(q, k, gq):
            x = [t.detach().requires_grad_() for t in (q, k, scale)]
            out = nn.norm_rotary(x[0], x[1], x[2], x[2], coords, freqs, sections)
            return (*out, *torch.autograd.grad(out, x, (gq, gk)))

        plain = run(q.contiguous(), k.contiguous(), gq)
        assert torch.isfinite(plain[2]).all() and not plain[0][5].any()
        loose = torch.zeros(n, h, d + 1, dtype=dtype, device="cuda")[..., 1:]
        loose.copy_(q)
        for other in ((q, k, gq), (loose, k, gq), (q, k.transpose(0, 1).contiguous().transpose(0, 1), gq.transpose(0, 1).contiguous().transpose(0, 1))):
            assert all(torch.equal(a, b) for a, b in zip(plain, run(*other)))
        x = [t[:0].detach().requires_grad_() for t in (q, k)] + [scale.clone().requires_grad_()]
        out = nn.norm_rotary(x[0], x[1], x[2], None, coords[:0], freqs, sections)
        assert out[0].shape == (0, h, d) and not torch.autograd.grad(out, x, (gq[:0], gk[:0]))[2].any()


def test_streams_and_graphs():
    from FGMS import nn
    sections = CASES["space"][4]
    leaves, coords, freqs, gq, gk = inputs("space", "fp16", 5)

    def step():
        out = nn.norm_rotary(*leaves, coords, freqs, sections)
        return tuple(t.detach() for t in out) + torch.autograd.grad(out, leaves, (gq, gk))

    want = step()
    side = U.own_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        kept = step()
    for shift in (0, 7, -100):
        coords.add_(shift)
        eager = step()
        for t in kept:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, kept))

"""Attention inside ragged segments and its gradients (FGMS.nn.segment_attention) against the plain formulas in 64 bits."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu

# queries of each segment, keys of each, heads, key heads, channels, causal
CASES = {
    "one": ([1], [1], 1, 1, 8, False),
    "cross-empty": ([5, 0, 33, 0], [7, 4, 0, 0], 6, 2, 40, False),
    "causal": ([130, 1, 64, 31], [130, 1, 64, 31], 4, 4, 64, True),
    "causal-rows-without-keys": ([50, 3, 90], [20, 9, 70], 2, 2, 32, True),
    "wide-group": ([300], [300], 8, 2, 128, False),
    "windows": ([1 + i * 7 % 20 for i in range(100)], [1 + i * 7 % 20 for i in range(100)], 3, 1, 16, False),
    "tokens": ([1] * 5, [1000, 3, 0, 257, 64], 8, 2, 128, True),
    "long-cache": ([1, 2], [5000, 3111], 4, 2, 64, True),
    "few-keys": ([4000, 17], [3, 40], 2, 2, 24, False),
    "group-of-three": ([100, 77], [100, 77], 6, 2, 96, True),
    "more-keys": ([40, 5], [700, 64], 3, 3, 72, True),
    "odd-group": ([37, 129], [45, 130], 5, 1, 112, True),
    "long-rows": ([2100], [2100], 1, 1, 48, True),
}


def inputs(case, dtype, seed=0, grad=True):
    ql, kl, h, hk, d, causal = CASES[case]
    gen = torch.Generator().manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen).to(U.DTYPES[dtype]).cuda()

    q, k, v, g = normal(sum(ql), h, d), normal(sum(kl), hk, d), normal(sum(kl), hk, d), normal(sum(ql), h, d)
    return tuple(t.requires_grad_(grad) for t in (q, k, v)) + (g, U.offsets(ql), U.offsets(kl))


@pytest.mark.parametrize("dtype", list(U.DTYPES))
@pytest.mark.parametrize("case", list(CASES))
def test_both_passes(case, dtype):
    from FGMS import nn
    ql, kl, h, hk, d, causal = CASES[case]
    q, k, v, g, qo, ko = inputs(case, dtype)
    out = nn.segment_attention(q, k, v, qo, ko, causal=causal)
    want = U.attention(q, k, v, ql, kl, causal, 1 / math.sqrt(d), g)
    U.within(out, want.out, want.out_off, "out")
    with torch.no_grad():
        assert torch.equal(nn.segment_attention(q, k, v, qo, ko, causal=causal), out)
    got = torch.autograd.grad(out, (q, k, v), g, retain_graph=True)
    for name, t in zip(("gq", "gk", "gv"), got):
        U.within(t, getattr(want, name), getattr(want, name + "_off"), name)
    again = torch.autograd.grad(out, (q, k, v), g, retain_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(got, again))      # no order of sums is left to chance
    # one gradient at a time is the same gradient
    for i, t in enumerate((q, k, v)):
        assert torch.equal(torch.autograd.grad(out, t, g, retain_graph=True)[0], got[i])


@pytest.mark.parametrize("dtype", list(U.DTYPES))
@pytest.mark.parametrize("case", ["causal-rows-without-keys", "tokens", "long-cache"])
def test_log_sums(case, dtype):
    from fgms_amd import capi
    ql, kl, h, hk, d, causal = CASES[case]
    q, k, v, _, qo, ko = inputs(case, dtype, 1, False)
    out, lse = torch.empty_like(q), torch.empty(q.shape[:2], device="cuda")
    capi.segment_attention_fwd(q, k, v, out, lse, qo, ko, causal=causal, scale=0.3)
    want = U.attention(q, k, v, ql, kl, causal, 0.3)
    none = want.lse == -math.inf
    assert torch.equal(lse.cpu() == -math.inf, none)
    assert torch.equal(out.cpu()[none], torch.zeros_like(out.cpu()[none]))
    U.within(lse.cpu()[~none], want.lse[~none], want.lse_off[~none] + 2.0 ** -22, "lse")
    U.within(out, want.out, want.out_off, "out")


def test_gradients_against_differences():
    """Central differences of the fp32 kernel's own results, in steps of 2^-6: their error is a sixth of the step squared
    times a third derivative (bounded by the sums of sizes below, scores being of order one) and the results' rounding."""
    from FGMS import nn
    ql, kl, h, hk, d, causal = CASES["group-of-three"]
    q, k, v, g, qo, ko = inputs("group-of-three", "fp32", 2)
    out = nn.segment_attention(q, k, v, qo, ko, causal=causal)
    grads = torch.autograd.grad(out, (q, k, v), g)
    gen = torch.Generator().manual_seed(3)
    step = 2.0 ** -6
    for i, grad in enumerate(grads):
        for _ in range(3):
            along = torch.randn(grad.shape, generator=gen).cuda()
            value = []
            for sign in (1, -1):
                x = [q.detach(), k.detach(), v.detach()]
                x[i] = x[i] + sign * step * along
                value.append((nn.segment_attention(*x, qo, ko, causal=causal).double() * g.double()).sum())
            change = float((value[0] - value[1]) / (2 * step))
            want = float((grad.double() * along.double()).sum())
            size = float((grad.double() * along.double()).norm())
            assert abs(change - want) <= step ** 2 * 4 * size * math.sqrt(d) + 1e-4 * size, (i, change, want, size)


def test_layouts():
    """Slices of one projection, expanded key heads, transposed and unaligned tensors give what contiguous copies give."""
    from FGMS import nn
    torch.manual_seed(4)
    lengths, h, hk, d = [70, 33, 5], 4, 2, 32
    n, at = sum(lengths), U.offsets([70, 33, 5])
    for dtype in U.DTYPES.values():
        qkv = torch.randn(n, (h + 2 * hk) * d, device="cuda").to(dtype)
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((h * d, hk * d, hk * d), 1))
        g = torch.randn(n, h, d, device="cuda").to(dtype)

        def run(q, k, v, g):
            x = [t.detach().requires_grad_() for t in (q, k, v)]
            out = nn.segment_attention(*x, at, causal=True)
            return (out, *torch.autograd.grad(out, x, g))

        plain = run(q.contiguous(), k.contiguous(), v.contiguous(), g)
        loose = torch.zeros(n, h, d + 1, dtype=dtype, device="cuda")[..., 1:]
        loose.copy_(q)
        by_head = q.transpose(0, 1).contiguous().transpose(0, 1)
        odd_g = torch.zeros(n * h * d + 1, dtype=dtype, device="cuda")[1:].view(n, h, d)
        odd_g.copy_(g)
        for other in ((q, k, v, g), (loose, k, v, g), (by_head, k, v, g.transpose(0, 1).contiguous().transpose(0, 1)), (q, k, v, odd_g)):
            assert all(torch.equal(a, b) for a, b in zip(plain, run(*other)))
        # one key head for all, by expansion or by grouping
        k1, v1 = k[:, :1], v[:, :1]
        wide = run(q, k1.expand(-1, h, -1), v1.expand(-1, h, -1), g)
        grouped = run(q, k1, v1, g)
        want = U.attention(q, k1, v1, lengths, lengths, True, 1 / math.sqrt(d), g)
        U.within(grouped[2], want.gk, want.gk_off, "grouped gk")
        U.within(wide[0], want.out, want.out_off, "expanded out")
        kx = k1.detach().requires_grad_()
        out = nn.segment_attention(q.detach(), kx.expand(-1, h, -1), v1.expand(-1, h, -1), at, causal=True)
        # (torch adds the heads' gradients up, each rounded once, in the type)
        summed = torch.autograd.grad(out, kx, g)[0]
        U.within(summed, want.gk, 2 * h * want.gk_off + 2 * h * U.UNIT[dtype] * wide[2].detach().cpu().double().abs().sum(1, keepdim=True), "expanded gk")


def test_caches():
    """Only the rows in use are keys: what lies behind them may be anything; lengths past the room or below zero are cut."""
    from FGMS import nn
    torch.manual_seed(5)
    used, room, h, hk, d = [100, 0, 257, 64], 300, 8, 2, 64
    for dtype in U.DTYPES.values():
        q = torch.randn(len(used), h, d, device="cuda").to(dtype)
        k = torch.full((len(used) * room, hk, d), math.nan, device="cuda", dtype=dtype)
        v = torch.full_like(k, math.inf)
        parts = []
        for s, n in enumerate(used):
            parts.append((torch.randn(n, hk, d, device="cuda").to(dtype), torch.randn(n, hk, d, device="cuda").to(dtype)))
            k[s * room:s * room + n], v[s * room:s * room + n] = parts[-1]
        at = torch.arange(len(used) + 1, dtype=torch.int32, device="cuda")
        lengths = torch.tensor(used, dtype=torch.int32, device="cuda")
        out = nn.segment_attention(q, k, v, at, at * room, causal=True, k_lengths=lengths)
        want = U.attention(q, torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]), [1] * len(used), used, True, 1 / math.sqrt(d))
        U.within(out, want.out, want.out_off, "cache")
        lengths[1] = -5
        assert torch.equal(out, nn.segment_attention(q, k, v, at, at * room, causal=True, k_lengths=lengths))
        k[3 * room:], v[3 * room:] = 1.0, 2.0
        lengths[3] = 1 << 30
        assert torch.isfinite(nn.segment_attention(q, k, v, at, at * room, k_lengths=lengths)).all()


def test_what_is_not_seen_does_not_matter():
    """Infinite and NaN keys behind a query and in other segments; huge scores; rows behind the last segment."""
    from FGMS import nn
    torch.manual_seed(6)
    d = 32
    for dtype in U.DTYPES.values():
        q, k, v, g = (torch.randn(200, 2, d, device="cuda").to(dtype) for _ in range(4))
        at = U.offsets([90, 70])      # 40 rows in no segment
        x = [t.clone().requires_grad_() for t in (q, k, v)]
        out = nn.segment_attention(*x, at, causal=True)
        grads = torch.autograd.grad(out, x, g)
        assert torch.equal(out[160:], torch.zeros_like(out[160:]))
        assert all(torch.equal(t[160:], torch.zeros_like(t[160:])) for t in grads)
        want = U.attention(q[:160], k[:160], v[:160], [90, 70], [90, 70], True, 1 / math.sqrt(d), g[:160])
        U.within(out[:160], want.out, want.out_off, "out")
        U.within(grads[1][:160], want.gk, want.gk_off, "gk")
        # keys that only the first segment's last rows see; values of the second segment
        k2, v2 = k.clone(), v.clone()
        k2[80:90] = math.nan
        k2[85] = math.inf
        v2[90:] = math.nan
        k2[90:] = -math.inf
        spoiled = nn.segment_attention(q, k2, v2, at, causal=True)
        assert torch.equal(spoiled[:80], out[:80].detach())
        assert torch.isnan(spoiled[80:90]).all()
        # scores of tens of thousands: probabilities of zero and one
        big = nn.segment_attention(q * 60, k * 60, v, at, causal=True)
        far = U.attention(q * 60, k * 60, v, [90, 70, 40], [90, 70, 0], True, 1 / math.sqrt(d))
        sure = far.out_off < 0.05
        assert float(sure.double().mean()) > 0.5
        U.within(big.cpu()[sure], far.out[sure], far.out_off[sure], "huge scores")


def test_small_gradients_keep_their_bits():
    """fp16: rows of thousands of like keys have probabilities at fp16's lower end, and ds below it."""
    from FGMS import nn
    torch.manual_seed(7)
    n, d = 3000, 16
    q, k, v = (torch.randn(n, 1, d, device="cuda").half() * s for s in (0.1, 0.1, 1.0))
    g = (torch.randn(n, 1, d, device="cuda") * 0.02).half()
    x = [t.requires_grad_() for t in (q, k, v)]
    out = nn.segment_attention(*x, U.offsets([n]))
    got = torch.autograd.grad(out, x, g)
    want = U.attention(q, k, v, [n], [n], False, 0.25, g)
    for name, t in zip(("gq", "gk", "gv"), got):
        U.within(t, getattr(want, name), getattr(want, name + "_off"), name)
        ref = getattr(want, name)
        rel = float((t.cpu().double() - ref).norm() / ref.norm())
        assert rel < 0.02, (name, rel)


def test_far_offsets():
    """Rows whose addresses pass 2^31 elements and 2^32 bytes."""
    from FGMS import nn
    torch.manual_seed(8)
    h, d, far, n = 8, 128, 2_200_000, 333
    k = torch.empty(far + n, h, d, dtype=torch.float16, device="cuda")
    v = torch.empty_like(k)
    k[far:].normal_()
    v[far:].normal_()
    q = torch.randn(3, h, d, device="cuda").half()
    ko = torch.tensor([0, far, far + n], dtype=torch.int32, device="cuda")
    out = nn.segment_attention(q, k, v, torch.tensor([0, 0, 3], dtype=torch.int32, device="cuda"), ko, causal=True)
    want = U.attention(q, k[far:], v[far:], [3], [n], True, 1 / math.sqrt(d))
    U.within(out, want.out, want.out_off, "far keys")
    del v
    out = nn.segment_attention(k, q[:, :8], q[:, :8], ko, torch.tensor([0, 0, 3], dtype=torch.int32, device="cuda"))
    want = U.attention(k[far:], q, q, [n], [3], False, 1 / math.sqrt(d))
    U.within(out[far:], want.out, want.out_off, "far queries")
    assert not out[:far].any()


def test_streams_and_graphs():
    from FGMS import nn
    q, k, v, g, qo, ko = inputs("long-cache", "fp16", 9)

    def step():
        out = nn.segment_attention(q, k, v, qo, ko, causal=True)
        return (out.detach(),) + torch.autograd.grad(out, (q, k, v), g)

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
    for scale in (1.0, 0.5, 2.0):
        with torch.no_grad():
            v.copy_(v * scale)
        eager = step()
        for t in kept:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, kept))


def test_saved_tensors_and_tangents():
    import torch.autograd.forward_ad as fwd
    from FGMS import nn
    q, k, v, g, qo, ko = inputs("wide-group", "fp16", 10)
    want = torch.autograd.grad(nn.segment_attention(q, k, v, qo, ko), (q, k, v), g)
    with torch.autograd.graph.save_on_cpu():
        out = nn.segment_attention(q, k, v, qo, ko)
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(out, (q, k, v), g)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()):
        out = nn.segment_attention(q, k, v, qo, ko)
    with pytest.raises(ValueError):
        torch.autograd.grad(out, q, g)
    with fwd.dual_level(), pytest.raises(NotImplementedError):
        nn.segment_attention(fwd.make_dual(q.detach(), g), k, v, qo, ko)
    traced = torch.jit.trace(lambda a, b, c: nn.segment_attention(a, b, c, qo, ko), (q.detach(), k.detach(), v.detach()), check_trace=False)
    assert torch.equal(traced(k.detach().repeat(1, 4, 1), k.detach(), v.detach()),
                       nn.segment_attention(k.detach().repeat(1, 4, 1), k.detach(), v.detach(), qo, ko))


def test_empty_sizes():
    from FGMS import nn
    for dtype in U.DTYPES.values():
        q, k = torch.randn(4, 2, 16, device="cuda").to(dtype), torch.randn(0, 2, 16, device="cuda").to(dtype)
        for lengths in ([], [4], [1, 3]):
            x = [t.clone().requires_grad_() for t in (q, k, k)]
            out = nn.segment_attention(*x, U.offsets(lengths), U.offsets([0] * len(lengths)))
            assert not out.any()
            assert not any(t.any() for t in torch.autograd.grad(out, x, q))
            x = [t.clone().requires_grad_() for t in (k, q, q)]
            out = nn.segment_attention(*x, U.offsets([0] * len(lengths)), U.offsets(lengths))
            assert out.shape == (0, 2, 16)
            assert not any(t.any() for t in torch.autograd.grad(out, x, k))


def test_layouts_that_are_copied():
    """Keys expanded over rows, rows that overlap, and heads too far apart for a tile's offsets give what copies of them give."""
    from FGMS import nn
    torch.manual_seed(11)
    at, d = U.offsets([50, 30]), 32
    q, v = torch.randn(80, 4, d, device="cuda").half(), torch.randn(80, 2, d, device="cuda").half()
    same = torch.randn(1, 2, d, device="cuda").half().expand(80, -1, -1)
    sliding = torch.randn(80 * 16 + 64, device="cuda").half().as_strided((80, 2, d), (16, 32, 1))
    for k in (same, sliding):
        for x in ((q, k, v), (q, v, k)):
            want = U.attention(*x, [50, 30], [50, 30], True, 1 / math.sqrt(d), q)
            leaves = [t.detach().requires_grad_() for t in x]
            out = nn.segment_attention(*leaves, at, causal=True)
            U.within(out, want.out, want.out_off, "out")
            for n, g in zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, q)):
                U.within(g, getattr(want, n), getattr(want, n + "_off"), n)
    apart = torch.zeros(4, (300 << 20) // 2, dtype=torch.float16, device="cuda")[:, :80 * d].unflatten(1, (80, d)).transpose(0, 1)
    apart.copy_(q)
    k, v = torch.randn(2, 80, 1, d, device="cuda").half()
    leaves = [apart.requires_grad_(), k.requires_grad_(), v.requires_grad_()]
    out = nn.segment_attention(*leaves, at)
    want = U.attention(q, k, v, [50, 30], [50, 30], False, 1 / math.sqrt(d), q)
    U.within(out, want.out, want.out_off, "out")
    for n, g in zip(("gq", "gk", "gv"), torch.autograd.grad(out, leaves, q)):
        U.within(g, getattr(want, n), getattr(want, n + "_off"), n)

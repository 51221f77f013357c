"""A block around attention over voxel clouds (FGMS.nn.VoxelBlock): its passes against its formula, in 8 bits, row by row over a cache,
with dropout; and the operators it is made of on other streams, in graphs, and with saved-tensor hooks."""
import threading

import pytest
import torch

from tests import attention_util as U
from tests import block_util as B

pytestmark = pytest.mark.gpu

LENGTHS = [33, 70, 1]


def inputs(dtype, seed=0, n=104, channels=64):
    gen = torch.Generator().manual_seed(seed)
    coords = torch.randint(0, 100, (n, 3), generator=gen, dtype=torch.int32).cuda()
    return torch.randn(n, channels, generator=gen).to(B.DTYPES[dtype]).cuda(), coords, U.offsets(LENGTHS)


def by_parts(block, feats, coords, offsets, factors=None):
    """The block's formula with torch's operations and VoxelAttention."""
    def norm(h, w):
        return h * w / torch.sqrt((h * h).mean(1, keepdim=True) + block.eps)
    one, two = factors if factors is not None else (1.0, 1.0)
    h = feats + one * block.attention(norm(feats, block.norm1), coords, offsets)
    a, b = block.up(norm(h, block.norm2)).chunk(2, 1)
    return h + two * block.down(torch.nn.functional.silu(a) * b)


def test_block_is_its_formula():
    """Both passes in fp32: sums of 64 to 128 products and a softmax, twenty operations in a row, each to 2^-24 of values of order
    one to ten: far below 4096 such steps."""
    from FGMS import nn
    torch.manual_seed(1)
    block = nn.VoxelBlock(64, 4, kv_heads=2, sections=(3, 3, 2), p=0.25, device="cuda")
    with torch.no_grad():
        block.norm1.normal_(1, 0.2), block.norm2.normal_(1, 0.2)
    feats, coords, offsets = inputs("fp32")
    g = torch.randn_like(feats)
    leaves = [feats.requires_grad_()] + list(block.parameters())

    def compare(factors):
        got = block(feats, coords, offsets)
        want = by_parts(block, feats, coords, offsets, factors)
        assert float((got - want).detach().abs().max()) < 4096 * 2.0 ** -24 * float(want.detach().abs().max())
        for a, b in zip(torch.autograd.grad(got, leaves, g), torch.autograd.grad(want, leaves, g)):
            assert float((a - b).abs().max()) < 4096 * 2.0 ** -24 * float(b.abs().max())

    block.eval()
    compare(None)
    block.train()
    # the seeds that the pass draws from torch's generator
    torch.manual_seed(5)
    drawn = [torch.randint(-1 << 63, (1 << 63) - 1, (2,), device="cuda") for _ in range(2)]
    torch.manual_seed(5)
    compare([B.factors(104, 64, 0.25, s).float().cuda() for s in drawn])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_block_in_eight_bits(dtype):
    from FGMS import nn
    torch.manual_seed(2)
    block = nn.VoxelBlock(64, 4, kv_heads=2, sections=(3, 3, 2), dtype=B.DTYPES[dtype], device="cuda").eval()
    feats, coords, offsets = inputs(dtype, 3)
    small = block.to_int8()
    assert block.up.weight.requires_grad and not any(p.requires_grad for p in small.parameters())
    assert small.up.weight.dtype == torch.int8 and small.attention.qkv.weight_scales.dtype == torch.float32
    with torch.no_grad():
        got, want = small(feats, coords, offsets), block(feats, coords, offsets)
        # step by step with the same operators
        q, s, h = nn.add_norm_int8(feats, None, small.norm1)
        x = small.attention((q, s), coords, offsets)
        q, s, h = nn.add_norm_int8(x, h, small.norm2)
        x = nn.int8_linear(q, s, small.up.weight, small.up.weight_scales, None, feats.dtype)
        x = nn.int8_linear(*nn.quantize_rows(x, gated=True), small.down.weight, small.down.weight_scales, None, feats.dtype)
        assert torch.equal(got, h + x)
    # 8 bits round at 1/254 of a row's largest, some 1/80 of its root mean square, on both sides of four products
    rms = float((got.double() - want.double()).square().mean().sqrt() / want.double().square().mean().sqrt())
    assert rms < 8 / 80
    # cast and moved layers keep their scales
    scales = small.down.weight_scales.clone()
    small.float()
    assert small.down.weight_scales.dtype == torch.float32 and torch.equal(small.down.weight_scales, scales)
    assert small(feats.float(), coords, offsets).dtype == torch.float32


@pytest.mark.parametrize("eight", [False, True])
def test_row_by_row(eight):
    """Rows one at a time over a cache are the causal block over all of them."""
    from FGMS import nn
    torch.manual_seed(3)
    scans, rows, channels = 3, 24, 64
    block = nn.VoxelBlock(channels, 4, kv_heads=2, sections=(3, 3, 2), causal=True, p=0.5, device="cuda").eval()
    block = block.to_int8() if eight else block
    feats = torch.randn(scans, rows, channels, device="cuda")
    coords = torch.randint(0, 50, (scans, rows, 3), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        whole = block(feats.flatten(0, 1), coords.flatten(0, 1), U.offsets([rows] * scans)).unflatten(0, (scans, rows))
        cache = nn.VoxelCache(scans, 32, block.attention.kv_heads, block.attention.dim, device="cuda")
        for i in range(rows):
            y = block.step(feats[:, i].contiguous(), coords[:, i].contiguous(), cache)
            off = (y - whole[:, i]).abs()
            if eight:      # (a value next to a border may be rounded the other way: a step of 1/127 of a row's largest, times weights of 1/8)
                assert float(off.max()) < 0.1 and float(off.median()) < 4096 * 2.0 ** -24, i
            else:
                assert float(off.max()) < 4096 * 2.0 ** -24, i


def test_moved_layers_keep_their_rows_on_sixteen_bytes():
    from FGMS import nn
    torch.manual_seed(6)
    linear = torch.nn.Linear(40, 7, device="cuda")
    layer = nn.Int8Linear(linear)
    x = torch.randn(9, 40, device="cuda")
    with torch.no_grad():
        want = layer(x)
        assert layer.weight.shape == (7, 40) and layer.weight.stride(0) == 48
        back = layer.cpu().cuda()
        assert back.weight.stride(0) == 48 and torch.equal(back(x), want)
        fresh = nn.Int8Linear(torch.nn.Linear(40, 7, device="cuda"))
        fresh.load_state_dict(layer.state_dict())
        assert torch.equal(fresh(x), want) and layer.half()(x.half()).dtype == torch.float16
        with pytest.raises(ValueError, match="Linear"):
            nn.Int8Linear(layer)
        # 8 bits of x and of the weights, each off by up to half a step of 1/127 of a row's largest
        exact = x.double() @ linear.weight.double().t() + linear.bias.double()
        off = (x.abs().amax(1, keepdim=True) / 254 * 1.01).double() * linear.weight.double().abs().sum(1) \
            + x.double().abs().sum(1, keepdim=True) * (linear.weight.abs().amax(1) / 254 * 1.02).double() + 1e-5
        assert ((want.double() - exact).abs() <= off).all()


def test_block_without_gradients_over_caches():
    from FGMS import nn
    block = nn.VoxelBlock(64, 4, device="cuda")
    cache = nn.VoxelCache(2, 8, 4, 16, device="cuda")
    feats, coords = torch.randn(2, 64, device="cuda"), torch.zeros(2, 3, dtype=torch.int32, device="cuda")
    with pytest.raises(ValueError, match="no_grad"):
        block.step(feats, coords, cache)
    assert cache.lengths.tolist() == [0, 0]


def step(s, seed):
    """A training step through the operators, as one list of results."""
    from FGMS import nn
    x, r, w, gy = s
    y, h = nn.add_norm(x, r, w, p=0.2, seed=seed)
    z = nn.dropout_add(y, h, 0.3, seed)
    return [t.detach() for t in (y, h, z)] + list(torch.autograd.grad(z, (x, r, w), gy))


def leaves(n, c, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    t = [torch.randn(n, c, generator=gen).to(dtype).cuda() for _ in range(3)]
    w = torch.randn(c, generator=gen).to(dtype).cuda()
    return [t[0].requires_grad_(), t[1].requires_grad_(), w.requires_grad_(), t[2]]


@pytest.mark.parametrize("shape", [(500, 64), (70, 1096)], ids=str)
def test_streams_and_graphs(shape):
    s = leaves(*shape, torch.float16, 1)
    seed = torch.tensor([1, 2], device="cuda")
    want = step(s, seed)
    side = U.own_stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(s, seed)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    # two graphs on one stream, replayed in turn over other seeds and values
    graphs, kept = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept.append(step(s, seed))
        graphs.append(graph)
    for i in range(4):
        with torch.no_grad():
            seed.copy_(torch.tensor([i, -i]))
            s[0].mul_(1.5)
        eager = step(s, seed)
        for t in kept[i % 2]:
            with torch.no_grad():
                t.zero_()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(eager, kept[i % 2])), i
    # both at once on two streams
    other = U.own_stream()
    for _ in range(3):
        with torch.cuda.stream(side):
            graphs[0].replay()
        with torch.cuda.stream(other):
            graphs[1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(eager, *kept))


def test_captured_backward_next_to_an_eager_graph():
    """A gradient that would leave the capture is refused, and the capture ends as it should."""
    from FGMS import nn
    x, r, w, g = leaves(64, 64, torch.float16, 8)
    seed = torch.tensor([1, 2], device="cuda")
    side = U.own_stream()
    for call in (lambda: nn.add_norm(x, r, w)[0], lambda: nn.dropout_add(x, r, 0.5, seed)):
        eager = call()
        want = torch.autograd.grad(eager, x, g, retain_graph=True)[0]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            y = call()
            with pytest.raises(RuntimeError, match="eager pass"):
                torch.autograd.grad(y, x, g)
        del eager, y
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            got = torch.autograd.grad(call(), x, g)[0]
        for _ in range(2):
            with torch.no_grad():
                got.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)


def test_inference_in_a_graph():
    from FGMS import nn
    torch.manual_seed(4)
    block = nn.VoxelBlock(64, 4, dtype=torch.float16, device="cuda").eval().to_int8()
    feats, coords, offsets = inputs("fp16", 6)
    side = U.own_stream()
    with torch.no_grad():
        with torch.cuda.stream(side):
            block(feats, coords, offsets)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            kept = block(feats, coords, offsets)
        for i in range(3):
            feats.mul_(1.25)
            want = block(feats, coords, offsets)
            kept.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(want, kept), i


def test_two_threads():
    """Calls of two threads, on a stream each and on one stream."""
    sets = [leaves(400, 96, torch.bfloat16, i) for i in range(2)]
    seed = torch.tensor([1, 2], device="cuda")
    want = [step(s, seed) for s in sets]
    torch.cuda.synchronize()
    streams = [U.own_stream(), U.own_stream()]
    for pair in (streams, [streams[0]] * 2):
        got, errors = [None, None], []

        def work(i):
            try:
                with torch.cuda.stream(pair[i]):
                    for _ in range(20):
                        got[i] = step(sets[i], seed)
            except Exception as e:      # (told by the assertion below)
                errors.append(e)

        threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        torch.cuda.synchronize()
        assert not errors
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(want[i], got[i]))


def test_saved_tensors_tangents_and_traces():
    import torch.autograd.forward_ad as fwd
    from FGMS import nn
    s = leaves(60, 64, torch.float16, 2)
    x, r, w, g = s
    seed = torch.tensor([3, 4], device="cuda")
    want = torch.autograd.grad(nn.add_norm(x, r, w, p=0.5, seed=seed)[0], (x, r, w), g)
    with torch.autograd.graph.save_on_cpu():
        y = nn.add_norm(x, r, w, p=0.5, seed=seed)[0]
    assert all(torch.equal(a, b) for a, b in zip(want, torch.autograd.grad(y, (x, r, w), g)))
    with torch.autograd.graph.saved_tensors_hooks(lambda t: t, lambda t: t.float()):
        y = nn.add_norm(x, r, w)[0]
    with pytest.raises(ValueError):
        torch.autograd.grad(y, x, g)
    with fwd.dual_level():
        dual = fwd.make_dual(x.detach(), g)
        for f in (lambda: nn.add_norm(dual), lambda: nn.add_norm(g, dual), lambda: nn.dropout_add(dual, p=0.0), lambda: nn.quantize_rows(dual)):
            with pytest.raises(NotImplementedError):
                f()

    constant = w.detach()

    def chain(x, r):
        y, h = nn.add_norm(x, r, constant, p=0.5, seed=seed)
        q, scales, h = nn.add_norm_int8(y, h)
        y = nn.int8_linear(q, scales, q[:8], scales[:8])
        q, scales = nn.quantize_rows(y)
        return nn.dropout_add(h, y.repeat(1, 8), 0.5, seed) * scales[:, None]

    traced = torch.jit.trace(chain, (x.detach(), r.detach()), check_trace=False)
    assert torch.equal(traced(g, x.detach()), chain(g, x.detach()))


def test_network_with_convolutions():
    """Blocks between sparse convolutions, as one network: every parameter has a gradient."""
    from fgms_amd import clouds
    from FGMS import nn
    from tests.test_gpu_voxel_attention import small_cloud
    torch.manual_seed(0)
    coords = small_cloud(1)
    order, offsets = nn.window_segments(coords, 6)
    coords = coords[order].contiguous()
    kmap = nn.KernelMap.from_coords(coords, coords, clouds.offsets_cube(3))
    first = nn.SparseConv(8, 32, 27, device="cuda")
    blocks = torch.nn.ModuleList(nn.VoxelBlock(32, 4, kv_heads=2, sections=(2, 1, 1), p=0.1, device="cuda") for _ in range(2))
    last = nn.SparseConv(32, 8, 27, device="cuda")
    x = torch.randn(len(coords), 8, device="cuda")

    def through(blocks):
        y = first(x, kmap)
        for block in blocks:
            y = block(y, coords, offsets)
        return last(y, kmap)

    through(blocks).square().mean().backward()
    for p in (p for m in (first, blocks, last) for p in m.parameters()):
        assert p.grad is not None and torch.isfinite(p.grad).all() and p.grad.any()
    with torch.no_grad():
        y = through([b.to_int8() for b in blocks])
    assert torch.isfinite(y).all()

"""What goes around attention, through the C entry points (fgms_amd.capi): the same bits as FGMS.nn, results between other values, and
what the binding refuses."""
import pytest
import torch

from tests import block_util as B

pytestmark = pytest.mark.gpu


@pytest.fixture(autouse=True)
def half_by_default():
    """(room that a binding makes has its own type, whatever torch's default is)"""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float16)
    yield
    torch.set_default_dtype(before)


@pytest.mark.parametrize("dtype", list(B.DTYPES))
@pytest.mark.parametrize("shape", [(300, 64), (70, 1096), (41, 37), (6, 9000)], ids=str)
def test_same_bits(shape, dtype):
    from FGMS import nn
    from fgms_amd import capi
    gen = torch.Generator().manual_seed(shape[1])
    n, c = shape
    x, r, gy, gh = (torch.randn(n, c, generator=gen, dtype=torch.float32).to(B.DTYPES[dtype]).cuda() for _ in range(4))
    w = torch.randn(c, generator=gen, dtype=torch.float32).to(B.DTYPES[dtype]).cuda()
    seed = torch.tensor([5, 6], device="cuda")
    leaves = [t.clone().requires_grad_() for t in (x, r, w)]
    y, h = nn.add_norm(*leaves, p=0.3, seed=seed)
    want = torch.autograd.grad((y, h), leaves, (gy, gh))
    out, total = torch.empty_like(x), torch.empty_like(x)
    capi.add_norm_fwd(x, r, w, total, out, p=0.3, seed=seed)
    assert torch.equal(out, y) and torch.equal(total, h)
    capi.add_norm_fwd(x, r, w, None, out.zero_(), p=0.3, seed=seed)
    assert torch.equal(out, y)
    grads = [torch.empty_like(t) for t in (x, r, w)]
    capi.add_norm_bwd(gy, gh, total, w, *grads, p=0.3, seed=seed)
    assert all(torch.equal(a, b) for a, b in zip(grads, want))
    # each on its own, and both names of one gradient without dropout
    for i in range(3):
        one = [torch.empty_like(t) if k == i else None for k, t in enumerate((x, r, w))]
        capi.add_norm_bwd(gy, gh, total, w, *one, p=0.3, seed=seed)
        assert torch.equal(one[i], want[i])
    capi.add_norm_bwd(gy, None, total, None, grads[0], grads[1])
    assert torch.equal(grads[0], grads[1])
    capi.dropout_add(x, r, out, 0.3, seed)
    assert torch.equal(out, nn.dropout_add(x, r, 0.3, seed))
    # rows of results between other values, beginning anywhere
    for lead, width in ((0, c), (5, c + 11), (16, c + 48)):
        held = torch.full((n, width), 99, dtype=torch.int8, device="cuda")
        q, scales = held[:, lead:lead + c], torch.empty(n, dtype=torch.float32, device="cuda")
        capi.quantize_rows(x, q, scales)
        want_q, want_s = nn.quantize_rows(x)
        assert torch.equal(q, want_q) and torch.equal(scales, want_s)
        capi.add_norm_int8(x, r, w, total, q, scales)
        want_q, want_s, want_h = nn.add_norm_int8(x, r, w)
        assert torch.equal(q, want_q) and torch.equal(scales, want_s) and torch.equal(total, want_h)
        assert (held[:, :lead] == 99).all() and (held[:, lead + c:] == 99).all()
    padded = (c + 15) // 16 * 16
    q = torch.zeros(n, padded, dtype=torch.int8, device="cuda")[:, :c]
    capi.quantize_rows(x, q, scales)
    out = torch.full((n + 2, n), 7, dtype=B.DTYPES[dtype], device="cuda")
    capi.int8_linear(q, scales, q, scales, w[:1].expand(n).contiguous(), out[1:-1])
    assert torch.equal(out[1:-1], nn.int8_linear(q, scales, q, scales, w[:1].expand(n), B.DTYPES[dtype]))
    assert (out[0] == 7).all() and (out[-1] == 7).all()


def test_results_stay_between_their_neighbours():
    """Results of every kind of launch that begin anywhere: what lies in front of them and behind is left as it was."""
    from fgms_amd import capi
    for n, outputs, c in ((1, 17, 64), (20, 300, 640), (100, 130, 100), (70, 1000, 2100), (3000, 777, 300), (9000, 71, 60), (4200, 4101, 1100), (40, 9000, 256)):
        x = torch.randint(-9, 9, (n, (c + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :c]
        w = torch.randint(-9, 9, (outputs, (c + 15) // 16 * 16), dtype=torch.int8, device="cuda")[:, :c]
        for dtype in B.DTYPES.values():
            held = torch.full((n * outputs + 21,), 5, dtype=dtype, device="cuda")
            out = held[3:3 + n * outputs].view(n, outputs)
            sx, sw = torch.ones(n, dtype=torch.float32, device="cuda"), torch.full((outputs,), 0.125, dtype=torch.float32, device="cuda")
            capi.int8_linear(x, sx, w, sw, None, out)
            want = (x.double() @ w.double().t().contiguous()) / 8
            assert ((out.double() - want).abs() <= B.UNIT[dtype] * want.abs()).all(), (n, outputs, c)
            assert (held[:3] == 5).all() and (held[3 + n * outputs:] == 5).all(), (n, outputs, c)


def test_results_end_anywhere():
    """Rows of results of every length over tiles of every size, that begin on four bytes, beside it, or in turns."""
    from fgms_amd import capi
    gen = torch.Generator().manual_seed(77)
    for n, c, lengths in ((33, 64, range(1, 140)), (33, 300, range(50, 140)), (70, 2100, range(60, 75)), (16500, 80, range(225, 262)), (16500, 200, range(225, 262)),
                          (33000, 1100, (511, 513, 523, 537, 549))):
        x = torch.randint(-9, 10, (n, (c + 15) // 16 * 16), generator=gen).char().cuda()[:, :c]
        w = torch.randint(-9, 10, (max(lengths), (c + 15) // 16 * 16), generator=gen).char().cuda()[:, :c]
        sx, sw = (torch.full((k,), v, dtype=torch.float32, device="cuda") for k, v in ((n, 1.0), (max(lengths), 2.0 ** -8)))
        sums = x.float() @ w.float().t() / 256      # (whole numbers under 2^24: exact)
        for outputs in lengths:
            for dtype in (torch.float16, torch.bfloat16):
                held = torch.full((n * outputs + 9,), 5, dtype=dtype, device="cuda")
                begin = 3 + outputs // 2 % 2
                out = held[begin:begin + n * outputs].view(n, outputs)
                capi.int8_linear(x, sx, w[:outputs], sw[:outputs], None, out)
                assert torch.equal(out, sums[:, :outputs].to(dtype)), (n, c, outputs, dtype)
                assert (held[:begin] == 5).all() and (held[begin + n * outputs:] == 5).all(), (n, c, outputs, dtype)


def test_binding_refuses():
    from fgms_amd import capi
    x, q, s = torch.zeros(4, 24, device="cuda"), torch.zeros(4, 24, dtype=torch.int8, device="cuda"), torch.zeros(4, dtype=torch.float32, device="cuda")
    w = torch.zeros(24, device="cuda")
    out = torch.zeros(4, 4, device="cuda")
    for call in (lambda: capi.add_norm_fwd(x, x[:3], None, None, x), lambda: capi.add_norm_fwd(x, None, w[:3], None, x), lambda: capi.add_norm_fwd(x.t(), None, None, None, x),
                 lambda: capi.add_norm_fwd(x, None, None, None, x.float()), lambda: capi.add_norm_bwd(x[:3], None, x, None, x, None),
                 lambda: capi.add_norm_bwd(x, x.float(), x, None, x, None), lambda: capi.dropout_add(x, None, x, 0.5), lambda: capi.dropout_add(x, None, x, 0.5, s),
                 lambda: capi.quantize_rows(x, q[:, :8], s), lambda: capi.quantize_rows(x, q, s[:3]), lambda: capi.quantize_rows(x[:, :23], q[:, :11], s, gated=True),
                 lambda: capi.quantize_rows(x, q[:1].expand(4, 24), s), lambda: capi.int8_linear(q, s, q, s, None, out), lambda: capi.add_norm_int8(x, None, w.float(), None, q, s)):
        with pytest.raises(ValueError):
            call()
    held = torch.zeros(4, 32, dtype=torch.int8, device="cuda")
    for call in (lambda: capi.int8_linear(held[:, :24], s[:3], held[:, :24], s, None, out), lambda: capi.int8_linear(held[:, :24], s, held[:, 8:], s, None, out),
                 lambda: capi.int8_linear(held[:, :24], s, held[:, :24], s, w, out), lambda: capi.int8_linear(held.flatten()[8:120].as_strided((4, 24), (32, 1)), s, held[:, :24], s, None, out)):
        with pytest.raises(ValueError):
            call()

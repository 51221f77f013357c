"""fp16 attention whose scores' gradients pass the type's range where the results do not."""
import math

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu


def gradients(q, k, v, g, scale, group):
    """gq, gk, gv in 64 bits and, for each, what the scores' gradients may be off by where they are held in a lower power of
    two because their row (gq) or column (gk) has one that 2^4 takes out of fp16's range: one at level s reaches 2^(1 - s), half
    a step there is 2^-(25 + s): 2^-26 of the largest."""
    q, k, v, g = (t.detach().cpu().double() for t in (q, k, v, g))
    gq, gk = torch.zeros_like(q), torch.zeros_like(k)
    gq_more, gk_more = torch.zeros_like(q), torch.zeros_like(k)
    largest = 0.0
    most_key = torch.zeros(k.shape[0], k.shape[1], dtype=torch.float64)
    for h in range(q.shape[1]):
        a, b, c, go = q[:, h], k[:, h // group], v[:, h // group], g[:, h]
        p = torch.softmax(a @ b.T * scale, 1)
        ds = p * (go @ c.T - (go * (p @ c)).sum(1, keepdim=True))
        largest = max(largest, float(ds.abs().max()))
        gq_more[:, h] = 2.0 ** -26 * ds.abs().amax(1, keepdim=True) * b.abs().sum(0) * scale
        most_key[:, h // group] = torch.maximum(most_key[:, h // group], ds.abs().amax(0))
    for h in range(q.shape[1]):
        gk_more[:, h // group] += 2.0 ** -26 * most_key[:, h // group, None] * q[:, h].abs().sum(0) * scale
    return largest, gq_more, gk_more


# queries, keys, heads, key heads, channels, size of q and k, of v, of g
LARGE = {
    "loss-scaled": (6, 4, 2, 2, 128, 1.0, 1.0, 2000.0),
    "few-rows-of-many": (300, 200, 4, 2, 64, 3.0, 4.0, 3000.0),
    "split-keys": (20, 3000, 2, 1, 32, 8.0, 16.0, 6000.0),
    "split-queries": (3000, 20, 1, 1, 96, 4.0, 4.0, 6000.0),
    "narrow": (130, 90, 3, 1, 16, 2.0, 16.0, 6000.0),
    "beyond": (40, 30, 2, 2, 128, 2.0 ** -18, 12000.0, 12000.0),
}


@pytest.mark.parametrize("case", list(LARGE))
def test_large_gradients(case):
    """Scores' gradients beyond 4094 (2^4 times which passes fp16's end) whose sums, the results, are inside fp16."""
    from FGMS import nn
    nq, nk, h, hk, d, size, v_size, g_size = LARGE[case]
    gen = torch.Generator().manual_seed(1)

    def normal(rows, heads, by):
        return (torch.randn(rows, heads, d, generator=gen) * by).half().cuda()

    q, k, v, g = normal(nq, h, size), normal(nk, hk, size), normal(nk, hk, v_size), normal(nq, h, g_size)
    if case in ("few-rows-of-many", "split-keys", "split-queries", "narrow"):
        g[3:] /= 4096      # the other rows' gradients stay small, and keep their bits
    scale = 2.0 ** -7 if case in ("split-keys", "split-queries") else 1 / math.sqrt(d) / 4
    leaves = [t.requires_grad_() for t in (q, k, v)]
    out = nn.segment_attention(*leaves, U.offsets([nq]), U.offsets([nk]), scale=scale)
    got = torch.autograd.grad(out, leaves, g, retain_graph=True)
    want = U.attention(q, k, v, [nq], [nk], False, scale, g)
    largest, gq_more, gk_more = gradients(q, k, v, g, scale, h // hk)
    assert largest > (65520 << 11 if case == "beyond" else 4100), largest
    assert max(float(t.abs().max()) for t in (want.gq, want.gk, want.gv)) < 65000
    U.within(got[0], want.gq, want.gq_off + gq_more, "gq")
    U.within(got[1], want.gk, want.gk_off + gk_more, "gk")
    U.within(got[2], want.gv, want.gv_off, "gv")
    assert all(torch.equal(a, b) for a, b in zip(got, torch.autograd.grad(out, leaves, g, retain_graph=True)))
    for i, t in enumerate(leaves):
        assert torch.equal(torch.autograd.grad(out, t, g, retain_graph=True)[0], got[i])


@pytest.mark.parametrize("spoil", ["g", "k", "v"])
def test_infinite_inputs_end(spoil):
    """Gradients that no power of two makes finite come out as they are, and other segments' do not change."""
    from FGMS import nn
    torch.manual_seed(2)
    lengths, d = [90, 70, 40], 64
    q, k, v, g = (torch.randn(200, 2, d, device="cuda").half() for _ in range(4))

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        out = nn.segment_attention(*leaves, U.offsets(lengths), causal=True)
        return torch.autograd.grad(out, leaves, g)

    plain = run()
    dict(g=g, k=k, v=v)[spoil][100] = math.inf
    got = run()
    for a, b in zip(plain, got):
        assert torch.equal(a[:90], b[:90]) and torch.equal(a[160:], b[160:])
    assert not torch.isfinite(got[0][100:160]).all()

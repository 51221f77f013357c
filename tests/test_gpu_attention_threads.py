"""Two host threads that share a stream: calls of several launches, which hand sums over in a buffer of the stream, do not come
between each other's."""
import threading

import pytest
import torch

from tests import attention_util as U

pytestmark = pytest.mark.gpu
ROUNDS = 60


def both(work):
    """work(0) and work(1) in threads of their own, on one stream; what either raised comes back."""
    stream, failed = U.own_stream(), []
    stream.wait_stream(torch.cuda.current_stream())
    start = threading.Barrier(2)

    def run(i):
        try:
            with torch.cuda.stream(stream):
                start.wait()
                for _ in range(ROUNDS):
                    work(i)
        except BaseException as e:      # noqa: B902 (re-raised below)
            failed.append(e)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    stream.synchronize()
    if failed:
        raise failed[0]


def test_rows_over_caches():
    from fgms_amd import capi
    gen = torch.Generator(device="cuda").manual_seed(0)
    q, k, v, want = [], [], [], []
    ko, qo = U.offsets([6000, 5000]), U.offsets([1, 1])
    for i in range(2):
        q.append(torch.randn(2, 8, 64, device="cuda", generator=gen).half())
        k.append(torch.randn(11000, 2, 64, device="cuda", generator=gen).half())
        v.append(torch.randn(11000, 2, 64, device="cuda", generator=gen).half())
        want.append(torch.empty_like(q[i]))
        capi.segment_attention_fwd(q[i], k[i], v[i], want[i], None, qo, ko, scale=0.125)
    got = [[torch.empty_like(q[i]) for _ in range(ROUNDS)] for i in range(2)]
    count = [0, 0]
    torch.cuda.synchronize()

    def work(i):
        capi.segment_attention_fwd(q[i], k[i], v[i], got[i][count[i]], None, qo, ko, scale=0.125)
        count[i] += 1

    both(work)
    assert all(torch.equal(t, want[i]) for i in range(2) for t in got[i])


def test_gradients():
    from FGMS import nn
    gen = torch.Generator(device="cuda").manual_seed(1)
    sections, at = (8, 8), U.offsets([700, 500])
    inputs, want = [], []
    for i in range(2):
        x = [torch.randn(1200, 2, 32, device="cuda", generator=gen).half().requires_grad_() for _ in range(3)]
        scale = torch.ones(32, device="cuda").half().requires_grad_()
        coords = torch.randint(0, 99, (1200, 2), dtype=torch.int32, device="cuda", generator=gen)
        inputs.append((x, scale, coords, torch.randn(1200, 2, 32, device="cuda", generator=gen).half()))
    freqs = nn.rotary_freqs(sections, device="cuda")

    def step(i):
        (q, k, v), scale, coords, g = inputs[i]
        out = nn.segment_attention(*nn.norm_rotary(q, k, scale, None, coords, freqs, sections), v, at)
        return torch.autograd.grad(out, (q, k, v, scale), g)

    want = [step(i) for i in range(2)]
    got = [[], []]
    torch.cuda.synchronize()
    both(lambda i: got[i].append(step(i)))
    assert all(torch.equal(a, b) for i in range(2) for grads in got[i] for a, b in zip(grads, want[i]))

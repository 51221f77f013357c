"""Plain attention inside segments and plain norms with rotation, in 64 bits on the CPU, with how far a kernel's results
may be off: each rounding of the kernels (to the inputs' type, of an fp32 sum) carried through the formulas."""
import ctypes
import math
from types import SimpleNamespace

import torch

from fgms_amd import capi

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
UNIT = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}      # half a step
TINY = {torch.float16: 2.0 ** -24, torch.bfloat16: 0.0, torch.float32: 0.0}                   # fp16's last step
SUM = 2.0 ** -24


def own_stream():
    """A stream of the caller's own, not one of torch's pool (made through the runtime that the library is linked to)."""
    runtime = ctypes.CDLL(capi.LIB_PATH)
    runtime.hipStreamCreateWithFlags.argtypes = [ctypes.POINTER(ctypes.c_void_p), ctypes.c_uint]
    handle = ctypes.c_void_p()
    assert runtime.hipStreamCreateWithFlags(ctypes.byref(handle), 1) == 0      # hipStreamNonBlocking
    return torch.cuda.ExternalStream(handle.value)


def offsets(lengths, device="cuda"):
    t = torch.zeros(len(lengths) + 1, dtype=torch.int32)
    t[1:] = torch.tensor(lengths, dtype=torch.int32).cumsum(0)
    return t.to(device)


def attention(q, k, v, q_lengths, k_lengths, causal, scale, g=None):
    """results: out, lse and, with g, gq, gk, gv; the same names with _off: how far each element may be off."""
    dtype, u, tiny = q.dtype, UNIT[q.dtype], TINY[q.dtype]
    # probabilities and ds are rounded to the type for their products (fp32: not)
    up = u if dtype != torch.float32 else 0.0
    q, k, v = (t.detach().cpu().double() for t in (q, k, v))
    g = None if g is None else g.detach().cpu().double()
    nq, h, d = q.shape
    group = h // k.shape[1]
    r = SimpleNamespace(out=torch.zeros_like(q), lse=torch.full((nq, h), -math.inf, dtype=torch.float64), out_off=torch.zeros_like(q),
                        lse_off=torch.zeros(nq, h, dtype=torch.float64))
    if g is not None:
        for n, t in (("gq", q), ("gk", k), ("gv", v)):
            setattr(r, n, torch.zeros_like(t))
            setattr(r, n + "_off", torch.zeros_like(t))
    q0 = k0 = 0
    for lq, lk in zip(q_lengths, k_lengths):
        rows, cols = slice(q0, q0 + lq), slice(k0, k0 + lk)
        q0, k0 = q0 + lq, k0 + lk
        if not lq or not lk:
            continue
        sees = torch.ones(lq, lk, dtype=torch.bool)
        if causal:
            sees = torch.arange(lk)[None] <= torch.arange(lq)[:, None] + (lk - lq)
        some = sees.any(1)
        for head in range(h):
            a, b, c = q[rows, head], k[cols, head // group], v[cols, head // group]
            s = (a @ b.T * scale).masked_fill(~sees, -math.inf)
            lse = torch.logsumexp(s, 1)
            p = torch.exp(s - lse[:, None]).masked_fill(~sees, 0.0)
            o = p @ c
            r.out[rows, head] = o
            r.lse[rows, head] = lse
            # a score: a sum of d products, its scaling, the exponent's argument and the exponential, beside the maximum
            ds_ = SUM * ((d + 8) * (a.abs() @ b.abs().T * scale) + 4 * s.masked_fill(~sees, 0.0).abs().amax(1, keepdim=True) + 16)
            pe = p * (ds_ + ds_.amax(1, keepdim=True) + SUM * (lk + 8))      # p, and the sum it is divided by
            r.lse_off[rows, head] = torch.where(some, ds_.amax(1) + SUM * (lk + 8) + 4 * SUM * lse.abs(), 0.0)
            # (fp16: a probability against the row's largest below 2^-14 is rounded to 2^-24 steps)
            least = tiny * p.amax(1, keepdim=True) * sees
            po = pe + 2 * up * p + least
            r.out_off[rows, head] = po @ c.abs() + u * o.abs() + SUM * (lk + 8) * (p @ c.abs()) + tiny
            if g is None:
                continue
            go = g[rows, head]
            dp = go @ c.T
            delta = (go * o).sum(1, keepdim=True)
            ds = p * (dp - delta)
            # delta from the rounded result; dp and delta are sums of d products
            dd = (go.abs() * (2 * r.out_off[rows, head] + u * o.abs())).sum(1, keepdim=True) + SUM * (d + 4) * (go.abs() * o.abs()).sum(1, keepdim=True)
            dse = pe * (dp - delta).abs() + p * (SUM * (d + 4) * (go.abs() @ c.abs().T) + dd) + 2 * up * ds.abs() + tiny / 8
            pse = pe + 2 * up * p + tiny / 512
            kv = head // group
            r.gq[rows, head] = ds @ b * scale
            r.gk[cols, kv] += ds.T @ a * scale
            r.gv[cols, kv] += p.T @ go
            r.gq_off[rows, head] = dse * sees @ b.abs() * scale + SUM * (lk + 8) * (ds.abs() @ b.abs() * scale) + u * r.gq[rows, head].abs() + tiny
            n = lq * group + 8
            r.gk_off[cols, kv] += (dse * sees).T @ a.abs() * scale + SUM * n * (ds.abs().T @ a.abs() * scale)
            r.gv_off[cols, kv] += (pse * sees).T @ go.abs() + SUM * n * (p.T @ go.abs())
    if g is not None:
        r.gk_off += u * r.gk.abs() + tiny
        r.gv_off += u * r.gv.abs() + tiny
    return r


def turned(x, w, coords, freqs, sections, eps, interleaved, g=None):
    """(y, how far it may be off, gx, off, gw, off) of one of the two tensors."""
    u, tiny = UNIT[x.dtype], TINY[x.dtype]
    x = x.detach().cpu().double()
    w = torch.ones(x.shape[2], dtype=torch.float64) if w is None else w.detach().cpu().double()
    n, h, d = x.shape
    axis = [a for a, c in enumerate(sections) for _ in range(c)]
    phi = torch.zeros(n, d // 2, dtype=torch.float64)
    phi[:, :len(axis)] = coords.cpu().double()[:, axis] * freqs.cpu().double()
    cos, sin = phi.cos()[:, None], phi.sin()[:, None]

    def pairs(t):
        return (t[..., 0::2], t[..., 1::2]) if interleaved else (t[..., :d // 2], t[..., d // 2:])

    def turn(t, sin):
        a, b = pairs(t)
        y = torch.empty_like(t)
        ya, yb = pairs(y)
        ya.copy_(a * cos - b * sin)
        yb.copy_(a * sin + b * cos)
        return y

    def size(t):      # of both channels of a pair
        a, b = pairs(t.abs())
        y = torch.empty_like(t)
        for part in pairs(y):
            part.copy_(a + b)
        return y

    r = 1 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    z = x * r * w
    y = turn(z, sin)
    y_off = u * y.abs() + SUM * (d + 16) * size(z) + tiny
    if g is None:
        return y, y_off
    g = g.detach().cpu().double()
    back = turn(g, -sin)
    along = (w * back * x).mean(-1, keepdim=True)
    gx = r * (w * back - x * r * r * along)
    gw = (back * x * r).sum((0, 1))
    e = SUM * (2 * d + 32)
    gx_off = u * gx.abs() + e * r * ((w * size(g)).abs() + x.abs() * r * r * (w * size(g) * x).abs().mean(-1, keepdim=True)) + tiny
    gw_off = u * gw.abs() + (SUM * (d + 64 + n * h) * (size(g) * x * r).abs()).sum((0, 1)) + tiny
    return y, y_off, gx, gx_off, gw, gw_off


def within(got, want, off, what=""):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), what + ": not finite"
    over = (got - want).abs() - off
    if over.numel() and over.max() > 0:
        i = int(over.argmax())
        raise AssertionError("%s: %d of %d off by more than they may, worst %g for %g, allowed %g"
                             % (what, int((over > 0).sum()), over.numel(), got.flatten()[i], want.flatten()[i], off.flatten()[i]))

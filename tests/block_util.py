"""Plain forms of what goes around attention in a block, in 64 bits on the CPU, with how far a kernel's results may be off: each
rounding (to the inputs' type, of an fp32 sum) carried through the formulas."""
import torch

from tests.attention_util import DTYPES, SUM, TINY, UNIT, within  # noqa: F401

MASK = 0xFFFFFFFF


def philox(counter, key):
    """Philox4x32 with ten rounds: counter four, key two whole numbers below 2^32 (or tensors of them)."""
    def product(a, factor):      # 32 x 32 bits, in halves (64-bit numbers have a sign)
        low, high = (a & 0xFFFF) * factor, (a >> 16) * factor
        middle = high + (low >> 16)
        return middle >> 16, (middle & 0xFFFF) << 16 | low & 0xFFFF
    c, k = list(counter), list(key)
    for _ in range(10):
        up0, low0 = product(c[0], 0xD2511F53)
        up1, low1 = product(c[2], 0xCD9E8D57)
        c = [up1 ^ c[1] ^ k[0], low1, up0 ^ c[3] ^ k[1], low0]
        k = [(k[0] + 0x9E3779B9) & MASK, (k[1] + 0xBB67AE85) & MASK]
    return c


def factors(rows, channels, p, seed):
    """What dropout multiplies each element with."""
    fall = round(p * 65536)
    if not fall:
        return torch.ones(rows, channels, dtype=torch.float64)
    per = (channels + 7) // 8
    key, stream = (int(s) & ((1 << 64) - 1) for s in seed.tolist())
    chunk = torch.arange(rows * per)
    words = philox([chunk & MASK, chunk >> 32, torch.full_like(chunk, stream & MASK), torch.full_like(chunk, stream >> 32)], [key & MASK, key >> 32])
    words = torch.stack([w >> shift & 0xFFFF for w in words for shift in (0, 16)], 1).reshape(rows, 8 * per)[:, :channels]
    return (words >= fall).double() * (65536 / (65536 - fall))


def cpu(t):
    return None if t is None else t.detach().cpu().double()


def total(x, residual, factor):
    """(h, how far it may be off) of a sum with dropout."""
    u, tiny = UNIT[x.dtype], TINY[x.dtype]
    part = cpu(x) * factor
    h = part if residual is None else part + cpu(residual)
    return h, u * (1 + u) * h.abs() + 4 * SUM * (part.abs() + h.abs()) + tiny


def normed(h, scale, eps, unit=None):
    """(y, how far it may be off) of the norm of stored rows; unit 0: before it is rounded to their type."""
    u, tiny = (UNIT[h.dtype], TINY[h.dtype]) if unit is None else (unit, 0.0)
    h = cpu(h)
    w = torch.ones(h.shape[1], dtype=torch.float64) if scale is None else cpu(scale)
    y = h * w / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    return y, (u + SUM * (h.shape[1] + 16)) * y.abs() + tiny


def norm_grads(h, scale, eps, gy, gh, factor):
    """(g of the sum, off, g of x, off, g of scale, off) for stored rows h."""
    u, tiny = UNIT[h.dtype], TINY[h.dtype]
    n, c = h.shape
    h, g = cpu(h), cpu(gy)
    w = torch.ones(c, dtype=torch.float64) if scale is None else cpu(scale)
    r = 1 / torch.sqrt((h * h).mean(1, keepdim=True) + eps)
    along = (w * g * h).mean(1, keepdim=True)
    gs = r * (w * g - h * r * r * along)
    off = SUM * (2 * c + 48) * r * ((w * g).abs() + h.abs() * r * r * (w * g * h).abs().mean(1, keepdim=True))
    if gh is not None:
        gs = gs + cpu(gh)
        off = off + SUM * gs.abs()
    gw = (g * h * r).sum(0)
    gw_off = u * gw.abs() + (SUM * (n + c + 64) * (g * h * r).abs()).sum(0) + tiny
    gx = gs * factor
    return gs, off + u * gs.abs() + tiny, gx, off * factor + (u + 4 * SUM) * gx.abs() + tiny, gw, gw_off


def check_eighths(q, scales, v, off, what=""):
    """Rows in 8 bits against the values that they stand for, each up to `off` from `v`."""
    q, scales = q.detach().cpu().double(), scales.detach().cpu().double()
    top, slack = v.abs().amax(1), off.amax(1)
    assert ((scales - top / 127).abs() <= slack / 127 + 2 * SUM * top / 127).all(), what + ": scales"
    there = scales > 0
    assert (q[~there] == 0).all() and (q.abs() <= 127).all(), what
    v, off, q, scales = v[there], off[there], q[there], scales[there][:, None]
    over = (q - v / scales).abs() - (0.5 + off / scales + 4 * SUM * 127)
    assert over.numel() == 0 or over.max() <= 0, (what, float(over.max()))


def product(q, q_scales, weight, weight_scales, bias, dtype):
    """(y, how far it may be off); the sums of whole numbers are exact in 64 bits."""
    u, tiny = UNIT[dtype], TINY[dtype]
    y = cpu(q) @ cpu(weight).T * cpu(q_scales)[:, None] * cpu(weight_scales)
    off = 4 * SUM * y.abs()
    if bias is not None:
        y = y + cpu(bias)
        off = off + SUM * y.abs()
    return y, off + u * y.abs() + tiny

"""Performance cases of what goes around attention over voxel clouds, through the public entry points of ``FGMS.nn``:
``add_norm`` (a branch joins the residual stream, with dropout, and the sum's norm goes into the next branch),
``dropout_add``, ``quantize_rows`` and ``add_norm_int8`` (rows in 8 bits with a scale each) and ``int8_linear``
(the product of such rows with weights in 8 bits).

A case is a dict of plain values:

``op``         ``norm`` (``add_norm``), ``drop`` (``dropout_add``), ``quantize`` or ``product`` (``int8_linear``)
``grad``       whether the pass is a training step: forward, then the gradients
``dtype``      ``fp16``, ``bf16``, ``fp32``: of the features, the results and the gradients
``rows``, ``channels``

of ``norm`` and ``drop``: ``residual`` whether there is one; ``p`` the share of elements that is dropped

of ``quantize``: ``kind``, ``rows`` (the features as they are), ``gated`` (silu(a) * b of rows of twice the channels) or ``norm``
(the norm of a sum); ``out`` channels of the product that reads them, 0: none, and the rows are returned as the values they stand for

of ``product``: ``out`` channels; ``bias``
"""
import math
import random

import torch

own = False      # False: the plain forms below; True: the framework's operators

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6


def _norm(rows, channels, dtype, grad, residual=True, p=0.0):
    return dict(op="norm", rows=rows, channels=channels, dtype=dtype, grad=grad, residual=residual, p=p)


def _drop(rows, channels, dtype, grad, residual=True, p=0.1):
    return dict(op="drop", rows=rows, channels=channels, dtype=dtype, grad=grad, residual=residual, p=p)


def _quantize(kind, rows, channels, dtype, out):
    return dict(op="quantize", kind=kind, rows=rows, channels=channels, dtype=dtype, grad=False, out=out)


def _product(rows, channels, out, dtype, bias=False):
    return dict(op="product", rows=rows, channels=channels, out=out, dtype=dtype, grad=False, bias=bias)


def listed():
    named = [
        # serving: the newest row of each of eight scans
        ("norm-8-512-fp16", _norm(8, 512, "fp16", False)),
        # inference in full precision over a thinned cloud, the widest layer of a backbone
        ("norm-50k-256-fp32", _norm(50000, 256, "fp32", False)),
        # training over LiDAR sweeps, 128 channels, dropout on the branch
        ("norm-120k-128-fp16-dropout-step", _norm(120000, 128, "fp16", True, p=0.1)),
        # odd sizes: wide rows that fill no power of two, no dropout
        ("norm-10007-1096-bf16-step", _norm(10007, 1096, "bf16", True)),
        # the branch behind which no norm follows: an indoor cloud in full precision
        ("dropout-200k-64-fp32", _drop(200000, 64, "fp32", False)),
        # training over long scans with wide rows
        ("dropout-16k-4096-bf16-step", _drop(16384, 4096, "bf16", True, p=0.2)),
        # inference in 8 bits: an indoor cloud on its way into the projections
        ("quantize-200k-64-fp16-norm", _quantize("norm", 200000, 64, "fp16", 0)),
        # ... a thinned cloud and its projection to queries, keys and values
        ("quantize-50k-256-768-fp16-norm", _quantize("norm", 50000, 256, "fp16", 768)),
        # serving: gated rows of a few scans, and the product that leads back
        ("quantize-16-11008-4096-bf16-gated", _quantize("gated", 16, 11008, "bf16", 4096)),
        # the smallest: one row
        ("product-1-512-1536-fp16", _product(1, 512, 1536, "fp16")),
        # serving a few scans, wide layers: the weights' way from memory
        ("product-16-4096-11008-bf16", _product(16, 4096, 11008, "bf16")),
        # long scans at once: products
        ("product-24k-4096-11008-bf16-bias", _product(24000, 4096, 11008, "bf16", True)),
    ]
    return [dict(c, name=n) for n, c in named]


def _spread(rng, low, high):
    """A whole number between them, even over the logarithm, any remainder as likely as any other."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def _cost(case):
    w = work(case)
    elements = case["rows"] * case["channels"]
    return w["flops"] / 1e15 + (w["bytes"] + 8 * elements) / 4e12


def draw(rng):
    ceiling = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(("norm", "norm", "drop", "quantize", "product", "product"))
        dtype = rng.choice(("fp16", "bf16", "fp32") if op in ("norm", "drop") else ("fp16", "bf16"))
        rows, channels = _spread(rng, 1, 200000), _spread(rng, 8, 8192)
        if rng.random() < 0.75:      # layers are wide by eights
            channels = (channels + 7) // 8 * 8
        if op == "norm":
            case = _norm(rows, channels, dtype, rng.random() < 0.5, rng.random() < 0.8, rng.choice((0.0, 0.1, 0.3)))
        elif op == "drop":
            case = _drop(rows, channels, dtype, rng.random() < 0.5, rng.random() < 0.8, rng.choice((0.05, 0.1, 0.5)))
        elif op == "quantize":
            case = _quantize(rng.choice(("rows", "gated", "norm")), rows, channels, dtype, rng.choice((0, 0, _spread(rng, 8, 8192))))
        else:
            case = _product(rows, channels, _spread(rng, 8, 11008), dtype, rng.random() < 0.5)
        if rows * channels <= 1 << 26 and rows * case.get("out", 1) <= 24000 * 11008 and _cost(case) <= ceiling:
            return case


# ------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, n, c = _TYPES[case["dtype"]], case["rows"], case["channels"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    def leaf(t):
        return t.requires_grad_(case["grad"])

    def eighths(rows, width):
        """Rows in 8 bits as a program keeps them: each begins on 16 bytes; their scales."""
        v = torch.randn(rows, width, generator=gen, device="cuda")
        scales = v.abs().amax(1) / 127
        held = torch.zeros(rows, (width + 15) // 16 * 16, dtype=torch.int8, device="cuda")
        held[:, :width] = torch.round(v / scales[:, None]).to(torch.int8)
        return held[:, :width], scales

    s = dict(op=case["op"], grad=case["grad"], dtype=dtype)
    if case["op"] in ("norm", "drop"):
        s.update(x=leaf(normal(n, c)), residual=leaf(2 * normal(n, c)) if case["residual"] else None, p=case["p"],
                 # what the generator's words depend on: a new one for every pass of a program
                 seed=torch.randint(-1 << 62, 1 << 62, (2,), generator=gen, device="cuda"))
        if case["op"] == "norm":
            s["scale"] = leaf((1 + 0.1 * torch.randn(c, generator=gen, device="cuda")).to(dtype))
        if case["grad"]:
            s["gy"] = normal(n, c)
            if case["op"] == "norm" and (case["residual"] or case["p"]):
                s["gh"] = normal(n, c)
        return s
    if case["op"] == "quantize":
        s.update(kind=case["kind"], x=normal(n, (2 if case["kind"] == "gated" else 1) * c))
        if case["kind"] == "norm":
            s.update(residual=2 * normal(n, c), scale=(1 + 0.1 * torch.randn(c, generator=gen, device="cuda")).to(dtype))
    else:
        s["q"], s["scales"] = eighths(n, c)
    if case["out"]:
        s["weight"], s["weight_scales"] = eighths(case["out"], c)
        s["weight_scales"] = s["weight_scales"] / math.sqrt(c)
        s["bias"] = normal(case["out"]) if case.get("bias") else None
    return s


# ------------------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return {"norm": _norm_plain, "drop": _drop_plain, "quantize": _quantize_plain, "product": _product_plain}[s["op"]](s)
    from FGMS import nn
    if s["op"] == "product":
        return nn.int8_linear(s["q"], s["scales"], s["weight"], s["weight_scales"], s["bias"], dtype=s["dtype"])
    if s["op"] == "quantize":
        h = ()
        if s["kind"] == "norm":
            q, scales, *h = nn.add_norm_int8(s["x"], s["residual"], s["scale"], eps=_EPS)
        else:
            q, scales = nn.quantize_rows(s["x"], gated=s["kind"] == "gated")
        if "weight" in s:
            return (nn.int8_linear(q, scales, s["weight"], s["weight_scales"], dtype=s["dtype"]), *h)
        values = torch.empty(q.shape, dtype=s["dtype"], device=q.device)
        return (torch.mul(q, scales[:, None], out=values), scales, *h)
    with torch.set_grad_enabled(s["grad"]):
        if s["op"] == "drop":
            out = (nn.dropout_add(s["x"], s["residual"], p=s["p"], seed=s["seed"]),)
        else:
            out = nn.add_norm(s["x"], s["residual"], s["scale"], eps=_EPS, p=s["p"], seed=s["seed"])
            if s["residual"] is None and not s["p"]:      # (the sum is x)
                out = out[:1]
    if not s["grad"]:
        return out
    inputs = [t for t in (s["x"], s["residual"], s.get("scale")) if t is not None]
    got = torch.autograd.grad(out, inputs, [s["gy"], s["gh"]] if len(out) > 1 else [s["gy"]])
    return tuple(t.detach() for t in out) + tuple(got)


_LOW = 0xFFFFFFFF


def _kept(s):
    """Where an element stays: Philox4x32-10 (Salmon, Moraes, Dror, Shaw, SC 2011), eight words of 16 bits a call."""
    n, c = s["x"].shape
    per = (c + 7) // 8
    counter = torch.arange(n * per, device="cuda")
    a, b = counter & _LOW, counter >> 32
    x, y = (s["seed"][1] & _LOW).expand_as(a), (s["seed"][1] >> 32 & _LOW).expand_as(a)
    k, m = s["seed"][0] & _LOW, s["seed"][0] >> 32 & _LOW
    for _ in range(10):
        p, q = a * 0xD2511F53, x * 0xCD9E8D57
        a, b, x, y = (q >> 32 & _LOW) ^ b ^ k, q & _LOW, (p >> 32 & _LOW) ^ y ^ m, p & _LOW
        k, m = k + 0x9E3779B9 & _LOW, m + 0xBB67AE85 & _LOW
    words = torch.stack([t >> d & 0xFFFF for t in (a, b, x, y) for d in (0, 16)], 1)
    return words.view(n, per * 8)[:, :c] >= round(s["p"] * 65536)


def _back(s):
    return 65536 / (65536 - round(s["p"] * 65536))


def _drop_plain(s):
    with torch.no_grad():
        kept, back = _kept(s), _back(s)
        h = torch.where(kept, s["x"].float() * back, 0.0)
        if s["residual"] is not None:
            h = h + s["residual"].float()
        out = [h]
        if s["grad"]:
            g = s["gy"].float()
            out.append(torch.where(kept, g * back, 0.0))
            if s["residual"] is not None:
                out.append(g)
        return tuple(t.to(s["dtype"]) for t in out)


def _norm_plain(s):
    with torch.no_grad():
        h, kept = s["x"].float(), None
        if s["p"]:
            kept, back = _kept(s), _back(s)
            h = torch.where(kept, h * back, 0.0)
        if s["residual"] is not None:
            h = h + s["residual"].float()
        h = h.to(s["dtype"]).float()      # (the sum is a result: its norm is taken of what is stored)
        w = s["scale"].float()
        r = 1.0 / torch.sqrt((h * h).mean(1, keepdim=True) + _EPS)
        out = [h * r * w]
        if kept is not None or s["residual"] is not None:
            out.append(h)
        if s["grad"]:
            g = s["gy"].float()
            wg = w * g
            gs = r * (wg - h * r * r * (wg * h).mean(1, keepdim=True))
            if len(out) > 1:
                gs = gs + s["gh"].float()
            out.append(gs if kept is None else torch.where(kept, gs * back, 0.0))
            if s["residual"] is not None:
                out.append(gs)
            out.append((g * h * r).sum(0))
        return tuple(t.to(s["dtype"]) for t in out)


def _quantize_plain(s):
    x, more = s["x"].float(), ()
    if s["kind"] == "gated":
        a, b = x.chunk(2, 1)
        x = a / (1.0 + torch.exp(-a)) * b
    elif s["kind"] == "norm":
        h = (x + s["residual"].float()).to(s["dtype"])
        more = (h,)
        x = h.float()
        x = x / torch.sqrt((x * x).mean(1, keepdim=True) + _EPS) * s["scale"].float()
    scales = x.abs().amax(1, keepdim=True) / 127
    q = torch.round(x / torch.where(scales > 0, scales, 1.0))
    if "weight" in s:
        return (((q @ s["weight"].float().t()) * scales * s["weight_scales"]).to(s["dtype"]), *more)
    return ((q * scales).to(s["dtype"]), scales[:, 0], *more)


def _product_plain(s):
    y = (s["q"].float() @ s["weight"].float().t()) * s["scales"][:, None] * s["weight_scales"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["dtype"])


# ------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"norm": _norm_exact, "drop": _drop_exact, "quantize": _quantize_exact, "product": _product_exact}[s["op"]](s, case)


def _times(a, factor):
    """(upper, lower) 32 bits of a product of two 32-bit numbers, by 16-bit halves"""
    low, high = a % 65536, a // 65536
    f, g = factor % 65536, factor // 65536
    middle = low * g + high * f + low * f // 65536
    return (high * g + middle // 65536) % (1 << 32), (middle % 65536) * 65536 + low * f % 65536


def _factor(case, s):
    """What each element of a branch is multiplied with, in 64 bits"""
    n, c = case["rows"], case["channels"]
    chunks = -(-c // 8)
    key, stream = (int(v) % (1 << 64) for v in s["seed"].tolist())
    keys = [key % (1 << 32), key >> 32]
    number = torch.arange(n, device="cuda")[:, None] * chunks + torch.arange(chunks, device="cuda")
    state = [number % (1 << 32), number // (1 << 32), torch.full_like(number, stream % (1 << 32)), torch.full_like(number, stream >> 32)]
    for i in range(10):
        up0, low0 = _times(state[0], 0xD2511F53)
        up1, low1 = _times(state[2], 0xCD9E8D57)
        round_key = [(keys[0] + i * 0x9E3779B9) % (1 << 32), (keys[1] + i * 0xBB67AE85) % (1 << 32)]
        state = [up1 ^ state[1] ^ round_key[0], low1, up0 ^ state[3] ^ round_key[1], low0]
    dropped = round(case["p"] * 65536)
    factor = torch.empty(n, chunks, 8, dtype=torch.float64, device="cuda")
    for e in range(8):
        word = state[e // 2] // 65536 if e % 2 else state[e // 2] % 65536
        factor[..., e] = (word >= dropped).double() * (65536 / (65536 - dropped))
    return factor.reshape(n, chunks * 8)[:, :c]


def _drop_exact(s, case):
    factor = _factor(case, s)
    h = factor * s["x"].detach().double()
    if case["residual"]:
        h += s["residual"].detach().double()
    if not case["grad"]:
        return (h,)
    g = s["gy"].double()
    return (h, g * factor, g) if case["residual"] else (h, g * factor)


def _norm_exact(s, case):
    factor = _factor(case, s) if case["p"] else None
    x = s["x"].detach().double()
    total = x if factor is None else x * factor
    if case["residual"]:
        total = total + s["residual"].detach().double()
    total = total.to(s["dtype"]).double().requires_grad_(case["grad"])
    w = s["scale"].detach().double().requires_grad_(case["grad"])
    y = total * w * torch.rsqrt(total.square().mean(-1, keepdim=True) + _EPS)
    both = case["residual"] or factor is not None
    out = (y.detach(), total.detach()) if both else (y.detach(),)
    if not case["grad"]:
        return out
    g_total, g_scale = torch.autograd.grad(y, (total, w), s["gy"].double())
    if both:
        g_total = g_total + s["gh"].double()
    g_x = g_total if factor is None else g_total * factor
    return (*out, g_x, g_total, g_scale) if case["residual"] else (*out, g_x, g_scale)


def _eight_bits(v):
    step = v.abs().max(dim=1).values / 127
    return torch.where(step[:, None] > 0, v / step[:, None], torch.zeros_like(v)).round(), step


def _quantize_exact(s, case):
    v, more = s["x"].double(), ()
    if case["kind"] == "gated":
        c = case["channels"]
        v = v[:, :c] * torch.sigmoid(v[:, :c]) * v[:, c:]
    elif case["kind"] == "norm":
        total = (v + s["residual"].double()).to(s["dtype"]).double()
        more = (total,)
        v = total * torch.rsqrt(total.square().mean(-1, keepdim=True) + _EPS) * s["scale"].double()
    q, step = _eight_bits(v)
    if case["out"]:
        return (torch.matmul(q * step[:, None], (s["weight"].double() * s["weight_scales"].double()[:, None]).t().contiguous()), *more)
    return (q * step[:, None], step, *more)


def _product_exact(s, case):
    rows, weight = s["q"].double() * s["scales"].double()[:, None], s["weight"].double() * s["weight_scales"].double()[:, None]
    y = torch.matmul(rows, weight.t().contiguous())
    return y if s["bias"] is None else y + s["bias"].double()


# ------------------------------------------------------------------------------- what it takes
def work(case):
    """Every input read once and every output written once (a gradient that two inputs share, once); for a norm eight operations an
    element, three times that with gradients; two for each product of two channels."""
    size = 4 if case["dtype"] == "fp32" else 2
    elements = case["rows"] * case["channels"]
    if case["op"] in ("norm", "drop"):
        inputs, sums = 1 + case["residual"], bool(case["residual"] or case["p"])
        if case["op"] == "drop":
            # x, the residual, the sum; with gradients the sum's and x's
            return {"bytes": size * elements * (inputs + 1 + (2 if case["grad"] else 0)), "flops": elements * (4 if case["grad"] else 2)}
        tensors = inputs + 1 + sums
        if case["grad"]:
            tensors += 1 + sums + (2 if case["p"] and case["residual"] else 1)
        return {"bytes": size * elements * tensors, "flops": elements * (24 if case["grad"] else 8)}
    out = case["out"]
    products = 2 * elements * out
    result = out * (case["channels"] + 4) + size * case["rows"] * out if out else 0
    if case["op"] == "product":
        return {"bytes": elements + 4 * case["rows"] + result + (size * out if case["bias"] else 0), "flops": products}
    read = {"rows": 1, "gated": 2, "norm": 3}[case["kind"]]      # (the norm's sum is written)
    return {"bytes": size * elements * read + (result if out else size * elements + 4 * case["rows"]), "flops": 8 * elements + products}

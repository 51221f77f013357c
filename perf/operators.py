"""Performance cases of attention over voxel clouds, through the public entry points of ``FGMS.nn``:
``norm_rotary`` (norms of queries and keys for each head, and their rotation by the voxels' coordinates),
``segment_attention`` over ragged segments (windows of a cloud, scans, caches) and both backward passes.

A case is a dict of plain values:

``op``        ``turn`` (``norm_rotary``) or ``attend`` (``segment_attention``)
``grad``      whether the pass is a training step: forward, then the gradients
``dtype``     ``fp16``, ``bf16``, ``fp32``
``heads``, ``kv_heads``, ``dim``    query heads, key heads, channels of a head

of ``turn``: ``rows``; ``axes`` coordinates a row; ``turned`` rotated channel pairs of ``dim / 2``, shared out
among the axes; ``interleaved`` pairs (2p, 2p + 1) instead of (p, p + dim / 2)

of ``attend``: ``kind``, from which with ``total``, ``segments``, ``longest``, ``mean`` and ``spread`` the lengths follow

    ``windows``     ragged windows of a cloud of ``total`` voxels, about ``mean`` to a window
    ``sequences``   ``segments`` scans in order of time, ``total`` rows together
    ``cache``       ``queries`` newest rows each over ``segments`` caches with room for ``longest`` keys
    ``cross``       queries over the keys of another cloud, some segments without any

and ``causal``: keys behind a query are not seen (ends of queries and keys aligned).
"""
import math
import random

import torch

own = False      # False: the plain forms below; True: the framework's operators

_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
_EPS = 1e-6


def _turn(rows, heads, kv_heads, dim, dtype, axes, grad, turned=None, interleaved=False):
    return dict(op="turn", rows=rows, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, axes=axes, grad=grad,
                turned=dim // 2 if turned is None else turned, interleaved=interleaved)


def _attend(kind, heads, kv_heads, dim, dtype, grad, causal=False, total=0, segments=0, longest=0, mean=0, queries=0, spread=1):
    return dict(op="attend", kind=kind, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype, grad=grad, causal=causal,
                total=total, segments=segments, longest=longest, mean=mean, queries=queries, spread=spread)


def listed():
    named = [
        # serving: the newest row of each of a few scans
        ("turn-8-8/2x64-fp16", _turn(8, 8, 2, 64, "fp16", 4, False)),
        # inference over a thinned cloud in full precision
        ("turn-50k-8/8x32-fp32", _turn(50000, 8, 8, 32, "fp32", 3, False)),
        # training over LiDAR sweeps, 128 channels, positions in space and time
        ("turn-120k-4/4x32-fp16-step", _turn(120000, 4, 4, 32, "fp16", 4, True)),
        # odd sizes: heads of 72 channels, a pair or two unrotated, neighbours as pairs, an odd row count
        ("turn-10007-16/4x72-bf16-step", _turn(10007, 16, 4, 72, "bf16", 3, True, 34, True)),
        # an indoor cloud in windows, 64 channels: the ordinary layer of inference
        ("attend-windows-200k-4/4x16-fp16", _attend("windows", 4, 4, 16, "fp16", False, total=200000, mean=160)),
        # all voxels of long scans in order of time, wide heads in groups: products dominate
        ("attend-scans-24k-16/4x128-bf16-causal", _attend("sequences", 16, 4, 128, "bf16", False, True, total=24000, segments=2)),
        # serving: one read-out row for each of 16 scans, over long caches
        ("attend-cache-16x65536-32/4x128-fp16", _attend("cache", 32, 4, 128, "fp16", False, True, segments=16, longest=65536, queries=1)),
        # serving, the smallest: one row over a hundred keys
        ("attend-cache-1x100-8/8x64-fp16", _attend("cache", 8, 8, 64, "fp16", False, True, segments=1, longest=100, queries=1)),
        # training over windows of LiDAR sweeps, 128 channels
        ("attend-windows-120k-4/4x32-fp16-step", _attend("windows", 4, 4, 32, "fp16", True, total=120000, mean=90)),
        # training over few long scans
        ("attend-scans-12k-16/16x64-bf16-causal-step", _attend("sequences", 16, 16, 64, "bf16", True, True, total=12000, segments=3)),
        # training in full precision: objects' queries over ragged sets of voxels, heads of 40 channels
        ("attend-cross-20k-6/2x40-fp32-step", _attend("cross", 6, 2, 40, "fp32", True, total=20011, segments=37)),
    ]
    return [dict(c, name=n) for n, c in named]


def _spread(rng, low, high):
    """A whole number between them, even over the logarithm, any remainder as likely as any other."""
    return max(low, min(high, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


_RATE = {"fp16": 5e14, "bf16": 5e14, "fp32": 5e13}


def _cost(case):
    w = work(case)
    return w["flops"] / _RATE[case["dtype"]] + w["bytes"] / 4e12


def draw(rng):
    ceiling = max(_cost(c) for c in listed())
    while True:
        dtype = rng.choice(("fp16", "fp16", "bf16", "bf16", "fp32"))
        kv_heads = rng.choice((1, 2, 3, 4, 8))
        heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 8))
        dim = rng.choice((8, 16, 24, 32, 32, 40, 48, 64, 64, 72, 80, 96, 112, 128, 128))
        grad = rng.random() < 0.5
        kind = rng.choice(("turn", "turn", "windows", "sequences", "cache", "cross"))
        spread = rng.randrange(1, 1 << 20)
        if kind == "turn":
            axes = rng.randint(1, min(4, dim // 2))
            case = _turn(_spread(rng, 1, 200000), heads, kv_heads, dim, dtype, axes, grad, rng.randint(max(axes, dim // 4), dim // 2),
                         rng.random() < 0.5)
        elif kind == "windows":
            case = _attend(kind, heads, kv_heads, dim, dtype, grad, total=_spread(rng, 300, 200000), mean=_spread(rng, 8, 500), spread=spread)
        elif kind == "sequences":
            case = _attend(kind, heads, kv_heads, dim, dtype, grad, rng.random() < 0.7, total=_spread(rng, 100, 16000),
                           segments=rng.randint(1, 6), spread=spread)
        elif kind == "cache":
            case = _attend(kind, heads, kv_heads, dim, dtype, False, True, segments=_spread(rng, 1, 64), longest=_spread(rng, 16, 65536),
                           queries=rng.choice((1, 1, 1, 2, 5)), spread=spread)
        else:
            case = _attend(kind, heads, kv_heads, dim, dtype, grad, total=_spread(rng, 300, 40000), segments=_spread(rng, 1, 100), spread=spread)
        if _cost(case) <= ceiling:
            return case


def _shares(rng, total, parts):
    weights = [rng.uniform(0.3, 2.0) for _ in range(parts)]
    sizes = [int(total * w / sum(weights)) for w in weights]
    sizes[-1] += total - sum(sizes)
    return sizes


def _lengths(case):
    """(queries of each segment, keys of each, rows that each has room for among the keys)"""
    rng = random.Random(case["spread"])
    kind, total = case["kind"], case["total"]
    if kind == "windows":
        sizes, left = [], total
        while left:
            n = max(1, min(left, int(case["mean"] * rng.lognormvariate(-0.18, 0.6))))
            sizes.append(n)
            left -= n
        return sizes, sizes, sizes
    if kind == "sequences":
        sizes = _shares(rng, total, case["segments"])
        return sizes, sizes, sizes
    if kind == "cache":
        used = [rng.randint(max(case["queries"], case["longest"] // 16), max(case["queries"], case["longest"])) for _ in range(case["segments"])]
        used[0] = max(case["queries"], case["longest"])
        return [case["queries"]] * len(used), used, [used[0]] * len(used)
    queries, keys = _shares(rng, total // 3, case["segments"]), _shares(rng, total, case["segments"])
    if len(keys) > 2:      # a segment without keys, and one without queries
        keys[1] = 0
        queries[2] = 0
    return queries, keys, keys


# ------------------------------------------------------------------------------- inputs
def _starts(sizes):
    starts = [0]
    for n in sizes:
        starts.append(starts[-1] + n)
    return starts


def _sections(case):
    """Rotated pairs of each axis: equal shares, what is left over to the first ones."""
    turned, axes = case["turned"], case["axes"]
    return tuple(turned // axes + (a < turned % axes) for a in range(axes))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype, h, hk, d = _TYPES[case["dtype"]], case["heads"], case["kv_heads"], case["dim"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda").to(dtype)

    def leaf(t):
        return t.detach().requires_grad_(case["grad"])

    s = dict(op=case["op"], grad=case["grad"])
    if case["op"] == "turn":
        n, sections = case["rows"], _sections(case)
        # queries, keys and values side by side, as one projection leaves them
        qkv = normal(n, (h + 2 * hk) * d)
        s.update(q=leaf(qkv[:, :h * d].unflatten(1, (h, d))), k=leaf(qkv[:, h * d:(h + hk) * d].unflatten(1, (hk, d))),
                 q_scale=leaf((1 + 0.1 * normal(d)).to(dtype)), k_scale=leaf((1 + 0.1 * normal(d)).to(dtype)),
                 # voxels of a scene some hundreds of cells wide, moving with the sensor; the last axis is low
                 coords=torch.randint(-300, 700, (n, case["axes"]), generator=gen, device="cuda", dtype=torch.int32),
                 freqs=torch.cat([100.0 ** (-torch.arange(c, dtype=torch.float32) / c) for c in sections]).cuda(),
                 sections=sections, interleaved=case["interleaved"])
        s["coords"][:, -1] %= 64
        if case["grad"]:
            s.update(gq=normal(n, h, d), gk=normal(n, hk, d))
        return s
    queries, keys, room = _lengths(case)
    nq, nk = sum(queries), sum(room)
    if case["kind"] in ("windows", "sequences"):
        qkv = normal(nq, (h + 2 * hk) * d)
        q, k, v = (t.unflatten(1, (-1, d)) for t in qkv.split((h * d, hk * d, hk * d), 1))
    else:
        q, k, v = normal(nq, h, d), normal(nk, hk, d), normal(nk, hk, d)
    s.update(q=leaf(q), k=leaf(k), v=leaf(v), causal=case["causal"], queries=queries, keys=keys, room=room,
             q_offsets=torch.tensor(_starts(queries), dtype=torch.int32, device="cuda"),
             k_offsets=torch.tensor(_starts(room), dtype=torch.int32, device="cuda"),
             k_lengths=torch.tensor(keys, dtype=torch.int32, device="cuda") if case["kind"] == "cache" else None)
    if case["grad"]:
        s["g"] = normal(nq, h, d)
    return s


# ------------------------------------------------------------------------------- one pass
def run(s):
    if not own:
        return (_turn_plain if s["op"] == "turn" else _attend_plain)(s)
    from FGMS import nn
    with torch.set_grad_enabled(s["grad"]):
        if s["op"] == "turn":
            out = nn.norm_rotary(s["q"], s["k"], s["q_scale"], s["k_scale"], s["coords"], s["freqs"], s["sections"],
                                 eps=_EPS, interleaved=s["interleaved"])
            inputs, grads = ("q", "k", "q_scale", "k_scale"), ("gq", "gk")
        else:
            out = (nn.segment_attention(s["q"], s["k"], s["v"], s["q_offsets"], s["k_offsets"], causal=s["causal"],
                                        k_lengths=s["k_lengths"]),)
            inputs, grads = ("q", "k", "v"), ("g",)
    if not s["grad"]:
        return tuple(out)
    got = torch.autograd.grad(out, [s[i] for i in inputs], [s[g] for g in grads])
    return tuple(t.detach() for t in out) + tuple(got)


def _angles(s):
    axis = [a for a, c in enumerate(s["sections"]) for _ in range(c)]
    return s["coords"].float()[:, axis] * s["freqs"]


def _halves(x, turned, interleaved):
    """(first channels of the rotated pairs, second ones)"""
    d = x.shape[-1]
    return (x[..., 0:2 * turned:2], x[..., 1:2 * turned:2]) if interleaved else (x[..., :turned], x[..., d // 2:d // 2 + turned])


def _rotate(x, cos, sin, interleaved):
    y = x.clone()
    a, b = _halves(x, cos.shape[-1], interleaved)
    ya, yb = _halves(y, cos.shape[-1], interleaved)
    ya.copy_(a * cos - b * sin)
    yb.copy_(a * sin + b * cos)
    return y


def _turn_plain(s):
    phi = _angles(s)
    cos, sin = phi.cos()[:, None], phi.sin()[:, None]
    out, grads, scale_grads = [], [], []
    with torch.no_grad():
        for name in ("q", "k"):
            x, w = s[name].float(), s[name + "_scale"].float()
            r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + _EPS)
            out.append(_rotate(x * r * w, cos, sin, s["interleaved"]).to(s[name].dtype))
            if s["grad"]:
                h = _rotate(s["g" + name].float(), cos, -sin, s["interleaved"])
                scale_grads.append((h * x * r).sum((0, 1)).to(s[name].dtype))
                wh = w * h
                grads.append((r * (wh - x * r * r * (wh * x).mean(-1, keepdim=True))).to(s[name].dtype))
    return tuple(out + grads + scale_grads)


def _blocks(s, limit):
    """Blocks of segments of like lengths, cut into ranges of queries where one alone has more than `limit` scores."""
    heads = s["q"].shape[1]
    order = sorted((i for i in range(len(s["keys"])) if s["keys"][i] and s["queries"][i]), key=lambda i: (s["keys"][i], s["queries"][i]))
    block, widest = [], 0
    for i in order:
        rows = max(widest, s["queries"][i])
        if block and (len(block) + 1) * heads * rows * s["keys"][i] > limit:
            yield block, 0, widest
            block, rows = [], s["queries"][i]
        block.append(i)
        widest = rows
        if len(block) == 1 and heads * rows * s["keys"][i] > limit:
            step = max(1, limit // (heads * s["keys"][i]))
            for first in range(0, rows, step):
                yield block, first, min(first + step, rows)
            block, widest = [], 0
    if block:
        yield block, 0, widest


def _attend_plain(s):
    dev, dtype = s["q"].device, s["q"].dtype
    q, k, v = (s[n].detach().float() for n in ("q", "k", "v"))
    (nq, h, d), hk = q.shape, k.shape[1]
    g = h // hk
    scale = 1.0 / math.sqrt(d)
    out = torch.zeros_like(q)
    if s["grad"]:
        go = s["g"].float()
        gq, gk, gv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    q_start, k_start = _starts(s["queries"]), _starts(s["room"])
    for block, first, last in _blocks(s, 1 << 28):
        b = len(block)
        qs, ql, ks, kl = (torch.tensor([t[i] for i in block], device=dev)[:, None] for t in (q_start, s["queries"], k_start, s["keys"]))
        i, j = torch.arange(first, last, device=dev)[None], torch.arange(max(s["keys"][x] for x in block), device=dev)[None]
        rows, cols = torch.where(i < ql, qs + i, 0).flatten(), torch.where(j < kl, ks + j, 0).flatten()
        there = (i < ql).flatten()[:, None, None]
        ni, nj = i.shape[1], j.shape[1]

        def by_query(t):      # [rows, heads, d] -> [b * hk, g * ni, d]
            return t[rows].reshape(b, ni, hk, g, d).permute(0, 2, 3, 1, 4).reshape(b * hk, g * ni, d)

        def by_key(t):
            return t[cols].reshape(b, nj, hk, d).permute(0, 2, 1, 3).reshape(b * hk, nj, d)

        def query_rows(t):
            return t.reshape(b, hk, g, ni, d).permute(0, 3, 1, 2, 4).reshape(b * ni, h, d)

        def key_rows(t):
            return t.reshape(b, hk, nj, d).permute(0, 2, 1, 3).reshape(b * nj, hk, d)

        bq, bk, bv = by_query(q), by_key(k), by_key(v)
        p = torch.bmm(bq, bk.transpose(1, 2).contiguous()).mul_(scale).view(b, hk * g, ni, nj)
        seen = (i < ql)[:, :, None] & (j < kl)[:, None, :]
        if s["causal"]:
            seen = seen & (j[:, None, :] - (kl - ql)[:, :, None] <= i[:, :, None])
        p.masked_fill_(~seen[:, None], -math.inf)
        most = p.amax(-1, keepdim=True)
        p.sub_(torch.where(most == -math.inf, 0.0, most)).exp_()
        total = p.sum(-1, keepdim=True)
        p.div_(torch.where(total > 0, total, 1.0))
        p = p.view(b * hk, g * ni, nj)
        o = torch.bmm(p, bv)
        out.index_add_(0, rows, query_rows(o) * there)
        if s["grad"]:
            bg = by_query(go)
            gv.index_add_(0, cols, key_rows(torch.bmm(p.transpose(1, 2).contiguous(), bg)))
            ds = torch.bmm(bg, bv.transpose(1, 2).contiguous()).sub_((bg * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
            gq.index_add_(0, rows, query_rows(torch.bmm(ds, bk)) * there)
            gk.index_add_(0, cols, key_rows(torch.bmm(ds.transpose(1, 2).contiguous(), bq)))
    outs = (out, gq, gk, gv) if s["grad"] else (out,)
    return tuple(t.to(dtype) for t in outs)


# ------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return _turn_exact(s) if case["op"] == "turn" else _attend_exact(s)


def _turn_exact(s):
    axis = torch.tensor([a for a, c in enumerate(s["sections"]) for _ in range(c)], device="cuda")
    phi = s["coords"].double().index_select(1, axis) * s["freqs"].double()
    turn = torch.polar(torch.ones_like(phi), phi)[:, None]      # a pair as a complex number, turned by phi
    pairs = phi.shape[1]
    results, leaves, upstream = [], [], []
    for name in ("q", "k"):
        x = s[name].detach().double().requires_grad_(s["grad"])
        w = s[name + "_scale"].detach().double().requires_grad_(s["grad"])
        z = w * x / torch.sqrt(torch.mean(x ** 2, -1, keepdim=True) + _EPS)
        n, h, d = z.shape
        two = z.reshape(n, h, d // 2, 2) if s["interleaved"] else torch.stack((z[..., :d // 2], z[..., d // 2:]), -1)
        c = torch.view_as_complex(two.contiguous())
        two = torch.view_as_real(torch.cat((c[..., :pairs] * turn, c[..., pairs:]), -1))
        results.append(two.reshape(n, h, d) if s["interleaved"] else torch.cat((two[..., 0], two[..., 1]), -1))
        leaves.append((x, w))
        if s["grad"]:
            upstream.append(s["g" + name].double())
    if not s["grad"]:
        return tuple(results)
    got = torch.autograd.grad(results, [leaves[0][0], leaves[1][0], leaves[0][1], leaves[1][1]], upstream)
    return tuple(t.detach() for t in results) + tuple(got)


def _attend_exact(s):
    h, d = s["q"].shape[1:]
    g = h // s["k"].shape[1]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    grads = [torch.zeros(s[n].shape, dtype=torch.float64, device="cuda") for n in "qkv"] if s["grad"] else []
    q0 = k0 = 0
    for nq, nk, room in zip(s["queries"], s["keys"], s["room"]):
        if nq and nk:
            block = max(1, (1 << 28) // (h * nk))
            k, v = (s[n].detach()[k0:k0 + nk].double().requires_grad_(s["grad"]) for n in "kv")
            for first in range(0, nq, block):
                rows = slice(q0 + first, q0 + min(first + block, nq))
                q = s["q"].detach()[rows].double().requires_grad_(s["grad"])
                kh, vh = (t.repeat_interleave(g, 1).permute(1, 2, 0).contiguous() for t in (k, v))      # [h, d, nk]
                score = q.transpose(0, 1) @ kh / math.sqrt(d)
                if s["causal"]:
                    position = torch.arange(first, first + q.shape[0], device="cuda") + nk - nq
                    hidden = torch.arange(nk, device="cuda")[None] > position[:, None]
                    score = score.masked_fill(hidden, -math.inf)
                    p = torch.softmax(score, -1).masked_fill(hidden.all(1)[None, :, None], 0.0)
                else:
                    p = torch.softmax(score, -1)
                o = (p @ vh.transpose(1, 2).contiguous()).transpose(0, 1)
                out[rows] = o.detach()
                if s["grad"]:
                    part = torch.autograd.grad(o, (q, k, v), s["g"][rows].double())
                    grads[0][rows] += part[0]
                    grads[1][k0:k0 + nk] += part[1]
                    grads[2][k0:k0 + nk] += part[2]
        q0 += nq
        k0 += room
    return (out, *grads)


# ------------------------------------------------------------------------------- what it takes
def work(case):
    """Every input read once and every output written once (a training step's forward results and what both passes
    read, once); ten operations an element for a norm and a turn, three times that with gradients; two for each
    product of two channels: two products a seen (query, key) forward, five more backward, which forms its scores anew."""
    size = 4 if case["dtype"] == "fp32" else 2
    h, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "turn":
        elements = case["rows"] * (h + hk) * d
        return {"bytes": size * elements * (4 if case["grad"] else 2) + 4 * case["rows"] * case["axes"], "flops": elements * (30 if case["grad"] else 10)}
    queries, keys, _ = _lengths(case)
    seen = 0
    for nq, nk in zip(queries, keys):
        if not case["causal"]:
            seen += nq * nk
        else:      # query i sees keys 0 .. i + nk - nq
            least = nk - nq + 1
            rows = nq if least > 0 else nk
            seen += rows * (max(least, 1) + nk) // 2
    q, kv = sum(queries) * h * d, 2 * sum(keys) * hk * d
    return {"bytes": size * ((4 * q + 2 * kv) if case["grad"] else (2 * q + kv)), "flops": (14 if case["grad"] else 4) * d * h * seen}

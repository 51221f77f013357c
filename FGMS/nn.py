"""Autograd wrapper over ``FGMS.backend``: the caller side that hkeee21/FGMS leaves to
an external library (``README.md:3``).  It owns exactly what the reference's scripts
repeat by hand before every call: the padded offset table ``qkpos``
(``cpu-check.py:6-14``), the outputs (``cpu-check.py:107-108``,
``cpu-check-back.py:104-107``) and the pairing of the forward call with the backward one
(``spconv-test.py:96-120``), as one native autograd node (``FGMS.backend.sparse_conv``).

    y = sparse_conv(feats, weight, kmap)          # differentiable in feats and weight
    layer = SparseConv(64, 64, k_vol=27); y = layer(feats, kmap)

``kmap`` is a :class:`KernelMap`: the pair lists of one kernel map on the device.  Every
layer, pass and iteration that shares a map shares its plan through ``FGMS.backend``'s
cache, which is keyed on these tensors.
"""
import math
import threading

import numpy as np
import torch

from . import backend
from fgms_amd.harness import kpos_quantized

_Q = 256   # padding quantum of the reference's scripts (cpu-check.py:106); advisory here


class KernelMap:
    """Pair lists of one kernel map: ``in_map[j] -> out_map[j]`` for j in
    ``[kpos[k], kpos[k+1])`` through offset k.  int32, on the device of the features."""

    def __init__(self, in_map, out_map, kernel_nnz, n_in, n_out):
        kn = torch.as_tensor(kernel_nnz, dtype=torch.int32).cpu()
        self.k_vol = int(kn.numel())
        self.kernel_nnz = kn                                        # host, as fgms_fwd_cuda wants it
        kpos = torch.zeros(self.k_vol + 1, dtype=torch.int32)
        kpos[1:] = torch.cumsum(kn, 0)
        if int(kpos[-1]) != in_map.numel() or in_map.numel() != out_map.numel():
            raise ValueError("kernel_nnz does not add up to the length of the pair lists")
        self.in_map = in_map.to(torch.int32).contiguous()
        self.out_map = out_map.to(torch.int32).contiguous()
        self.kpos = kpos.to(self.in_map.device)
        self.qkpos, self.qsum = kpos_quantized(kn, self.kpos, self.k_vol, _Q)
        self.n_in, self.n_out = int(n_in), int(n_out)

    @classmethod
    def from_coords(cls, in_coords, out_coords, offsets, stride=1):
        """Builds the map on the device from int32 voxel coordinates ``[N, 3]``: pairs
        (i, o) with ``in_coords[i] == out_coords[o] * stride + offsets[k]``, and the plan along
        with it.  Everything is queued on the stream; the first use of the map waits for it."""
        offs = torch.from_numpy(np.ascontiguousarray(np.asarray(offsets, dtype=np.int32).reshape(-1, 3)))
        m = cls.__new__(cls)
        m._on_its_way = backend.MapOnItsWay(in_coords, out_coords, offs, int(stride))
        m._lock = threading.Lock()
        m.k_vol, m.n_in, m.n_out = offs.shape[0], in_coords.shape[0], out_coords.shape[0]
        return m

    def __getattr__(self, name):
        # a map from coordinates is waited for when something first needs it
        if name in ("in_map", "out_map", "kernel_nnz", "kpos", "qkpos", "qsum") and "_lock" in self.__dict__:
            with self._lock:
                if "_on_its_way" in self.__dict__:
                    parts = self._on_its_way.finish()
                    del self._on_its_way
                    self.in_map, self.out_map, self.kernel_nnz, self.kpos, self.qkpos, self.qsum = parts
            if name in self.__dict__:
                return self.__dict__[name]
        raise AttributeError(name)

    def __getstate__(self):
        self.kpos                                                   # (copies are taken of a finished map)
        return {k: v for k, v in self.__dict__.items() if k != "_lock"}

    def transposed(self):
        """The map of the transposed convolution: the same pairs, roles swapped.  It keeps
        this map's tensors (not copies), so ``FGMS.backend`` recognises the pair lists and lets
        both maps share one plan."""
        t = KernelMap.__new__(KernelMap)
        t.k_vol, t.kernel_nnz = self.k_vol, self.kernel_nnz
        t.in_map, t.out_map = self.out_map, self.in_map
        t.kpos, t.qkpos, t.qsum = self.kpos, self.qkpos, self.qsum
        t.n_in, t.n_out = self.n_out, self.n_in
        return t


def sparse_conv(feats, weight, kmap, allow_tf32=False):
    """out[out_map[j]] += feats[in_map[j]] @ weight[k]; differentiable in feats and weight."""
    return backend.sparse_conv(feats, weight, kmap.kpos, kmap.in_map, kmap.out_map, kmap.n_in, kmap.n_out,
                               bool(allow_tf32))


class SparseConv(torch.nn.Module):
    """A sparse convolution layer over a precomputed :class:`KernelMap`.  Weights
    ``[k_vol, c_in, c_out]``, Kaiming-uniform with fan-in ``k_vol * c_in``; optional bias."""

    def __init__(self, c_in, c_out, k_vol=27, bias=False, dtype=None, device=None, allow_tf32=False):
        super().__init__()
        self.c_in, self.c_out, self.k_vol = c_in, c_out, k_vol
        self.allow_tf32 = allow_tf32
        self.weight = torch.nn.Parameter(torch.empty(k_vol, c_in, c_out, dtype=dtype, device=device))
        self.bias = torch.nn.Parameter(torch.zeros(c_out, dtype=dtype, device=device)) if bias else None
        self.reset_parameters()

    def reset_parameters(self):
        bound = 1.0 / math.sqrt(self.k_vol * self.c_in)
        with torch.no_grad():
            self.weight.uniform_(-bound, bound)
            if self.bias is not None:
                self.bias.zero_()

    def forward(self, feats, kmap):
        out = sparse_conv(feats, self.weight, kmap, self.allow_tf32)
        return out if self.bias is None else out + self.bias


# ------------------------------------------------------------------------------- attention
def rotary_freqs(sections, base=100.0, device=None):
    """Radians a step for each rotated pair of channels: ``base ** (-i / count)`` for the pairs i of every section."""
    return torch.cat([torch.empty(0)] + [base ** (-torch.arange(c, dtype=torch.float32) / c) for c in sections if c]).to(device)


def norm_rotary(q, k, q_scale, k_scale, coords, freqs, sections, eps=1e-6, interleaved=False):
    """Root-mean-square norms of queries and keys for each head and their rotation by the rows' coordinates, in one pass;
    differentiable in q, k and the scales.

    q ``[N, heads, D]``, k ``[N, key heads, D]`` (slices of one projection are read as they lie), scales ``[D]`` or None,
    coords int32 ``[N, axes]``.  The first ``sections[0]`` pairs of channels turn by ``coords[:, 0] * freqs[pair]``, the next
    ``sections[1]`` with the second axis, ...; pairs behind the last section stay.  Pair p is channels (p, p + D / 2), with
    ``interleaved`` (2p, 2p + 1).  coords and freqs must not be written to before the backward pass."""
    return backend.norm_rotary(q, k, q_scale, k_scale, coords, freqs, list(sections), float(eps), bool(interleaved))


def segment_attention(q, k, v, q_offsets, k_offsets=None, causal=False, scale=None, k_lengths=None):
    """Softmax attention inside ragged segments; differentiable in q, k and v.

    q ``[Nq, heads, D]``, k and v ``[Nk, key heads, D]``, heads a multiple of key heads.  Segment s is rows
    ``q_offsets[s]`` to ``q_offsets[s + 1]`` of q and likewise of k and v (``k_offsets``; None: the same): int32 tensors on
    the device, from which no size has to come back.  ``causal``: ends of queries and keys aligned, keys behind a query not
    seen.  A row that sees no key comes out as zeros.  Offsets must not be written to before the backward pass.  ``k_lengths``
    (int32, one a segment; no gradients): how much of each segment of k and v is in use, for caches with room left.  ``scale`` is
    positive, None: ``1 / sqrt(D)``."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1])
    return backend.segment_attention(q, k, v, q_offsets, q_offsets if k_offsets is None else k_offsets, k_lengths, bool(causal), float(scale))


def window_segments(coords, size):
    """Voxels by window: (order, offsets) so that rows ``order[offsets[s]:offsets[s + 1]]`` are the voxels of window s, cells of
    ``size`` voxels (a number, or one for each axis).  Waits for the number of windows."""
    cells = torch.div(coords, torch.as_tensor(size, device=coords.device), rounding_mode="floor")
    _, window, counts = torch.unique(cells, dim=0, return_inverse=True, return_counts=True)
    offsets = torch.zeros(counts.numel() + 1, dtype=torch.int32, device=coords.device)
    offsets[1:] = torch.cumsum(counts, 0)
    return torch.argsort(window, stable=True), offsets


class VoxelCache:
    """Keys and values of ``segments`` scans with room for ``capacity`` rows each, filled row by row."""

    def __init__(self, segments, capacity, kv_heads, dim, dtype=None, device=None):
        self.capacity = capacity
        self.k = torch.zeros(segments * capacity, kv_heads, dim, dtype=dtype, device=device)
        self.v = torch.zeros_like(self.k)
        self.offsets = torch.arange(segments + 1, dtype=torch.int32, device=device) * capacity
        self.lengths = torch.zeros(segments, dtype=torch.int32, device=device)

    @torch.no_grad()
    def append(self, k, v):
        """One new row for every scan (its values: a cache is in no graph); a full scan keeps its last row replaced."""
        rows = (self.offsets[:-1] + self.lengths.clamp(max=self.capacity - 1)).long()
        self.k.index_copy_(0, rows, k)
        self.v.index_copy_(0, rows, v)
        self.lengths.add_(1).clamp_(max=self.capacity)


class VoxelAttention(torch.nn.Module):
    """Attention among the voxels of each segment, positions by rotation: ``y = layer(feats, coords, offsets)`` with the rows
    of a segment next to each other (:func:`window_segments`), or row by row over a :class:`VoxelCache`:
    ``y = layer.step(feats, coords, cache)``.

    ``sections`` shares the ``channels / heads / 2`` pairs of a head out among the coordinates' axes."""

    def __init__(self, channels, heads, kv_heads=None, sections=None, base=100.0, causal=False, dtype=None, device=None):
        super().__init__()
        self.heads, self.kv_heads, self.causal = heads, kv_heads or heads, causal
        if heads < 1 or self.kv_heads < 1 or channels % heads or heads % self.kv_heads:
            raise ValueError("channels must be a multiple of heads, and heads of kv_heads")
        self.dim = channels // heads
        if self.dim % 8 or not 8 <= self.dim <= 128:
            raise ValueError("the channels of a head, channels / heads, must be a multiple of 8 from 8 to 128")
        pairs = self.dim // 2
        self.sections = tuple(sections) if sections is not None else (pairs - 2 * (pairs // 3), pairs // 3, pairs // 3)
        if not 1 <= len(self.sections) <= 4 or min(self.sections) < 0 or sum(self.sections) > pairs:
            raise ValueError("sections must be one to four shares of the %d pairs of a head" % pairs)
        self.qkv = torch.nn.Linear(channels, (heads + 2 * self.kv_heads) * self.dim, bias=False, dtype=dtype, device=device)
        self.q_scale = torch.nn.Parameter(torch.ones(self.dim, dtype=dtype, device=device))
        self.k_scale = torch.nn.Parameter(torch.ones(self.dim, dtype=dtype, device=device))
        self.out = torch.nn.Linear(channels, channels, bias=False, dtype=dtype, device=device)
        # (angles stay fp32 whatever the layer is cast to)
        self._freqs = rotary_freqs(self.sections, base)

    def _heads(self, feats, coords):
        h, hk, d = self.heads, self.kv_heads, self.dim
        q, k, v = (t.unflatten(-1, (-1, d)) for t in self.qkv(feats).split((h * d, hk * d, hk * d), -1))
        if self._freqs.device != feats.device:
            self._freqs = self._freqs.to(feats.device)
        q, k = norm_rotary(q, k, self.q_scale, self.k_scale, coords, self._freqs, self.sections)
        return q, k, v

    def forward(self, feats, coords, offsets):
        q, k, v = self._heads(feats, coords)
        return self.out(segment_attention(q, k, v, offsets, causal=self.causal).flatten(1))

    def step(self, feats, coords, cache):
        """One new row of every scan: its keys and values join the cache, its query sees all of them.  There are no gradients over
        caches: call it under ``torch.no_grad()`` where the layer or the rows ask for some."""
        if torch.is_grad_enabled() and (feats.requires_grad or any(p.requires_grad for p in self.parameters())):
            raise ValueError("a step over a cache has no gradients: call it under torch.no_grad()")
        q, k, v = self._heads(feats, coords)
        cache.append(k, v)
        ones = torch.arange(feats.shape[0] + 1, dtype=torch.int32, device=feats.device)
        y = segment_attention(q, cache.k, cache.v, ones, cache.offsets, k_lengths=cache.lengths)
        return self.out(y.flatten(1))

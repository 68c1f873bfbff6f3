"""A paged cache on numpy arrays: pools, tables, the C-ABI calls, and the rotation in 64 bits."""
from __future__ import annotations

import ctypes

import numpy as np

from attention_util import Placed, ints, layouts, pointers
from trs_backend import abi
from trs_backend.abi import DeviceArray, contiguous_strides, layout_of

BF16, F32 = abi.PAGES_BF16, abi.PAGES_F32


def bf16_bits(x):
    """float32 to bfloat16's bits, to the nearest, ties to even (NaN stays one)."""
    u = np.ascontiguousarray(x, np.float32).view(np.uint32)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) >> 16).astype(np.uint16)
    return np.where(np.isnan(x), np.uint16(0x7FC0), r)


def bf16_values(bits):
    return (bits.astype(np.uint32) << 16).view(np.float32)


def held(x, kind):
    """What pages hold of x."""
    return bf16_values(bf16_bits(x)) if kind == BF16 else np.asarray(x, np.float32)


class Cache:
    """Pools whose pages go to sequences in a random order, as views of device memory.

    `form`: "heads" [page, head, token, dim], "tokens" [page, token, head, dim],
    "both" [page, 2, head, token, dim] in one buffer, "odd" rows one entry longer than
    dim at an odd offset.  Everything that no sequence has is NaN.  keys and values:
    [batch, head, token, dim] of which sequence b has the first lengths[b] (or None).
    The first `shared` tokens of the others are not in their own pages: rows behind the
    first hold `elsewhere` for the pages that are shared as a whole."""

    def __init__(self, batch, heads, page, dim, lengths, kind=F32, form="heads", keys=None, values=None, shared=0, width=None, extra=2, seed=0,
                 elsewhere=-1, written=None):
        rng = np.random.default_rng(seed)
        self.kind, self.page, self.lengths, self.shared = kind, page, list(lengths), shared
        width = max([-(-n // page) for n in lengths] + [0]) if width is None else width
        whole = shared // page
        # The first row has the shared tokens' pages however few of them are its own sequence's.
        has = [min(max(n, shared if b == 0 and any(m > 0 for m in lengths) else 0, 0), width * page) for b, n in enumerate(lengths)]
        has = [min(n, keys.shape[2]) if keys is not None and n > lengths[b] else n for b, n in enumerate(has)]
        count = sum(-(-n // page) for n in has) + extra
        free = iter(rng.permutation(count))
        self.table = np.full((batch, width), -1, np.int32)
        for b, n in enumerate(has):
            for i in range(-(-n // page)):
                if b > 0 and i < whole:
                    self.table[b, i] = elsewhere
                else:
                    self.table[b, i] = next(free)
        self.shape = (count, heads, page, dim)
        strides = {"heads": (heads * page * dim, page * dim, dim, 1), "tokens": (page * heads * dim, dim, heads * dim, 1),
                   "both": (2 * heads * page * dim, page * dim, dim, 1), "odd": (heads * page * (dim + 1), page * (dim + 1), dim + 1, 1)}[form]
        offset = 3 if form == "odd" else 0
        size = count * strides[0] + offset
        dtype = np.uint16 if kind == BF16 else np.float32
        nan = np.uint16(0x7FC0) if kind == BF16 else np.float32(np.nan)
        # The pools' elements as they lie in memory.
        self.host = [np.full(size, nan, dtype) for _ in range(1 if form == "both" else 2)]
        self.form, self.strides = form, strides
        self.offsets = (0, heads * page * dim) if form == "both" else (offset, offset)
        for which, x in enumerate((keys, values)):
            if x is None:
                continue
            view = self.view(which)
            for b, n in enumerate(has):
                for t in range(n):
                    if written is not None and t not in written:
                        continue
                    at = self.table[0 if t < shared else b, t // page]
                    view[at, :, t % page] = bf16_bits(x[b, :, t]) if kind == BF16 else x[b, :, t]
        self.dev = [DeviceArray.from_numpy(h) for h in self.host]
        self.table_dev = ints(self.table if self.table.size else np.zeros(1, np.int32))
        self.lengths_dev = ints(np.asarray(lengths if len(lengths) else [0], np.int32))
        self.struct = abi.PagedCache(
            k=self.dev[0].addr, v=self.dev[-1].addr, lk=layout_of(self.shape, strides, self.offsets[0]),
            lv=layout_of(self.shape, strides, self.offsets[1]), type=kind, table=self.table_dev.addr, table_width=width, lengths=self.lengths_dev.addr)

    def view(self, which):
        flat = self.host[which % len(self.host)][self.offsets[which]:]
        return np.lib.stride_tricks.as_strided(flat, self.shape, tuple(s * flat.itemsize for s in self.strides))

    def fetch(self):
        """The pools from the device: [page, head, token, dim] each, as the values that they stand for."""
        for i, d in enumerate(self.dev):
            self.host[i] = d.to_numpy(self.host[i].dtype)
        out = [self.view(i).copy() for i in range(2)]
        return [bf16_values(x) if self.kind == BF16 else x for x in out]

    @property
    def ref(self):
        return ctypes.byref(self.struct)


# ---- the rotation -----------------------------------------------------------

def turned(x, cos, sin, positions, pair_axes, interleaved, inverse=False):
    """x [batch, head, token, dim] turned, in 64 bits; positions [axes, batch, token]."""
    x = x.astype(np.float64)
    pairs = cos.shape[1]
    j = np.arange(pairs)
    first, second = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    axes = np.asarray(pair_axes if pair_axes is not None else np.zeros(pairs, int), int)
    at = np.moveaxis(np.asarray(positions)[axes], 0, -1).reshape(x.shape[0], x.shape[2], pairs)  # [batch, token, pair]
    known = (at >= 0) & (at < cos.shape[0])
    row = np.where(known, at, 0)
    if cos.shape[0] == 0:
        c = s = np.full(at.shape, np.nan)
    else:
        c, s = (np.where(known, t.astype(np.float64)[row, j], np.nan) for t in (cos, sin))
    c, s = c[:, None], (-s if inverse else s)[:, None]
    y = x.copy()
    y[..., first] = x[..., first] * c - x[..., second] * s
    y[..., second] = x[..., second] * c + x[..., first] * s
    return y


def turned_bound(x, pairs, interleaved):
    """Two products and a sum, each rounded once: 3/2 ulp of the magnitudes' sum, and of the least float each."""
    x = abs(x.astype(np.float64))
    j = np.arange(pairs)
    first, second = (2 * j, 2 * j + 1) if interleaved else (j, j + pairs)
    bound = np.zeros_like(x)
    both = 2 * 2.0 ** -24 * (x[..., first] + x[..., second]) * 1.0001 + 3 * 2.0 ** -149
    bound[..., first] = bound[..., second] = both
    return bound


def rope(xs, cos, sin, interleaved, axes, pair_axes, positions, start, inverse, outs):
    """The status of the call; tensors are Placed, positions a DeviceArray or None."""
    return abi.lib.trs_rope_axes_f32(len(xs), pointers([x.dev for x in xs]), layouts(xs), cos.dev.ptr, sin.dev.ptr, ctypes.byref(cos.layout),
                                     int(interleaved), axes, None if pair_axes is None else bytes(pair_axes),
                                     None if positions is None else positions.ptr, start, int(inverse), pointers([o.dev for o in outs]), layouts(outs))


def append(cache, k, v, q=None, q_out=None, cos=None, sin=None, interleaved=False, axes=1, pair_axes=None, positions=None):
    none = (None, None)
    tables = (None, None, None) if cos is None else (cos.dev.ptr, sin.dev.ptr, ctypes.byref(cos.layout))
    return abi.lib.trs_paged_append_f32(cache.ref if isinstance(cache, Cache) else cache, *k.arg, *v.arg, *(none if q is None else q.arg),
                                        *(none if q_out is None else q_out.arg), *tables, int(interleaved), axes,
                                        None if pair_axes is None else bytes(pair_axes), None if positions is None else positions.ptr)


def paged_attention(q, cache, shared, window, sinks, scale, out, lse=None):
    return abi.lib.trs_paged_attention_f32(*q.arg, cache.ref if isinstance(cache, Cache) else cache, shared, window, sinks, scale, *out.arg,
                                           None if lse is None else lse.ptr)


__all__ = [n for n in dir() if not n.startswith("_")]
_ = Placed, contiguous_strides

"""The attention block's operators in 64 bits, and their C-ABI calls on numpy arrays."""
from __future__ import annotations

import ctypes

import numpy as np

from trs_backend import abi
from trs_backend.abi import DeviceArray, Layout, check, contiguous_strides, layout_of

U = 2.0 ** -24  # half a unit in the last place of 1
LEAST = 2.0 ** -149  # the least float: what is smaller is off by up to that
EVERY = (1 << 63) - 1  # no window


class Placed:
    """An array in device memory behind a layout: `order` lists the dims from the
    slowest to the fastest in memory, `pad` lengthens the fastest dim's rows, `step`
    is the fastest dim's stride, and `offset` elements precede the view.  What is
    not the view's is NaN (and stays so, `untouched`)."""

    def __init__(self, values=None, shape=None, order=None, pad=0, step=1, offset=0):
        shape = tuple(values.shape if values is not None else shape)
        order = tuple(order if order is not None else range(len(shape)))
        strides, s = [0] * len(shape), step
        for i, d in enumerate(reversed(order)):
            strides[d] = s
            s *= max(shape[d], 1)
            if i == 0:
                s += pad
        self.shape, self.strides, self.offset = shape, tuple(strides), offset
        self.size = offset + max(s, 1) + 8
        host = np.full(self.size, np.nan, np.float32)
        if values is not None and values.size:
            self.view(host)[...] = values
        self.dev = DeviceArray.from_numpy(host)
        self.layout = layout_of(shape, strides, offset)

    def view(self, flat):
        at = flat[self.offset:]
        return np.lib.stride_tricks.as_strided(at, self.shape, tuple(4 * s for s in self.strides))

    def numpy(self):
        self.host = self.dev.to_numpy()
        return self.view(self.host).copy()

    def untouched(self):
        """Whether everything beside the view still is NaN (after numpy())."""
        rest = self.host.copy()
        if np.prod(self.shape):
            self.view(rest)[...] = np.nan
        return bool(np.isnan(rest).all())

    @property
    def arg(self):
        return self.dev.ptr, ctypes.byref(self.layout)


def ints(values):
    return DeviceArray.from_numpy(np.ascontiguousarray(values, dtype=np.int32))


# ---- dropout ----------------------------------------------------------------

def dropout_words(n, seed, offset):
    """Word i of the counters' words, i < n: Philox4x32-10 in numpy."""
    c = np.arange(-(-n // 4), dtype=np.uint64) + np.uint64(offset)
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    x = [c & low, c >> half, np.zeros_like(c), np.zeros_like(c)]
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        a, b = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(b >> half) ^ x[1] ^ np.uint64(k0), b & low, (a >> half) ^ x[3] ^ np.uint64(k1), a & low]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(x, 1).reshape(-1)[:n]


def dropout_reference(x, p, seed, offset):
    keep = dropout_words(x.size, seed, offset).reshape(x.shape) >= np.uint64(int(np.floor(p * 2.0**32 + 0.5)))
    scale = np.float32(1.0 / (1.0 - p)) if p < 1 else np.float32(0)
    with np.errstate(invalid="ignore", over="ignore"):
        return np.where(keep, x * scale, np.float32(0))


def dropout(x: Placed, p, seed, offset, out: Placed):
    return abi.lib.trs_dropout_f32(*x.arg, p, seed, offset, *out.arg)


# ---- head norm and rotation -------------------------------------------------

def rotation_tables(rows, rot, base=100.0):
    half = rot // 2
    angle = np.outer(np.arange(rows), base ** (-np.arange(half) / max(half, 1)))
    return np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)


def _pairs(rot, interleaved):
    i = np.arange(rot // 2)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + rot // 2)


def norm_rope_reference(x, w, eps, cos, sin, positions, interleaved, up=None):
    """y, or (dx, dw) where `up` is given; positions [batch, token]."""
    x, w = x.astype(np.float64), np.ones(x.shape[-1]) if w is None else w.astype(np.float64)
    first, second = _pairs(2 * cos.shape[1], interleaved)
    c, s = (t.astype(np.float64)[positions][:, None] for t in (cos, sin))
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + eps)
    if up is None:
        n = x * r * w
        y = n.copy()
        y[..., first] = n[..., first] * c - n[..., second] * s
        y[..., second] = n[..., second] * c + n[..., first] * s
        return y
    u = up.astype(np.float64)
    g = u.copy()
    g[..., first] = u[..., first] * c + u[..., second] * s
    g[..., second] = u[..., second] * c - u[..., first] * s
    dw = (g * x * r).sum((0, 1, 2))
    dx = r * (w * g - x * r * r * (w * g * x).mean(-1, keepdims=True))
    return dx, dw


def pointers(devs):
    return (ctypes.c_void_p * len(devs))(*[None if d is None else d.addr for d in devs])


def layouts(placed):
    return (Layout * len(placed))(*[p.layout for p in placed])


def norm_rope(xs, ws, eps, cos, sin, interleaved, positions, start, outs, ups=None, dws=None):
    """The status of the call; tensors are Placed, weights DeviceArray or None."""
    args = (len(xs), pointers([x.dev for x in xs]), layouts(xs), pointers(ws), eps, cos.dev.ptr, sin.dev.ptr,
            ctypes.byref(cos.layout), int(interleaved), positions.ptr if positions is not None else None, start)
    if ups is None:
        return abi.lib.trs_head_norm_rope_f32(*args, pointers([o.dev for o in outs]), layouts(outs))
    return abi.lib.trs_head_norm_rope_backward_f32(*args, pointers([u.dev for u in ups]), layouts(ups),
                                                   pointers([o.dev for o in outs]), layouts(outs), pointers(dws))


# ---- attention --------------------------------------------------------------

def seen(sq, n, window, sinks):
    """[query, key]: whether the query of a sequence of n keys sees the key."""
    p = (n - sq + np.arange(sq))[:, None]
    j = np.arange(n)[None, :]
    return (j <= p) & ((p - j < window) | (j < sinks))


def attention_reference(q, k, v, window, sinks, scale, lengths=None, up=None):
    """{name: (value, bound)}: out and lse, and with `up` dq, dk and dv, in 64
    bits; `bound` is how far fp32 arithmetic may be off, from the sums of
    magnitudes (no cancellation assumed):
      s: (D+8) u sum|q||k| scale =: d; p: 2 d + (n+8) u of itself; and so on.
    A weight p below the least float is off by that, and so is each product."""
    B, H, sq, D = q.shape
    hk, sk = k.shape[1:3]
    G = H // hk
    res = {n: (np.zeros(s), np.zeros(s)) for n, s in (("out", q.shape), ("dq", q.shape), ("dk", k.shape), ("dv", k.shape))}
    res["lse"] = (np.full((B, H, sq), -np.inf), np.zeros((B, H, sq)))
    R = sq * G
    for b in range(B):
        n = sk if lengths is None else int(min(max(lengths[b], 0), sk))
        if n == 0:
            continue
        mask = seen(sq, n, window, sinks)
        live = mask.any(1)
        for h in range(H):
            Q, K, V = (t.astype(np.float64) for t in (q[b, h][live], k[b, h // G, :n], v[b, h // G, :n]))
            m = mask[live]
            if not live.any():
                continue
            s = np.where(m, Q @ K.T * scale, -np.inf)
            top = s.max(1, keepdims=True)
            e = np.exp(s - top)
            tot = e.sum(1, keepdims=True)
            P = e / tot
            o = P @ V
            d = (D + 8) * U * np.where(m, abs(Q) @ abs(K).T * abs(scale), 0).max(1, keepdims=True)
            rel = 2 * d + (n + 16) * U
            res["out"][0][b, h, live] = o
            res["out"][1][b, h, live] = rel * (P @ abs(V))
            lse = (top + np.log(tot))[:, 0]
            res["lse"][0][b, h, live] = lse
            res["lse"][1][b, h, live] = (rel + 8 * U * (1 + abs(lse[:, None])))[:, 0]
            if up is None:
                continue
            W = up[b, h][live].astype(np.float64)
            delta = (W * o).sum(1, keepdims=True)
            dS = P * (W @ V.T - delta) * scale
            # lse is read back in fp32: its rounding counts in P too
            rp = 2 * rel + 8 * U * (1 + abs(lse[:, None]))
            A = P * (abs(W) @ abs(V).T + (abs(W) * (P @ abs(V))).sum(1, keepdims=True)) * abs(scale)
            least = LEAST * (1 + A / np.where(P > 0, P, 1))
            eS = A * (2 * rp + (2 * D + 32) * U) + least
            res["dq"][0][b, h, live] = dS @ K
            res["dq"][1][b, h, live] = eS @ abs(K) + (n + 16) * U * (A @ abs(K))
            res["dk"][0][b, h // G, :n] += dS.T @ Q
            res["dk"][1][b, h // G, :n] += eS.T @ abs(Q) + (R + 64) * U * (A.T @ abs(Q)) + R * LEAST
            res["dv"][0][b, h // G, :n] += P.T @ W
            res["dv"][1][b, h // G, :n] += (P * rp).T @ abs(W) + (R + 64) * U * (P.T @ abs(W)) + LEAST * (R + abs(W).sum(0))
    return res


def attention(q, k, v, window, sinks, scale, out, lse=None, lengths=None):
    """The status of the forward call; tensors are Placed, lse and lengths DeviceArray."""
    return abi.lib.trs_window_attention_f32(*q.arg, *k.arg, *v.arg, lengths.ptr if lengths is not None else None, window, sinks,
                                            scale, *out.arg, lse.ptr if lse is not None else None)


def attention_grad(q, k, v, window, sinks, scale, out, lse, up, dq, dk, dv, lengths=None):
    return abi.lib.trs_window_attention_backward_f32(
        *q.arg, *k.arg, *v.arg, lengths.ptr if lengths is not None else None, window, sinks, scale, *out.arg,
        lse.ptr if lse is not None else None, *up.arg, *dq.arg, *dk.arg, *dv.arg)


def assert_within(got, want, bound, what=""):
    """|got - want| <= bound at every element (both NaN, or the same infinity, count as equal)."""
    got = np.asarray(got, np.float64)
    same = (got == want) | (np.isnan(got) & np.isnan(want))
    with np.errstate(invalid="ignore"):
        off = np.where(same, 0.0, abs(got - want))
        ok = same | (off <= bound)
    assert ok.all(), f"{what}: {(~ok).sum()} of {ok.size} off, worst {np.nanmax(off)} where {bound.reshape(-1)[np.nanargmax(off - bound)]} is allowed, at {np.argwhere(~ok)[:4].tolist()}"


__all__ = [n for n in dir() if not n.startswith("_")]
_ = check, contiguous_strides

"""The attention block's operators, as cases to measure.

  kind        what it stands for
  dropout     dropout from a counter-based generator; with "grad", a training step's forward and gradient
  norm_rope   the norm of each head's queries and keys with the position rotation; with "grad", its gradients
  attention   causal attention with a sliding window and first tokens that stay visible, over prompts;
              with "grad", a training step's output and gradients; with q < len, new tokens over a cache

Every case calls the C ABI of include/trs_hip.h (own) or computes the same in
elementary torch operations (the plain form).  Everything is float32, the
framework's tensor type; lengths are int32.
"""
import ctypes
import functools
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False  # whether run() calls the framework's operators or computes their plain forms

_EPS = 1e-6
_BASE = 10000.0  # of the rotation's frequencies


def listed():
    return [
        # An activation of a few rows: the call itself is the cost.
        {"name": "dropout_small", "kind": "dropout", "rows": 32, "cols": 1000, "p": 0.5, "grad": False},
        # The benchmark's hidden activation in a training step: forward and gradient.
        {"name": "dropout_train", "kind": "dropout", "rows": 8192, "cols": 4096, "p": 0.1, "grad": True},
        # One new token of a small batch, in front of a cache.
        {"name": "norm_rope_token", "kind": "norm_rope", "batch": 8, "heads": 32, "kv_heads": 8, "q": 1, "dim": 128, "past": 2047,
         "rot": 128, "interleaved": False, "grad": False},
        # A long prompt's queries and keys.
        {"name": "norm_rope_prompt", "kind": "norm_rope", "batch": 2, "heads": 32, "kv_heads": 8, "q": 4096, "dim": 128, "past": 0,
         "rot": 128, "interleaved": False, "grad": False},
        # Training's gradients, an odd length, neighbours rotated in pairs.
        {"name": "norm_rope_grad", "kind": "norm_rope", "batch": 4, "heads": 16, "kv_heads": 4, "q": 2047, "dim": 64, "past": 0,
         "rot": 64, "interleaved": True, "grad": True},
        # A prompt of ordinary length through one layer.
        {"name": "attention_prompt", "kind": "attention", "batch": 1, "heads": 32, "kv_heads": 8, "q": 4096, "len": 4096, "dim": 128,
         "window": 1024, "sinks": 4, "ragged": False, "grad": False},
        # A ragged batch with heads of 80 and a key head for each: queries padded in front, so that every sequence
        # ends at the last one, over keys that begin at the first place of their rows.
        {"name": "attention_ragged", "kind": "attention", "batch": 3, "heads": 6, "kv_heads": 6, "q": 1000, "len": 1000, "dim": 80,
         "window": 200, "sinks": 3, "ragged": True, "grad": False},
        # A small model's training step at an odd length.
        {"name": "attention_grad_small", "kind": "attention", "batch": 1, "heads": 4, "kv_heads": 2, "q": 333, "len": 333, "dim": 32,
         "window": 64, "sinks": 2, "ragged": False, "grad": True},
        # Training, ordinary sizes.
        {"name": "attention_grad", "kind": "attention", "batch": 2, "heads": 16, "kv_heads": 4, "q": 2048, "len": 2048, "dim": 64,
         "window": 512, "sinks": 4, "ragged": False, "grad": True},
        # Training on long rows: the largest.
        {"name": "attention_grad_long", "kind": "attention", "batch": 1, "heads": 32, "kv_heads": 8, "q": 4096, "len": 4096, "dim": 128,
         "window": 2048, "sinks": 16, "ragged": False, "grad": True},
        # One token for one user: latency.
        {"name": "token_small", "kind": "attention", "batch": 1, "heads": 8, "kv_heads": 8, "q": 1, "len": 1000, "dim": 64,
         "window": 512, "sinks": 4, "ragged": False, "grad": False},
        # One token each for a batch of users with caches of different lengths.
        {"name": "token_batch", "kind": "attention", "batch": 16, "heads": 32, "kv_heads": 8, "q": 1, "len": 8192, "dim": 128,
         "window": 4096, "sinks": 4, "ragged": True, "grad": False},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, even over its logarithm; half of them multiples of 32 where that fits."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))
    if rng.random() < 0.5 and n >= 64:
        n = n // 32 * 32
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(("dropout", "norm_rope", "attention", "attention", "token"))
    if kind == "dropout":
        return {"kind": kind, "rows": _size(rng, 1, 8192), "cols": _size(rng, 32, 4096), "p": round(rng.uniform(0.05, 0.6), 3),
                "grad": rng.random() < 0.5}
    kv = rng.choice((1, 2, 3, 4, 8))
    heads = kv * rng.choice((1, 1, 2, 4, 5, 8))
    if kind == "norm_rope":
        dim = rng.choice((32, 64, 80, 96, 128, 128, 256))
        most = (8192 * 40 * 128) // ((heads + kv) * dim)
        batch = rng.choice((1, 2, 3, 8))
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv, "q": _size(rng, 1, min(4096, most // batch)), "dim": dim,
                "past": rng.choice((0, 0, 100, 2047)), "rot": rng.choice((dim, dim, dim // 2)), "interleaved": rng.random() < 0.3,
                "grad": rng.random() < 0.5}
    case = {"kind": "attention", "batch": rng.choice((1, 2, 3, 5)), "heads": heads, "kv_heads": kv, "q": 1, "len": 1,
            "dim": rng.choice((32, 48, 64, 64, 80, 96, 128, 128, 200, 256)), "window": _size(rng, 16, 4096), "sinks": rng.choice((0, 1, 4, 16, 40)),
            "ragged": rng.random() < 0.4, "grad": False}
    if kind == "token":
        case["batch"] = rng.choice((1, 1, 2, 7, 16, 32))
        case["q"] = rng.choice((1, 1, 1, 2, 4))
        case["len"] = _size(rng, 16, min(16384, 16 * 8 * 8192 * 128 // (case["batch"] * kv * case["dim"])))
        return case
    case["grad"] = rng.random() < 0.5
    # No more scores than the largest case has, nor more products.
    most = math.sqrt(32 * 4096 * 4096 * min(1.0, 128 / case["dim"]) / (case["batch"] * heads))
    case["q"] = case["len"] = _size(rng, 8, min(4096, int(most)))
    if rng.random() < 0.2 and not case["grad"]:  # a later part of a prompt, over what the cache holds
        case["q"] = max(1, case["len"] // rng.choice((2, 3, 10)))
    return case


def _lengths(case):
    """The keys that each sequence of the batch has: all alike, or down to a fifth of the most."""
    b, most = case["batch"], case["len"]
    if not case["ragged"]:
        return [most] * b
    return [max(1, most - (most * 4 * i) // (5 * max(1, b - 1)) - i % 3) for i in range(b)]


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    if kind == "dropout":
        n, m = case["rows"], case["cols"]
        st = {"case": case, "x": normal(n, m), "seed": seed * 0x9E3779B97F4A7C15 % (1 << 64), "offset": seed % 1000}
        if case["grad"]:
            st["up"] = normal(n, m)
        return st
    b, h, hk, s, d = case["batch"], case["heads"], case["kv_heads"], case["q"], case["dim"]
    # Queries and new keys as a projection leaves them: [batch, token, head, dim], read as [batch, head, token, dim].
    q = normal(b, s, h, d).transpose(1, 2)
    if kind == "norm_rope":
        k = normal(b, s, hk, d).transpose(1, 2)
        half = case["rot"] // 2
        freq = _BASE ** (-np.arange(half) / half)
        angle = np.outer(np.arange(case["past"] + s), freq)
        st = {"case": case, "x": [q, k], "w": [1 + 0.1 * normal(d), 1 + 0.1 * normal(d)]}
        st["cos"], st["sin"] = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
        if case["grad"]:
            st["up"] = [normal(b, s, h, d).transpose(1, 2), normal(b, s, hk, d).transpose(1, 2)]
        return st
    st = {"case": case, "q": q, "scale": 1 / math.sqrt(d)}
    if case["q"] == case["len"]:  # a prompt's keys and values
        st["k"], st["v"] = (normal(b, s, hk, d).transpose(1, 2) for _ in range(2))
    else:  # a cache
        st["k"], st["v"] = (normal(b, hk, case["len"], d) for _ in range(2))
    st["lengths"] = torch.tensor(_lengths(case), dtype=torch.int32).cuda() if case["ragged"] else None
    if case["grad"]:
        st["up"] = normal(b, s, h, d).transpose(1, 2)
    return st


# ---- the framework's calls --------------------------------------------------

@functools.lru_cache(None)
def _backend():
    pkg = str(Path(__file__).resolve().parent.parent / "pytorch-rs_amd")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    from trs_backend import abi

    abi.check(abi.lib.trs_init())
    return abi


@functools.lru_cache(256)
def _layout(shape, strides):
    return _backend().layout_of(shape, strides)


def _arg(t):
    """A tensor's address and layout."""
    return t.data_ptr(), ctypes.byref(_layout(t.shape, t.stride()))


def _like(t):
    """An output for a [batch, head, token, dim] view, its memory in token order."""
    b, h, s, d = t.shape
    return torch.empty(b, s, h, d, device="cuda").transpose(1, 2)


def _own_dropout(st):
    abi, case = _backend(), st["case"]
    got = []
    for x in (st["x"], st["up"]) if case["grad"] else (st["x"],):
        y = torch.empty_like(x)
        abi.check(abi.lib.trs_dropout_f32(*_arg(x), case["p"], st["seed"], st["offset"], *_arg(y)))
        got.append(y)
    return got


def _pair(tensors):
    """Two tensors' addresses, and their layouts."""
    abi = _backend()
    return (ctypes.c_void_p * 2)(*(t.data_ptr() for t in tensors)), (abi.Layout * 2)(*(_layout(t.shape, t.stride()) for t in tensors))


def _own_norm_rope(st):
    abi, case = _backend(), st["case"]
    (xs, lx), out = _pair(st["x"]), [_like(t) for t in st["x"]]
    ws = (ctypes.c_void_p * 2)(*(w.data_ptr() for w in st["w"]))
    cos, tab = _arg(st["cos"])
    rotation = (_EPS, cos, st["sin"].data_ptr(), tab, int(case["interleaved"]), None, case["past"])
    os, lo = _pair(out)
    if not case["grad"]:
        abi.check(abi.lib.trs_head_norm_rope_f32(2, xs, lx, ws, *rotation, os, lo))
        return [t.transpose(1, 2) for t in out]
    dw = [torch.empty_like(w) for w in st["w"]]
    dws = (ctypes.c_void_p * 2)(*(w.data_ptr() for w in dw))
    abi.check(abi.lib.trs_head_norm_rope_backward_f32(2, xs, lx, ws, *rotation, *_pair(st["up"]), os, lo, dws))
    return [t.transpose(1, 2) for t in out] + dw


def _own_attention(st):
    abi, case = _backend(), st["case"]
    q, k, v = st["q"], st["k"], st["v"]
    out = _like(q)
    lens = None if st["lengths"] is None else st["lengths"].data_ptr()
    mask = (lens, case["window"], case["sinks"], st["scale"])
    if not case["grad"]:
        abi.check(abi.lib.trs_window_attention_f32(*_arg(q), *_arg(k), *_arg(v), *mask, *_arg(out), None))
        return [out.transpose(1, 2)]
    lse = torch.empty(q.shape[:3], device="cuda")
    abi.check(abi.lib.trs_window_attention_f32(*_arg(q), *_arg(k), *_arg(v), *mask, *_arg(out), lse.data_ptr()))
    dq, dk, dv = _like(q), _like(k), _like(v)
    abi.check(abi.lib.trs_window_attention_backward_f32(*_arg(q), *_arg(k), *_arg(v), *mask, *_arg(out), lse.data_ptr(),
                                                        *_arg(st["up"]), *_arg(dq), *_arg(dk), *_arg(dv)))
    return [t.transpose(1, 2) for t in (out, dq, dk, dv)]


# ---- the plain forms --------------------------------------------------------

def _philox(counter, seed):
    """The four words of each 64-bit counter: ten rounds of Philox4x32, in 64-bit integers."""
    low = 0xFFFFFFFF
    x0, x1 = counter & low, (counter >> 32) & low
    x2 = x3 = torch.zeros_like(x0)
    k0, k1 = seed & low, seed >> 32
    for _ in range(10):
        a, b = x0 * 0xD2511F53, x2 * 0xCD9E8D57
        x0, x1, x2, x3 = ((b >> 32) & low) ^ x1 ^ k0, b & low, ((a >> 32) & low) ^ x3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((x0, x1, x2, x3), 1)


def _plain_dropout(st):
    x, case = st["x"], st["case"]
    words = _philox(torch.arange(-(-x.numel() // 4), device="cuda") + st["offset"], st["seed"])
    keep = (words.reshape(-1)[: x.numel()] >= math.floor(case["p"] * 2**32 + 0.5)).view(x.shape)
    scale = float(np.float32(1 / (1 - case["p"])))
    zero = torch.zeros((), device="cuda")
    return [torch.where(keep, t * scale, zero) for t in ((x, st["up"]) if case["grad"] else (x,))]


def _halves(x, case):
    """The first and the second entry of every rotated pair, and the entries that are not rotated."""
    r = case["rot"]
    if case["interleaved"]:
        return x[..., 0:r:2], x[..., 1:r:2], x[..., r:]
    return x[..., : r // 2], x[..., r // 2: r], x[..., r:]


def _joined(a, b, rest, case):
    pairs = torch.stack((a, b), -1).flatten(-2) if case["interleaved"] else torch.cat((a, b), -1)
    return torch.cat((pairs, rest), -1)


def _plain_norm_rope(st):
    case = st["case"]
    at = slice(case["past"], case["past"] + case["q"])
    cos, sin = st["cos"][at], st["sin"][at]
    outs, dws = [], []
    for i, (x, w) in enumerate(zip(st["x"], st["w"])):
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + _EPS)
        if not case["grad"]:
            a, b, rest = _halves(x * r * w, case)
            outs.append(_joined(a * cos - b * sin, b * cos + a * sin, rest, case))
            continue
        a, b, rest = _halves(st["up"][i], case)
        g = _joined(a * cos + b * sin, b * cos - a * sin, rest, case)
        n = x * r
        dws.append((g * n).sum((0, 1, 2)))
        wg = g * w
        outs.append(r * (wg - n * (wg * n).mean(-1, keepdim=True)))
    return [t.transpose(1, 2).contiguous() for t in outs] + dws


def _visible(case, lengths):
    """[batch, query, key]: whether the query sees the key."""
    length = torch.full((case["batch"],), case["len"], device="cuda") if lengths is None else lengths.long()
    at = (length - case["q"])[:, None, None] + torch.arange(case["q"], device="cuda")[None, :, None]
    j = torch.arange(case["len"], device="cuda")[None, None, :]
    return (j <= at) & ((at - j < case["window"]) | (j < case["sinks"]))


def _plain_attention(st):
    case, scale = st["case"], st["scale"]
    b, h, hk, s, d, n = case["batch"], case["heads"], case["kv_heads"], case["q"], case["dim"], case["len"]

    def rows(t):  # the query heads that share a key head, as its rows
        return t.reshape(b, hk, (h // hk) * s, d)

    q, k, v = rows(st["q"]), st["k"], st["v"]
    seen = _visible(case, st["lengths"])[:, None, None]
    x = (q @ k.transpose(-1, -2) * scale).view(b, hk, h // hk, s, n)
    x = torch.where(seen, x, -math.inf)
    most = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(b, hk, -1, n)
    out = p @ v

    def tokens(t, heads):
        return t.reshape(b, heads, -1, d).transpose(1, 2).contiguous()

    if not case["grad"]:
        return [tokens(out, h)]
    up = rows(st["up"])
    dx = p * (up @ v.transpose(-1, -2) - (up * out).sum(-1, keepdim=True)) * scale
    return [tokens(out, h), tokens(dx @ k, h), tokens(dx.transpose(-1, -2) @ q, hk), tokens(p.transpose(-1, -2) @ up, hk)]


def run(state):
    kind = state["case"]["kind"]
    if kind == "dropout":
        return _own_dropout(state) if own else _plain_dropout(state)
    if kind == "norm_rope":
        return _own_norm_rope(state) if own else _plain_norm_rope(state)
    return _own_attention(state) if own else _plain_attention(state)


# ---- what a pass cannot do without, and its exact result ---------------------

def work(case):
    kind = case["kind"]
    if kind == "dropout":
        n = case["rows"] * case["cols"] * (2 if case["grad"] else 1)
        return {"bytes": 8 * n, "flops": n}
    if kind == "norm_rope":
        n = case["batch"] * (case["heads"] + case["kv_heads"]) * case["q"] * case["dim"]
        tables = 4 * case["q"] * case["rot"]
        return {"bytes": (12 if case["grad"] else 8) * n + tables, "flops": (16 if case["grad"] else 8) * n}
    pairs = keys = 0
    for n in _lengths(case):
        at = np.arange(max(0, n - case["q"]), n)
        near = np.minimum(at + 1, case["window"])
        pairs += int((near + np.minimum(case["sinks"], at + 1 - near)).sum())
        first = max(0, max(0, n - case["q"]) + 1 - case["window"])  # of the window of the first query
        keys += n - first + min(case["sinks"], first)
    d = case["dim"]
    rows = case["batch"] * case["heads"] * case["q"] * d
    kv = case["kv_heads"] * keys * d
    if case["grad"]:
        return {"bytes": 4 * (4 * rows + 2 * kv + 2 * case["batch"] * case["kv_heads"] * case["len"] * d), "flops": 14 * d * case["heads"] * pairs}
    return {"bytes": 4 * (2 * rows + 2 * kv), "flops": 4 * d * case["heads"] * pairs}


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "dropout":
        return _exact_dropout(st)
    if kind == "norm_rope":
        return _exact_norm_rope(st)
    return _exact_attention(st)


def _exact_dropout(st):
    """On the host, a counter's words in numpy's unsigned integers."""
    case, n = st["case"], st["x"].numel()
    c = np.arange(-(-n // 4), dtype=np.uint64) + np.uint64(st["offset"])
    mask, shift = np.uint64(0xFFFFFFFF), np.uint64(32)
    words = [c & mask, c >> shift, np.zeros_like(c), np.zeros_like(c)]
    key = [st["seed"] % 2**32, st["seed"] // 2**32]
    for _ in range(10):
        first, second = words[0] * np.uint64(3528531795), words[2] * np.uint64(3449720151)
        words = [(second >> shift) ^ words[1] ^ np.uint64(key[0]), second & mask, (first >> shift) ^ words[3] ^ np.uint64(key[1]), first & mask]
        key = [(key[0] + 2654435769) % 2**32, (key[1] + 3144134277) % 2**32]
    kept = np.stack(words, 1).reshape(-1)[:n] >= np.uint64(int(case["p"] * 2**32 + 0.5))
    kept = torch.from_numpy(kept).cuda().view(st["x"].shape)
    return [t.double() / (1 - case["p"]) * kept for t in ((st["x"], st["up"]) if case["grad"] else (st["x"],))]


def _exact_norm_rope(st):
    """The rotation as a product of complex numbers; the gradients by autograd of the definition."""
    case = st["case"]
    r, outs, dws = case["rot"], [], []
    at = slice(case["past"], case["past"] + case["q"])
    turn = torch.complex(st["cos"][at].double(), st["sin"][at].double())
    for i, (x, w) in enumerate(zip(st["x"], st["w"])):
        x, w = x.double().requires_grad_(case["grad"]), w.double().requires_grad_(case["grad"])
        n = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + _EPS).sqrt() * w
        pairs = n[..., :r].unflatten(-1, (r // 2, 2)) if case["interleaved"] else n[..., :r].unflatten(-1, (2, r // 2)).transpose(-1, -2)
        z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn)
        y = torch.cat(((z if case["interleaved"] else z.transpose(-1, -2)).flatten(-2), n[..., r:]), -1)
        if case["grad"]:
            dx, dw = torch.autograd.grad(y, (x, w), st["up"][i].double())
            outs.append(dx)
            dws.append(dw)
        else:
            outs.append(y)
    return [t.transpose(1, 2).contiguous() for t in outs] + dws


def _exact_attention(st):
    """Head by head over the keys that a sequence has, with the logarithm of each row's sum."""
    case = st["case"]
    b, h, hk, s, d = case["batch"], case["heads"], case["kv_heads"], case["q"], case["dim"]
    out, dq = (torch.zeros(b, s, h, d, dtype=torch.float64, device="cuda") for _ in range(2))
    dk, dv = (torch.zeros(b, case["len"], hk, d, dtype=torch.float64, device="cuda") for _ in range(2))
    for i, n in enumerate(_lengths(case)):
        first = max(0, s - n)  # the queries before it stand before the sequence
        place = torch.arange(n - s + first, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None, :]
        hidden = (key > place) | ((key <= place - case["window"]) & (key >= case["sinks"]))
        for head in range(h):
            kv = head // (h // hk)
            q, k, v = st["q"][i, head, first:].double(), st["k"][i, kv, :n].double(), st["v"][i, kv, :n].double()
            x = torch.mm(q, k.t()).mul_(st["scale"]).masked_fill_(hidden, -math.inf)
            p = x.sub_(torch.logsumexp(x, 1, keepdim=True)).exp_()
            o = torch.mm(p, v)
            out[i, first:, head] = o
            if case["grad"]:
                up = st["up"][i, head, first:].double()
                dv[i, :n, kv] += torch.mm(p.t(), up)
                dx = torch.mm(up, v.t()).sub_((up * o).sum(1, keepdim=True)).mul_(p).mul_(st["scale"])
                dq[i, first:, head] = torch.mm(dx, k)
                dk[i, :n, kv] += torch.mm(dx.t(), q)
    return [out, dq, dk, dv] if case["grad"] else [out]

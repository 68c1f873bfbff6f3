"""The paged cache's operators, as cases to measure.

  kind        what it stands for
  rope        queries and keys turned by positions of several axes (time, height, width); with "grad", a training
              step's forward and gradient
  append      keys and values of new tokens written to a paged cache, the keys turned by their positions on the way,
              and the queries in the same call
  attention   causal attention of new tokens over a paged cache, with a window and first tokens that stay visible;
              with "shared", over keys that the whole batch has in common and each sequence's own
  step        a new token of every sequence appended, then its attention

Every case calls the C ABI of include/trs_hip.h (own) or computes the same in
elementary torch operations (the plain form).  Queries, keys, values and outputs
are float32, the framework's tensor type; pages hold float32 or bfloat16.

The library's stream is not ordered with torch's: whoever calls run() with `own`
waits for the device between making or changing a state with torch and the call,
and between the call and reading its outputs or letting go of them with torch.
Passes one behind another need no waiting between them, as long as what a pass
takes from torch's allocator is not written by torch's own work meanwhile.
"""
import ctypes
import functools
import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False  # whether run() calls the framework's operators or computes their plain forms

_BASE = 10000.0  # of the rotation's frequencies


def listed():
    return [
        # One new token of a small batch: the call itself is the cost.
        {"name": "rope_token", "kind": "rope", "batch": 8, "heads": 32, "kv_heads": 8, "q": 1, "dim": 128, "rot": 128, "axes": 3,
         "interleaved": False, "grad": False},
        # Long prompts with a video in them.
        {"name": "rope_video", "kind": "rope", "batch": 2, "heads": 32, "kv_heads": 8, "q": 4096, "dim": 128, "rot": 128, "axes": 3,
         "interleaved": False, "grad": False},
        # Training on images at an odd length, half of a head turned, neighbours in pairs.
        {"name": "rope_grad", "kind": "rope", "batch": 4, "heads": 16, "kv_heads": 4, "q": 2047, "dim": 64, "rot": 32, "axes": 2,
         "interleaved": True, "grad": True},
        # One token each for a batch of users.
        {"name": "append_token", "kind": "append", "batch": 16, "heads": 32, "kv_heads": 8, "q": 1, "len": 512, "dim": 128, "page": 16,
         "bf16": True, "ragged": True, "axes": 1},
        # Two long prompts.
        {"name": "append_prompt", "kind": "append", "batch": 2, "heads": 32, "kv_heads": 8, "q": 4096, "len": 4096, "dim": 128, "page": 64,
         "bf16": False, "ragged": False, "axes": 3},
        # One token for one user: latency.
        {"name": "paged_token_small", "kind": "attention", "batch": 1, "heads": 8, "kv_heads": 8, "q": 1, "len": 1000, "dim": 64, "page": 16,
         "bf16": False, "ragged": False, "window": 0, "sinks": 0, "shared": 0},
        # One token each for a batch of users with caches of different lengths.
        {"name": "paged_token_batch", "kind": "attention", "batch": 32, "heads": 32, "kv_heads": 8, "q": 1, "len": 8192, "dim": 128, "page": 16,
         "bf16": True, "ragged": True, "window": 0, "sinks": 0, "shared": 0},
        # A part of a long prompt over what the cache holds already.
        {"name": "paged_prompt", "kind": "attention", "batch": 2, "heads": 32, "kv_heads": 8, "q": 1024, "len": 4096, "dim": 128, "page": 64,
         "bf16": True, "ragged": False, "window": 0, "sinks": 0, "shared": 0},
        # Ragged prompts of a small model with heads of 80, sliding window.
        {"name": "paged_prompt_ragged", "kind": "attention", "batch": 3, "heads": 6, "kv_heads": 6, "q": 333, "len": 1000, "dim": 80, "page": 16,
         "bf16": False, "ragged": True, "window": 200, "sinks": 3, "shared": 0},
        # A batch of users behind one system prompt.
        {"name": "shared_batch", "kind": "attention", "batch": 64, "heads": 32, "kv_heads": 8, "q": 1, "len": 8704, "dim": 128, "page": 16,
         "bf16": True, "ragged": True, "window": 0, "sinks": 0, "shared": 8192},
        # A few answers to one prompt of a small model.
        {"name": "shared_small", "kind": "attention", "batch": 5, "heads": 8, "kv_heads": 2, "q": 1, "len": 1100, "dim": 64, "page": 16,
         "bf16": False, "ragged": True, "window": 0, "sinks": 0, "shared": 1000},
        # What a served token costs a layer beside its products.
        {"name": "step_batch", "kind": "step", "batch": 8, "heads": 32, "kv_heads": 8, "q": 1, "len": 2000, "dim": 128, "page": 16,
         "bf16": True, "ragged": True, "axes": 1, "window": 1024, "sinks": 4, "shared": 0},
    ]


def _size(rng, lo, hi):
    """A size between lo and hi, even over its logarithm; half of them multiples of 32 where that fits."""
    n = int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))
    if rng.random() < 0.5 and n >= 64:
        n = n // 32 * 32
    return max(lo, min(hi, n))


def draw(rng):
    kind = rng.choice(("rope", "append", "token", "token", "prompt", "shared", "shared", "step"))
    kv = rng.choice((1, 2, 3, 4, 8))
    heads = kv * rng.choice((1, 1, 2, 4, 5, 8))
    dim = rng.choice((32, 48, 64, 64, 80, 96, 128, 128, 200, 256))
    batch = rng.choice((1, 2, 3, 8))
    most = (8192 * 40 * 128) // ((heads + 2 * kv) * dim)  # tokens with as many entries as the largest rotation's
    if kind == "rope":
        return {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv, "q": _size(rng, 1, min(4096, most // batch)), "dim": dim,
                "rot": rng.choice((dim, dim, dim // 2)), "axes": rng.choice((1, 2, 3, 3, 4)), "interleaved": rng.random() < 0.3,
                "grad": rng.random() < 0.4}
    case = {"kind": kind, "batch": batch, "heads": heads, "kv_heads": kv, "q": 1, "len": 1, "dim": dim, "page": rng.choice((8, 16, 16, 32, 48, 64, 128)),
            "bf16": rng.random() < 0.6, "ragged": rng.random() < 0.5}
    if kind == "append":
        case["axes"] = rng.choice((1, 1, 3))
        case["q"] = rng.choice((1, 1, 2, 0)) or _size(rng, 3, min(4096, most // batch))
        case["len"] = case["q"] + rng.choice((0, 0, 100, 500))
        return case
    case["window"] = rng.choice((0, 0, _size(rng, 16, 4096)))
    case["sinks"] = rng.choice((0, 4, 40)) if case["window"] else 0
    case["shared"] = 0
    if kind == "prompt":
        case["kind"] = "attention"
        pairs = math.sqrt(1024 * 4096 * 2 * 32 * 128 / (batch * heads * dim) / (1 if case["bf16"] else 2))  # as many products as the largest prompt's
        case["len"] = _size(rng, 16, min(4096, int(pairs)))
        case["q"] = max(1, case["len"] // rng.choice((1, 2, 4, 10)))
        return case
    if kind == "shared":
        case["kind"] = "attention"
        case["batch"] = rng.choice((2, 3, 7, 16, 33, 64))
        case["q"] = rng.choice((1, 1, 1, 2, 4))
        rows = case["batch"] * heads * case["q"] * dim
        case["shared"] = _size(rng, 16, min(8192, 64 * 32 * 128 * 8192 // rows // (1 if case["bf16"] else 2)))
        case["len"] = case["shared"] + _size(rng, 1, 512)
        return case
    case["batch"] = rng.choice((1, 1, 2, 7, 16, 32))
    case["q"] = rng.choice((1, 1, 1, 2, 4))
    case["len"] = _size(rng, 16, min(16384, 32 * 8 * 4915 * 128 // (case["batch"] * kv * dim) // (1 if case["bf16"] else 2)))
    if kind == "step":
        case["axes"] = rng.choice((1, 1, 3))
        case["len"] = min(case["len"], _size(rng, 16, 2048))
    else:
        case["kind"] = "attention"
    return case


def _lengths(case):
    """The keys that each sequence of the batch has, its new ones among them: all alike, or down to a fifth of the most (of what is
    not shared)."""
    b, most = case["batch"], case["len"] - case.get("shared", 0)
    if not case["ragged"]:
        return [case["len"]] * b
    return [case["len"] - most + max(1, most - (most * 4 * i) // (5 * max(1, b - 1)) - i % 3) for i in range(b)]


def _pair_axes(case):
    """The axis of every pair: a quarter time's, the rest divided among the others."""
    pairs, axes = case.get("rot", case["dim"]) // 2, case["axes"]
    if axes == 1:
        return [0] * pairs
    first = pairs // 4
    return [0] * first + [1 + (axes - 1) * i // (pairs - first) for i in range(pairs - first)]


def _positions(case, past):
    """[axes, batch, token]: text, then frames of an image grid or a video, then text; on one axis the token's own place."""
    b, s, axes = case["batch"], case["q"], case["axes"]
    pos = np.empty((axes, b, s), np.int32)
    for i in range(b):
        for a in range(axes):
            pos[a, i] = np.maximum(past[i] + np.arange(s), 0)  # padding in front of a sequence stands at 0
        if axes > 1 and s >= 48:
            text, wide = s // 6, max(2, int((s // 2) ** (1 / 3)))
            n = s - 2 * text
            at = np.arange(n)
            grid = (at // (wide * wide), at // wide % wide, at % wide, at % 2)
            if axes == 2:
                grid = (at // wide, at % wide)
            for a in range(axes):
                pos[a, i, text: text + n] = max(0, past[i]) + text + grid[a]
            after = pos[:, i, : text + n].max() + 1
            pos[:, i, text + n:] = after + np.arange(text)
    return pos


# ---- inputs -----------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")

    kind = case["kind"]
    b, h, hk, s, d = case["batch"], case["heads"], case["kv_heads"], case["q"], case["dim"]
    # Queries and new keys as a projection leaves them: [batch, token, head, dim], read as [batch, head, token, dim].
    st = {"case": case, "q": normal(b, s, h, d).transpose(1, 2)}
    if kind != "attention":
        st["k"] = normal(b, s, hk, d).transpose(1, 2)
        lens = _lengths(case) if kind != "rope" else [s + 17 * i for i in range(b)]
        pos = _positions(case, [n - s for n in lens])
        pairs = case.get("rot", d) // 2
        angle = np.outer(np.arange(int(pos.max()) + 1), _BASE ** (-np.arange(pairs) / pairs))
        st["cos"], st["sin"] = (torch.from_numpy(f(angle).astype(np.float32)).cuda() for f in (np.cos, np.sin))
        st["positions"] = torch.from_numpy(pos).cuda()
        st["pair_axes"] = bytes(_pair_axes(case))
        st["axes"] = torch.tensor(_pair_axes(case), device="cuda")
    if kind == "rope":
        if case["grad"]:
            st["up"] = [normal(b, s, h, d).transpose(1, 2), normal(b, s, hk, d).transpose(1, 2)]
        return st
    if kind != "attention":
        st["v"] = normal(b, s, hk, d).transpose(1, 2)
    # A pool whose pages have been given out and taken back for some time: a sequence's lie anywhere.  Pages of what is shared stand
    # in every row of the table; rows hold -1 behind a sequence's last page.
    page, lens, shared = case["page"], _lengths(case), case.get("shared", 0)
    width, whole = -(-case["len"] // page), shared // page
    counts = [-(-n // page) - whole for n in lens]
    pages = whole + sum(counts) + 3
    free = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    table = torch.full((b, width), -1, dtype=torch.int32)
    table[:, :whole] = free[:whole]
    at = whole
    for i, n in enumerate(counts):
        table[i, whole: whole + n] = free[at: at + n]
        at += n
    if shared % page:  # the first row has the shared keys' last page
        assert counts[0] > 0
    st["table"], st["lengths"] = table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda()
    dtype = torch.bfloat16 if case["bf16"] else torch.float32
    st["pages"] = [normal(pages, hk, page, d).to(dtype) for _ in range(2)]
    st["scale"] = 1 / math.sqrt(d)
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


def _cache(st):
    """The cache's description, which a program keeps beside its pages, table and lengths for as long as these stay where they are."""
    abi = _backend()
    k, v = st["pages"]
    table, lengths = st["table"], st["lengths"]
    of = (k.data_ptr(), v.data_ptr(), table.data_ptr(), lengths.data_ptr(), table.shape[1], k.dtype, k.shape, k.stride(), v.stride())
    kept = st.get("cache")
    if kept is None or kept[0] != of:
        kept = st["cache"] = of, abi.PagedCache(k=of[0], v=of[1], lk=_layout(k.shape, k.stride()), lv=_layout(v.shape, v.stride()),
                                                type=abi.PAGES_BF16 if k.dtype == torch.bfloat16 else abi.PAGES_F32, table=of[2], table_width=of[4],
                                                lengths=of[3])
    return kept[1]


def _rotation(st):
    cos, tab = _arg(st["cos"])
    return cos, st["sin"].data_ptr(), tab, int(st["case"].get("interleaved", False)), st["case"]["axes"], st["pair_axes"], st["positions"].data_ptr()


def _own_rope(st):
    abi = _backend()

    def pair(tensors):
        return (ctypes.c_void_p * 2)(*(t.data_ptr() for t in tensors)), (abi.Layout * 2)(*(_layout(t.shape, t.stride()) for t in tensors))

    outs = []
    for inverse, xs in enumerate([[st["q"], st["k"]], st["up"]] if st["case"]["grad"] else [[st["q"], st["k"]]]):
        out = [_like(t) for t in xs]
        abi.check(abi.lib.trs_rope_axes_f32(2, *pair(xs), *_rotation(st), 0, inverse, *pair(out)))
        outs += [t.transpose(1, 2) for t in out]
    return outs


def _own_append(st):
    abi = _backend()
    out = _like(st["q"])
    abi.check(abi.lib.trs_paged_append_f32(ctypes.byref(_cache(st)), *_arg(st["k"]), *_arg(st["v"]), *_arg(st["q"]), *_arg(out), *_rotation(st)))
    return out


def _own_attention(st, q):
    abi, case = _backend(), st["case"]
    out = _like(q)
    abi.check(abi.lib.trs_paged_attention_f32(*_arg(q), ctypes.byref(_cache(st)), case["shared"], case["window"] or (1 << 63) - 1, case["sinks"],
                                              st["scale"], *_arg(out), None))
    return out.transpose(1, 2)


def _run_own(st):
    kind = st["case"]["kind"]
    if kind == "rope":
        return _own_rope(st)
    if kind == "attention":
        return [_own_attention(st, st["q"])]
    q = _own_append(st)
    return [q.transpose(1, 2), *st["pages"]] if kind == "append" else [_own_attention(st, q), *st["pages"]]


# ---- the plain forms --------------------------------------------------------

def _turned(x, st, sign=1):
    """The pairs of x [batch, head, token, dim] turned by their axes' angles."""
    at = st["positions"].long()[st["axes"]].permute(1, 2, 0)  # [batch, token, pair]
    pair = torch.arange(len(st["pair_axes"]), device="cuda")
    cos, sin = st["cos"][at, pair][:, None], st["sin"][at, pair][:, None] * sign
    r = 2 * len(st["pair_axes"])
    if st["case"].get("interleaved", False):
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
    else:
        a, b = x[..., : r // 2], x[..., r // 2: r]
        turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
    return torch.cat((turned, x[..., r:]), -1) if r < x.shape[-1] else turned


def _plain_append(st):
    case, table, lens = st["case"], st["table"], st["lengths"].long()
    page, s = case["page"], case["q"]
    k, v = _turned(st["k"], st).transpose(1, 2), st["v"].transpose(1, 2)
    place = lens[:, None] - s + torch.arange(s, device="cuda")  # [batch, token]
    if s > 1 and case["ragged"]:  # tokens in front of a sequence are padding
        real = place >= 0
        row = torch.arange(case["batch"], device="cuda")[:, None].expand_as(place)[real]
        place, k, v = place[real], k[real], v[real]
    else:
        row = torch.arange(case["batch"], device="cuda")[:, None]
    at = table[row, place // page].long()
    for pool, x in zip(st["pages"], (k, v)):
        pool[at, :, place % page] = x.to(pool.dtype)
    return _turned(st["q"], st)


def _gathered(st, rows, first, last):
    """Keys first to last of some rows of the table, as float32: K and V [rows, kv_heads, keys, dim]."""
    page = st["case"]["page"]
    j = torch.arange(first, last, device="cuda")
    at = st["table"][rows][:, j // page].long().clamp(min=0)
    return [pool[at, :, j % page].transpose(1, 2).float() for pool in st["pages"]]


def _plain_attention(st, q):
    case = st["case"]
    b, h, hk, s, d, n, shared = case["batch"], case["heads"], case["kv_heads"], case["q"], case["dim"], case["len"], case["shared"]
    g = h // hk
    q = q.reshape(b, hk, g * s, d) * st["scale"]
    k, v = _gathered(st, slice(None), shared, n)
    x = q @ k.transpose(-1, -2)
    if shared:  # once for all rows of the batch
        k0, v0 = _gathered(st, slice(0, 1), 0, shared)
        together = q.transpose(0, 1).reshape(hk, b * g * s, d) @ k0[0].transpose(-1, -2)
        x = torch.cat((together.view(hk, b, g * s, shared).transpose(0, 1), x), -1)
    place = (st["lengths"].long() - s)[:, None, None] + torch.arange(s, device="cuda")[None, :, None]
    j = torch.arange(n, device="cuda")
    seen = j <= place
    if case["window"]:
        seen = seen & ((place - j < case["window"]) | (j < case["sinks"]))
    x = torch.where(seen[:, None, None], x.view(b, hk, g, s, n), -math.inf)
    most = x.amax(-1, keepdim=True)
    p = torch.exp(x - torch.where(most == -math.inf, 0.0, most))
    total = p.sum(-1, keepdim=True)
    p = (p / torch.where(total == 0, 1.0, total)).view(b, hk, g * s, n)
    out = p[..., shared:] @ v
    if shared:
        part = p[..., :shared].transpose(0, 1).reshape(hk, b * g * s, shared) @ v0[0]
        out = out + part.view(hk, b, g * s, d).transpose(0, 1)
    return out.view(b, hk, g, s, d).flatten(1, 2).transpose(1, 2).contiguous()


def _run_plain(st):
    kind = st["case"]["kind"]
    if kind == "rope":
        outs = [_turned(x, st) for x in (st["q"], st["k"])]
        if st["case"]["grad"]:
            outs += [_turned(x, st, -1) for x in st["up"]]
        return [t.transpose(1, 2).contiguous() for t in outs]
    if kind == "attention":
        return [_plain_attention(st, st["q"])]
    q = _plain_append(st)
    return [q.transpose(1, 2).contiguous() if kind == "append" else _plain_attention(st, q), *st["pages"]]


def run(state):
    return _run_own(state) if own else _run_plain(state)


# ---- what a pass cannot do without, and its exact result ---------------------

def _attention_work(case):
    """Pairs of a query and a key that it sees, and the keys to read, over the batch and of one key head."""
    pairs, keys, shared_seen = 0, 0, 0
    s, shared = case["q"], case["shared"]
    window = case["window"] or 1 << 40
    for n in _lengths(case):
        at = np.arange(max(0, n - s), n)
        near = np.minimum(at + 1, window)
        pairs += int((near + np.minimum(case["sinks"], at + 1 - near)).sum())
        first = max(0, max(0, n - s) + 1 - window)  # of the window of the first query
        sinks = min(case["sinks"], first)
        keys += max(0, n - max(first, shared)) + max(0, sinks - shared)
        shared_seen = max(shared_seen, max(0, shared - first) + min(sinks, shared))
    return pairs, keys + shared_seen


def work(case):
    kind = case["kind"]
    b, h, hk, s, d = case["batch"], case["heads"], case["kv_heads"], case["q"], case["dim"]
    size = 2 if case.get("bf16") else 4
    total = {"bytes": 0, "flops": 0}
    if kind == "rope":
        n = b * (h + hk) * s
        times = 2 if case["grad"] else 1
        return {"bytes": times * 8 * n * d + 4 * case["axes"] * b * s, "flops": times * 3 * n * case["rot"]}
    if kind in ("append", "step"):
        new = b * hk * s * d
        total["bytes"] += (4 + size) * 2 * new + 8 * b * h * s * d + 4 * case["axes"] * b * s
        total["flops"] += 3 * b * (h + hk) * s * d
    if kind in ("attention", "step"):
        pairs, keys = _attention_work(case)
        total["bytes"] += 8 * b * h * s * d + 2 * size * hk * keys * d
        total["flops"] += 4 * d * h * pairs
    return total


def exact(case, seed):
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "rope":
        outs = [_exact_turned(x, st) for x in (st["q"], st["k"])]
        if case["grad"]:  # the gradient of sum(up * y) by autograd of the definition
            for x, up in zip((st["q"], st["k"]), st["up"]):
                x = x.double().requires_grad_(True)
                outs.append(torch.autograd.grad(_exact_turned(x, st), x, up.double())[0])
        return [t.transpose(1, 2).contiguous() for t in outs]
    pages = [p.double() for p in st["pages"]]
    if kind == "attention":
        return [_exact_attention(st, st["q"], pages)]
    k = _exact_turned(st["k"], st)
    for i, n in enumerate(_lengths(case)):
        for t in range(max(0, case["q"] - n), case["q"]):
            place = n - case["q"] + t
            at = int(st["table"][i, place // case["page"]]) if t == max(0, case["q"] - n) or place % case["page"] == 0 else at
            pages[0][at, :, place % case["page"]] = k[i, :, t]
            pages[1][at, :, place % case["page"]] = st["v"][i, :, t].double()
    q = _exact_turned(st["q"], st)
    if kind == "append":
        return [q.transpose(1, 2).contiguous(), *pages]
    held = [p.to(st["pages"][0].dtype).double() for p in pages]  # the attention reads what the cache holds
    return [_exact_attention(st, q, held), *pages]


def _exact_turned(x, st):
    """The rotation as a product of complex numbers."""
    case, x = st["case"], x.double()
    half = len(st["pair_axes"])
    turn = torch.empty(case["batch"], case["q"], half, dtype=torch.complex128, device="cuda")
    for p, axis in enumerate(st["pair_axes"]):
        at = st["positions"][axis].long()
        turn[..., p] = torch.complex(st["cos"][at, p].double(), st["sin"][at, p].double())
    inter = case.get("interleaved", False)
    first = x[..., : 2 * half]
    pairs = first.unflatten(-1, (half, 2)) if inter else first.unflatten(-1, (2, half)).transpose(-1, -2)
    z = torch.view_as_real(torch.complex(pairs[..., 0], pairs[..., 1]) * turn[:, None])
    return torch.cat(((z if inter else z.transpose(-1, -2)).flatten(-2), x[..., 2 * half:]), -1)


def _exact_attention(st, q, pages):
    """Sequence by sequence and key head by key head, over a list of the keys that it has."""
    case = st["case"]
    b, h, hk, s, d, page, shared = (case[x] for x in ("batch", "heads", "kv_heads", "q", "dim", "page", "shared"))
    g = h // hk
    out = torch.zeros(b, s, h, d, dtype=torch.float64, device="cuda")
    table = st["table"].cpu().numpy()
    for i, n in enumerate(_lengths(case)):
        row = [int(table[0 if j < shared else i, j // page]) * page + j % page for j in range(n)]
        slot = torch.tensor(row, device="cuda")
        first = max(0, s - n)  # the queries before it stand before the sequence
        place = torch.arange(n - s + first, n, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")[None, :]
        hidden = key > place
        if case["window"]:
            hidden |= (key <= place - case["window"]) & (key >= case["sinks"])
        hidden = hidden.repeat(g, 1)
        for kv in range(hk):
            k, v = (p[slot // page, kv, slot % page] for p in pages)
            rows = q[i, kv * g: kv * g + g, first:].double().reshape(-1, d)
            x = torch.mm(rows, k.t()).mul_(st["scale"]).masked_fill_(hidden, -math.inf)
            o = torch.mm(x.sub_(torch.logsumexp(x, 1, keepdim=True)).exp_(), v)
            out[i, first:, kv * g: kv * g + g] = o.view(g, s - first, d).transpose(0, 1)
    return out

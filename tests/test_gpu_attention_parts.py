"""Attention whose keys are split into parts, at offsets past 32 bits, without
memory for workspaces, and over scores of -inf; against 64 bits."""
import ctypes

import numpy as np
import pytest

from attention_util import (EVERY, Placed, assert_within, attention, attention_grad, attention_reference, ints)
from trs_backend import abi
from trs_backend.abi import DeviceArray, check, layout_of

pytestmark = pytest.mark.gpu

ALLOCATION_FAILED = -1


def inputs(seed, B, H, hk, sq, sk, D):
    rng = np.random.default_rng(seed)
    return tuple(rng.standard_normal(s).astype(np.float32) for s in ((B, H, sq, D), (B, hk, sk, D), (B, hk, sk, D), (B, H, sq, D)))


def run(q, k, v, window, sinks, scale, lengths=None):
    P = [Placed(t) for t in (q, k, v)]
    out, rows = Placed(shape=q.shape), int(np.prod(q.shape[:3]))
    lse = DeviceArray(4 * rows)
    check(attention(*P, window, sinks, scale, out, lse, None if lengths is None else ints(lengths)))
    got = out.numpy(), lse.to_numpy(count=rows).reshape(q.shape[:3])
    assert out.untouched()
    return got


#        B  H hk  sq    sk    D  window sinks lengths
PARTS = [
    (1, 1, 1, 2500, 2500, 16, EVERY, 0, None),     # ten blocks of rows, from few keys to all
    (1, 4, 2, 900, 900, 64, EVERY, 0, None),
    (1, 2, 1, 1000, 1000, 128, 300, 5, None),
    (2, 2, 1, 300, 1100, 40, 700, 5, [1100, 130]),  # the second has no key for its first rows, and fewer parts
    (3, 6, 6, 500, 500, 80, 200, 3, [500, 0, 257]),
    (2, 1, 1, 600, 600, 96, EVERY, 0, [1, 599]),
    (1, 300, 300, 20, 20, 8, EVERY, 0, None),       # as many heads as CUs and more: no parts
    (1, 3, 1, 2, 3001, 64, EVERY, 0, None),         # few rows
    (2, 4, 4, 1, 2000, 128, 900, 70, [2000, 33]),
    (1, 1, 1, 500, 700, 160, EVERY, 0, None),       # wide heads
]


@pytest.mark.parametrize("shape", PARTS, ids=str)
def test_parts_join_to_the_whole(shape):
    *sizes, window, sinks, lengths = shape
    q, k, v, _ = inputs(sum(sizes), *sizes)
    want = attention_reference(q, k, v, window, sinks, np.float32(0.2), lengths)
    out, lse = run(q, k, v, window, sinks, 0.2, lengths)
    assert_within(out, *want["out"], "out")
    assert_within(lse, *want["lse"], "lse")


@pytest.mark.parametrize("D", [32, 128, 160])
@pytest.mark.parametrize("sq", [1, 40, 300])
def test_scores_of_minus_infinity(sq, D):
    """A key whose scores are -inf weighs nothing; a row that sees no other has none to
    weigh, 0/0, and a row that sees no key gives 0."""
    q, k, v, _ = inputs(5, 2, 2, 1, sq, 320, D)
    q[..., 0] = 1 + abs(q[..., 0])
    far = k.copy()
    far[:, :, 100] = 0
    far[:, :, 100, 0] = -np.inf
    out, _ = run(q, far, v, EVERY, 0, 0.2)
    others = [np.delete(t, 100, 2) for t in (k, v)]
    rows = slice(max(0, 101 - (320 - sq)), sq)  # those behind the key, all of which see it
    want = attention_reference(q[:, :, rows], *others, EVERY, 0, np.float32(0.2))
    assert_within(out[:, :, rows], *want["out"], "out beside a key of -inf")
    far[:, :, :, 0] = -np.inf
    lengths = [320, min(sq, 320) - 1]  # one row less than the queries: the first sees nothing
    out, lse = run(q, far, v, EVERY, 0, 0.2, lengths)
    assert np.isnan(out[0]).all() and np.isnan(out[1, :, 1:]).all() and (out[1, :, 0] == 0).all()
    assert (lse == -np.inf).all()


class Far:
    """A [1, 1, n, D] tensor whose tokens lie 2^24 floats apart in `buffer`."""
    STEP = 1 << 24

    def __init__(self, buffer, at, n, D, values=None):
        self.at, self.n, self.D, self.buffer = at, n, D, buffer
        self.layout = layout_of((1, 1, n, D), (n * self.STEP, n * self.STEP, self.STEP, 1), at)
        if values is not None:
            for i, row in enumerate(np.ascontiguousarray(values[0, 0])):
                check(abi.lib.trs_memcpy_h2d(self.row(i), row.ctypes.data, 4 * D))

    def row(self, i):
        return ctypes.c_void_p(self.buffer.addr + 4 * (self.at + i * self.STEP))

    def numpy(self):
        got = np.empty((1, 1, self.n, self.D), np.float32)
        for i in range(self.n):
            check(abi.lib.trs_memcpy_d2h(got[0, 0, i].ctypes.data, self.row(i), 4 * self.D))
        return got

    @property
    def arg(self):
        return self.buffer.ptr, ctypes.byref(self.layout)


@pytest.mark.parametrize("D, sq", [(64, 1), (64, 260), (160, 260)])
def test_offsets_past_32_bits(D, sq):
    """260 tokens over 17 GB: the last are 2^32 elements from the first."""
    n = 260
    inside, outside = (DeviceArray(4 * ((n - 1) * Far.STEP + 65536)) for _ in range(2))
    q, k, v, up = inputs(6, 1, 1, 1, sq, n, D)
    F = [Far(inside, 4096 * i, t.shape[2], D, t) for i, t in enumerate((q, k, v, up))]
    want = attention_reference(q, k, v, 200, 3, np.float32(0.2), up=up)
    lse = DeviceArray(4 * sq)
    out = Far(outside, 0, sq, D)
    check(attention(*F[:3], 200, 3, 0.2, out, lse))
    held = out.numpy()
    assert_within(held, *want["out"], "out")
    near = Placed(held)
    for far in ("dq", "dk", "dv"):
        grads = {name: Placed(shape=t.shape) for name, t in (("dq", q), ("dk", k), ("dv", v))}
        grads[far] = Far(outside, 0, grads[far].shape[2], D)
        check(attention_grad(*F[:3], 200, 3, 0.2, near, lse, F[3], *grads.values()))
        for name, g in grads.items():
            assert_within(g.numpy(), *want[name], name)
    for buffer in (inside, outside):
        buffer.free()
    check(abi.lib.trs_empty_cache())


def test_no_memory_for_workspaces():
    """The forward pass needs none (its parts are for speed); the gradients say so."""
    for sq, sk, D in ((1, 2000, 64), (600, 600, 64), (600, 600, 160)):
        q, k, v, up = inputs(9, 1, 2, 2, sq, sk, D)
        want = attention_reference(q, k, v, EVERY, 0, np.float32(0.2), up=up)
        P, out, lse = [Placed(t) for t in (q, k, v)], Placed(shape=q.shape), DeviceArray(4 * 2 * sq)
        U, grads = Placed(up), [Placed(shape=t.shape) for t in (q, k, v)]
        check(abi.lib.trs_debug_fail_allocs_after(0))
        try:
            done = attention(*P, EVERY, 0, 0.2, out, lse), attention_grad(*P, EVERY, 0, 0.2, out, lse, U, *grads)
        finally:
            check(abi.lib.trs_debug_fail_allocs_after(-1))
        assert done == (0, ALLOCATION_FAILED)
        assert_within(out.numpy(), *want["out"], "out")
        check(attention_grad(*P, EVERY, 0, 0.2, out, lse, U, *grads))
        for name, g in zip(("dq", "dk", "dv"), grads):
            assert_within(g.numpy(), *want[name], name)


def test_refusals_of_the_gradients():
    q, k, v, up = (Placed(t) for t in inputs(0, 2, 4, 2, 8, 8, 16))
    out, lse, g = Placed(shape=(2, 4, 8, 16)), DeviceArray(4 * 64), [Placed(shape=t.shape) for t in (q, k, v)]

    def refused(code, words, *args):
        assert attention_grad(*args) == code
        assert words in abi.lib.trs_last_error().decode()
    E, S = abi.TRS_E_INVALID_ARGUMENT, abi.TRS_E_SHAPE_MISMATCH
    refused(E, "window", q, k, v, 0, 0, 1.0, out, lse, up, *g)
    refused(S, "query gradient", q, k, v, 4, 0, 1.0, out, lse, up, g[1], g[1], g[2])
    refused(S, "key gradient", q, k, v, 4, 0, 1.0, out, lse, up, g[0], g[0], g[2])
    refused(S, "output", q, k, v, 4, 0, 1.0, k, lse, up, *g)
    refused(E, "overlaps", q, k, v, 4, 0, 1.0, out, lse, up, q, g[1], g[2])
    refused(E, "overlaps", q, k, v, 4, 0, 1.0, out, lse, up, up, g[1], g[2])
    turned = Placed(shape=(2, 2, 8, 16), order=(0, 1, 3, 2))
    refused(E, "unit stride", q, k, v, 4, 0, 1.0, out, lse, up, g[0], turned, g[2])
    assert abi.lib.trs_window_attention_backward_f32(
        *q.arg, *k.arg, *v.arg, None, 4, 0, 1.0, *out.arg, lse.ptr, up.dev.ptr, None, *g[0].arg, *g[1].arg, *g[2].arg) == E


#        H hk  tokens D  window sinks lengths   parts
SHIFTED = [
    (3, 1, 174, 16, 40, 0, [174, 134], 3),
    (3, 1, 174, 64, 66, 3, [161, 174], 3),
    (10, 2, 174, 40, 53, 3, [174, 134], 3),
    (6, 2, 211, 128, 40, 3, [211, 171], 3),
]


@pytest.mark.parametrize("shape", SHIFTED, ids=str)
def test_a_shorter_window_over_one_tile_more(shape):
    """A shorter sequence's window begins elsewhere in a tile of keys than the longest's and
    touches one tile more; all of its parts are computed.  What the workspace holds before
    is NaN."""
    H, hk, n, D, window, sinks, lengths, parts = shape
    q, k, v, _ = inputs(7, 2, H, hk, n, n, D)
    want = attention_reference(q, k, v, window, sinks, np.float32(0.2), lengths)
    DeviceArray.from_numpy(np.full(parts * 2 * H * n * (D + 2), np.nan, np.float32)).free()
    out, lse = run(q, k, v, window, sinks, 0.2, lengths)
    assert_within(out, *want["out"], "out")
    assert_within(lse, *want["lse"], "lse")


#        B  H hk  sq  sk   D  window sinks lengths
WHOLE = [
    (1, 8, 8, 1, 300, 64, EVERY, 0, None),     # few keys: blocks of 16 waves, no parts
    (1, 8, 2, 3, 383, 32, 200, 5, None),
    (3, 4, 2, 2, 290, 48, EVERY, 0, [290, 1, 0]),
    (1, 2, 1, 5, 257, 20, EVERY, 0, None),
    (1, 2, 2, 1, 260, 50, EVERY, 0, None),     # a width in parts all the same
    (2, 128, 128, 1, 500, 64, EVERY, 0, None),  # a head for every CU: blocks of 16 waves, and of 8
    (2, 128, 128, 1, 500, 80, 130, 7, None),
    (4, 64, 64, 2, 270, 128, EVERY, 0, None),
    (4, 128, 64, 1, 270, 100, EVERY, 0, [270, 33, 1, 0]),
]


@pytest.mark.parametrize("shape", WHOLE, ids=str)
def test_few_rows_in_blocks_of_many_waves(shape):
    *sizes, window, sinks, lengths = shape
    q, k, v, _ = inputs(8, *sizes)
    v[0, 0, sizes[4] - 1] = np.inf  # the last key: not seen by any but the last query
    seen_last = slice(sizes[3] - 1, sizes[3])
    want = attention_reference(q, k, np.where(np.isfinite(v), v, 0), window, sinks, np.float32(0.2), lengths)
    out, lse = run(q, k, v, window, sinks, 0.2, lengths)
    group = sizes[1] // sizes[2]
    assert np.isinf(out[0, :group, seen_last]).all()
    out[0, :group, seen_last] = want["out"][0][0, :group, seen_last]
    assert_within(out, *want["out"], "out")
    assert_within(lse, *want["lse"], "lse")

"""Sliding-window attention with first tokens that stay visible, against 64 bits:
lengths from none and one to several tiles, windows and sinks at tile borders,
shared key heads, ragged lengths, strides, hidden NaN, and the gradients by the
formula and by differences."""
import ctypes

import numpy as np
import pytest

from attention_util import (EVERY, Placed, assert_within, attention, attention_grad, attention_reference, ints, seen)
from trs_backend import abi
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu

TOKENS = (0, 2, 1, 3)  # [batch, token, head, dim] in memory


def inputs(seed, B, H, hk, sq, sk, D, std=1.0):
    rng = np.random.default_rng(seed)
    return tuple((std * rng.standard_normal(s)).astype(np.float32)
                 for s in ((B, H, sq, D), (B, hk, sk, D), (B, hk, sk, D), (B, H, sq, D)))


def run(q, k, v, window, sinks, scale, lengths=None, up=None, order=None, **place):
    """Every output as an array, by name."""
    P = [Placed(t, order=order, **place) for t in (q, k, v)]
    out = Placed(shape=q.shape, order=order)
    lse = DeviceArray(max(4, 4 * int(np.prod(q.shape[:3]))))
    lens = None if lengths is None else ints(lengths)
    check(attention(*P, window, sinks, scale, out, lse, lens))
    got = {"out": out.numpy(), "lse": lse.to_numpy(count=int(np.prod(q.shape[:3]))).reshape(q.shape[:3])}
    assert out.untouched()
    if up is not None:
        U = Placed(up, order=order, **place)
        grads = [Placed(shape=t.shape, order=order) for t in (q, k, v)]
        check(attention_grad(*P, window, sinks, scale, out, lse, U, *grads, lens))
        got.update(zip(("dq", "dk", "dv"), (g.numpy() for g in grads)))
        assert all(g.untouched() for g in grads)
    return got


def compare(got, want):
    for name, value in got.items():
        assert_within(value, *want[name], what=name)


#        B  H hk  sq   sk   D  window sinks
SHAPES = [
    (1, 1, 1, 1, 1, 1, 1, 0),
    (1, 1, 1, 1, 1, 32, 1, 1),
    (1, 2, 1, 1, 33, 64, 8, 2),         # one token over a cache
    (2, 4, 2, 1, 300, 128, 100, 4),
    (1, 8, 1, 2, 129, 80, EVERY, 0),
    (1, 1, 1, 5, 5, 7, EVERY, 0),       # a dim that no vector divides
    (1, 1, 1, 32, 32, 32, 32, 0),
    (1, 1, 1, 33, 33, 32, 1, 0),        # each query sees itself alone
    (1, 1, 1, 33, 33, 32, 1, 1),
    (2, 3, 3, 64, 64, 64, 31, 2),
    (1, 2, 2, 129, 129, 96, 32, 32),    # sinks that fill a tile
    (1, 2, 1, 130, 130, 128, 33, 33),   # and one more
    (1, 4, 2, 200, 200, 33, 64, 5),
    (1, 6, 2, 257, 257, 128, 50, 3),    # three query heads a key head
    (1, 5, 1, 140, 140, 64, EVERY, 0),  # five
    (1, 2, 1, 100, 100, 256, 40, 6),
    (1, 1, 1, 70, 70, 129, 40, 6),
    (1, 1, 1, 300, 300, 200, 20, 40),   # more sinks than window
    (2, 2, 1, 40, 25, 48, 9, 2),        # more queries than keys: the first see nothing
    (1, 2, 2, 17, 400, 64, 64, 4),      # the end of a prompt over a cache
    (1, 2, 2, 200, 333, 16, 1000, 8),   # a window longer than the keys
    (1, 32, 4, 40, 40, 64, 16, 1),
    (1, 1, 1, 700, 700, 32, 8, 1),      # rows far past the sinks, by many tiles
    (1, 4, 1, 1000, 1000, 24, 30, 70),  # sinks of three tiles
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_and_its_gradients_match_64_bits(shape):
    B, H, hk, sq, sk, D, window, sinks = shape
    q, k, v, up = inputs(sq * 7 + D, B, H, hk, sq, sk, D)
    scale = 1 / np.sqrt(D)
    compare(run(q, k, v, window, sinks, scale, up=up, order=TOKENS),
            attention_reference(q, k, v, window, sinks, np.float32(scale), up=up))


@pytest.mark.parametrize("lengths", [[0, 1, 90], [90, 31, 32], [33, 64, 65], [-5, 1000, 7]], ids=str)
@pytest.mark.parametrize("sq", [1, 40])
def test_sequences_of_their_own_lengths(sq, lengths):
    """Lengths of none and one; those out of range are taken into it."""
    q, k, v, up = inputs(sq, 3, 4, 2, sq, 90, 40)
    args = (20, 3, 0.2)
    compare(run(q, k, v, *args, lengths=lengths, up=up), attention_reference(q, k, v, *args[:2], np.float32(0.2), lengths, up))


def test_no_keys_and_no_queries():
    q, k, v, up = inputs(0, 2, 2, 1, 3, 0, 16)
    got = run(q, k, v, 4, 1, 1.0, up=up)
    assert not got["out"].any() and (got["lse"] == -np.inf).all() and not got["dq"].any() and got["dk"].size == 0
    q, k, v, up = inputs(0, 2, 2, 1, 0, 70, 16)
    got = run(q, k, v, 4, 1, 1.0, up=up)
    assert got["out"].size == 0 and not got["dk"].any() and not got["dv"].any()
    q, k, v, up = inputs(0, 0, 2, 1, 3, 3, 16)
    assert run(q, k, v, 4, 1, 1.0, up=up)["dq"].size == 0


PLACES = [
    {"order": (0, 1, 2, 3), "offset": 3},       # rows at any float
    {"order": TOKENS, "pad": 5},                # rows of odd pitch
    {"order": (2, 0, 1, 3)},                    # tokens slowest
    {"order": (0, 1, 2, 3), "step": 2},         # a dim with a stride: copied
    {"order": (0, 1, 3, 2)},                    # tokens fastest: copied
]


@pytest.mark.parametrize("place", PLACES, ids=str)
@pytest.mark.parametrize("D", [30, 64])
def test_strides_and_orders(D, place):
    q, k, v, up = inputs(5, 2, 4, 2, 70, 70, D)
    place = dict(place)
    order = place.pop("order")
    P = [Placed(t, order=order, **place) for t in (q, k, v, up)]
    out, lse = Placed(shape=q.shape, order=TOKENS, pad=3, offset=1), DeviceArray(4 * 2 * 4 * 70)
    check(attention(*P[:3], 30, 2, 0.1, out, lse))
    grads = [Placed(shape=t.shape, order=(1, 2, 0, 3), pad=1) for t in (q, k, v)]
    check(attention_grad(*P[:3], 30, 2, 0.1, out, lse, P[3], *grads))
    want = attention_reference(q, k, v, 30, 2, np.float32(0.1), up=up)
    compare({"out": out.numpy(), **dict(zip(("dq", "dk", "dv"), (g.numpy() for g in grads)))}, want)
    assert out.untouched() and all(g.untouched() for g in grads)


def test_a_broadcast_key_head_and_value():
    """Strides of 0: one key head and one batch's values read by all."""
    q, k, v, _ = inputs(11, 2, 2, 2, 50, 50, 32)
    k[:, 1] = k[:, 0]
    v[1] = v[0]
    pq, pk, pv, out = Placed(q), Placed(k), Placed(v), Placed(shape=q.shape)
    pk.layout.stride[1] = 0
    pv.layout.stride[0] = 0
    check(attention(pq, pk, pv, 20, 1, 0.2, out))
    assert_within(out.numpy(), *attention_reference(q, k, v, 20, 1, np.float32(0.2))["out"])


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf, 3e38])
@pytest.mark.parametrize("D", [32, 128, 160])
def test_what_a_query_does_not_see_does_not_reach_it(D, bad):
    """Infinities, NaN and the largest values in keys, values, queries and upstream
    rows: outputs whose pairs leave them out are as without them."""
    B, H, hk, n, window, sinks = 1, 2, 1, 150, 40, 3
    q, k, v, up = inputs(3, B, H, hk, n, n, D)
    want = attention_reference(q, k, v, window, sinks, np.float32(0.1), up=up)
    mask = seen(n, n, window, sinks)
    at = 71
    sees_key = mask[:, at]
    # A value: rows that do not see it.
    v2 = v.copy()
    v2[0, 0, at] = bad
    got = run(q, k, v2, window, sinks, 0.1)
    assert_within(got["out"][:, :, ~sees_key], *(t[:, :, ~sees_key] for t in want["out"]), "out past a bad value")
    if not np.isfinite(bad):
        assert not np.isfinite(got["out"][:, :, sees_key]).any()
    # A key: the same, and the gradients of those rows.
    k2 = k.copy()
    k2[0, 0, at] = bad
    got = run(q, k2, v, window, sinks, 0.1, up=up)
    for name in ("out", "dq"):
        assert_within(got[name][:, :, ~sees_key], *(t[:, :, ~sees_key] for t in want[name]), name + " past a bad key")
    # A query, and an upstream row: keys that it does not see.
    unseen = ~mask[at]
    q2, up2 = q.copy(), up.copy()
    q2[0, 0, at] = bad
    got = run(q2, k, v, window, sinks, 0.1, up=up)
    for name in ("dk", "dv"):
        assert_within(got[name][:, :, unseen], *(t[:, :, unseen] for t in want[name]), name + " past a bad query")
    up2[0, 0, at] = bad
    got = run(q, k, v, window, sinks, 0.1, up=up2)
    for name in ("dk", "dv"):
        assert_within(got[name][:, :, unseen], *(t[:, :, unseen] for t in want[name]), name + " past a bad upstream row")


def test_keys_past_a_sequence_and_rows_before_it_are_not_read():
    """A cache's tail and the queries before a sequence hold NaN."""
    q, k, v, up = inputs(8, 2, 2, 1, 20, 100, 64)
    lengths = [70, 11]
    want = attention_reference(q, k, v, 30, 2, np.float32(0.2), lengths, up)
    for b, n in enumerate(lengths):
        k[b, :, n:] = v[b, :, n:] = np.nan
        if n < 20:
            q[b, :, :20 - n] = up[b, :, :20 - n] = np.nan
    compare(run(q, k, v, 30, 2, 0.2, lengths=lengths, up=up), want)


def test_large_scores_and_scales_of_either_sign():
    q, k, v, up = inputs(21, 1, 2, 2, 90, 90, 64, std=3.0)
    for scale in (2.0, -0.5, 0.0):
        compare(run(q, k, v, 50, 1, scale, up=up), attention_reference(q, k, v, 50, 1, np.float32(scale), up=up))


def test_the_same_bits_each_time():
    q, k, v, up = inputs(2, 2, 8, 2, 400, 400, 64)
    first, second = (run(q, k, v, 100, 4, 0.125, up=up, order=TOKENS) for _ in range(2))
    for name in first:
        assert np.array_equal(first[name].view(np.uint32), second[name].view(np.uint32)), name


@pytest.mark.parametrize("shape", [(1, 4, 2, 60, 60, 24, 16, 3), (1, 2, 2, 30, 50, 32, EVERY, 0)], ids=str)
def test_gradients_match_differences_of_the_definition(shape):
    """<gradient, direction> against a central difference of the 64-bit output.
    The difference is off by O(step^2) of the third derivative (below 1e-6 of
    the sum of magnitudes here) and the gradient by its bound."""
    B, H, hk, sq, sk, D, window, sinks = shape
    q, k, v, up = inputs(31, B, H, hk, sq, sk, D)
    got = run(q, k, v, window, sinks, 0.2, up=up)
    want = attention_reference(q, k, v, window, sinks, np.float32(0.2), up=up)
    rng = np.random.default_rng(4)
    for at, name in enumerate(("dq", "dk", "dv")):
        ways = [rng.standard_normal(t.shape) if i == at else np.zeros(t.shape) for i, t in enumerate((q, k, v))]
        step = 1e-4
        ends = [(attention_reference(*(t + s * step * w for t, w in zip((q, k, v), ways)), window, sinks, np.float32(0.2))["out"][0]
                 * up).sum() for s in (1, -1)]
        slope = (ends[0] - ends[1]) / (2 * step)
        mine = (got[name].astype(np.float64) * ways[at]).sum()
        size = (abs(want[name][0]) * abs(ways[at])).sum()
        assert abs(mine - slope) <= (want[name][1] * abs(ways[at])).sum() + 1e-6 * size, name


def refused(rc, code, words):
    assert rc == code, (rc, abi.lib.trs_last_error())
    message = abi.lib.trs_last_error().decode()
    assert words in message, message


def test_refusals():
    q, k, v, up = (Placed(t) for t in inputs(0, 2, 4, 2, 8, 8, 16))
    out, lse = Placed(shape=(2, 4, 8, 16)), DeviceArray(4 * 64)
    E = abi.TRS_E_INVALID_ARGUMENT
    S = abi.TRS_E_SHAPE_MISMATCH
    refused(attention(q, k, v, 0, 0, 1.0, out), E, "window")
    refused(attention(q, k, v, 4, -1, 1.0, out), E, "sinks")
    refused(attention(q, k, v, 4, 0, float("nan"), out), E, "scale")
    refused(attention(q, k, v, 4, 0, float("inf"), out), E, "scale")
    refused(attention(q, k, v, 4, 0, 1.0, k), S, "output")
    refused(attention(q, Placed(shape=(2, 3, 8, 16)), Placed(shape=(2, 3, 8, 16)), 4, 0, 1.0, out), S, "cannot share")
    refused(attention(q, k, Placed(shape=(2, 2, 9, 16)), 4, 0, 1.0, out), S, "value")
    refused(attention(q, Placed(shape=(2, 2, 8, 15)), v, 4, 0, 1.0, out), S, "key")
    refused(attention(Placed(shape=(4, 8, 16)), k, v, 4, 0, 1.0, out), E, "rank")
    wide = [Placed(shape=(1, 1, 2, 257)) for _ in range(4)]
    refused(attention(*wide[:3], 4, 0, 1.0, wide[3]), E, "head dim")
    refused(attention(q, k, v, 4, 0, 1.0, Placed(shape=(2, 4, 8, 16), order=(0, 1, 3, 2))), E, "unit stride")
    flat = Placed(shape=(2, 4, 8, 16))
    flat.layout.stride[1] = 0
    refused(attention(q, k, v, 4, 0, 1.0, flat), E, "overlaps itself")
    refused(attention(q, k, v, 4, 0, 1.0, q), E, "overlaps")
    null = Placed(shape=(2, 4, 8, 16))
    null.dev = type("Null", (), {"ptr": None})()
    refused(attention(q, k, v, 4, 0, 1.0, null), E, "null")
    g = [Placed(shape=t.shape) for t in (q, k, v)]
    refused(attention_grad(q, k, v, 4, 0, 1.0, out, None, up, *g), E, "lse")
    refused(attention_grad(q, k, v, 4, 0, 1.0, out, lse, up, g[0], g[1], g[1]), E, "overlaps")
    refused(attention_grad(q, k, v, 4, 0, 1.0, out, lse, k, *g), S, "upstream")
    huge = Placed(shape=(2, 4, 8, 16))
    huge.layout.shape[2] = 1 << 31
    huge.layout.stride[2] = 0
    refused(attention(huge, k, v, 4, 0, 1.0, huge), abi.ERROR_NAMES and -2, "2^30")
    assert ctypes.sizeof(ctypes.c_void_p) == 8

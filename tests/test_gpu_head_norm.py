"""The norm of each head's vectors with the rotation by position, and its
gradients, against 64 bits and against differences."""
import numpy as np
import pytest

from attention_util import Placed, U, assert_within, ints, norm_rope, norm_rope_reference, rotation_tables
from trs_backend import abi
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu
TOKENS = (0, 2, 1, 3)
EPS = 1e-6


def make(seed, B, H, S, D):
    rng = np.random.default_rng(seed)
    x, up = (rng.standard_normal((B, H, S, D)).astype(np.float32) for _ in range(2))
    return x, up, (1 + 0.2 * rng.standard_normal(D)).astype(np.float32)


def bounds(x, w, up=None):
    """How far fp32 may be off.  y: the mean's (D+2) u halves in r, then five
    roundings of |x| r |w|, of both partners.  dx and dw: the same of sums of
    magnitudes, over D entries or all rows."""
    D = x.shape[-1]
    x, w = abs(x.astype(np.float64)), abs(np.ones(D) if w is None else w.astype(np.float64))
    r = 1 / np.sqrt((x * x).mean(-1, keepdims=True) + EPS)
    if up is None:
        return (D / 2 + 12) * U * 2 * (x * w).max(-1, keepdims=True) * r * np.ones(D)
    g = 2 * abs(up.astype(np.float64)).max(-1, keepdims=True)
    dot = (w * g * x).mean(-1, keepdims=True)
    dx = (3 * D + 24) * U * r * (w * g + x * r * r * dot)
    rows = x.size / D
    dw = (rows + D + 24) * U * (g * x * r).sum((0, 1, 2))
    return dx, dw


def run(tensors, ws, rot, interleaved, positions=None, start=0, rows=None, grad=False, order=TOKENS, **place):
    B, _, S, D = tensors[0][0].shape
    rows = rows if rows is not None else start + S
    cos, sin = rotation_tables(rows, rot)
    C, Sn = Placed(cos, pad=2), Placed(sin, pad=2)
    X = [Placed(x, order=order, **place) for x, _ in tensors]
    outs = [Placed(shape=x.shape, order=TOKENS, pad=1) for x, _ in tensors]
    W = [None if w is None else DeviceArray.from_numpy(w) for w in ws]
    pos = None if positions is None else ints(positions)
    if not grad:
        check(norm_rope(X, W, EPS, C, Sn, interleaved, pos, start, outs))
        got = [o.numpy() for o in outs]
    else:
        UP = [Placed(u, order=order, **place) for _, u in tensors]
        dw = [DeviceArray(4 * D) for _ in tensors]
        check(norm_rope(X, W, EPS, C, Sn, interleaved, pos, start, outs, UP, dw))
        got = [(o.numpy(), d.to_numpy()) for o, d in zip(outs, dw)]
    assert all(o.untouched() for o in outs)
    at = np.broadcast_to(start + np.arange(S), (B, S)) if positions is None else np.asarray(positions)
    return got, cos, sin, at


#        B  Hq Hk  S    D   rot  interleaved
SHAPES = [
    (1, 1, 1, 1, 2, 2, False), (1, 2, 1, 3, 8, 8, True), (2, 4, 2, 5, 16, 16, False), (1, 3, 1, 33, 64, 64, False),
    (2, 8, 2, 17, 128, 128, False), (1, 4, 4, 9, 128, 128, True), (1, 2, 1, 70, 80, 80, False), (1, 2, 1, 7, 96, 96, True),
    (1, 1, 1, 20, 256, 256, False), (1, 1, 1, 3, 512, 512, True), (1, 2, 2, 6, 64, 32, False), (1, 2, 1, 6, 64, 32, True),
    (1, 2, 1, 11, 6, 6, False), (1, 1, 1, 5, 7, 4, True), (1, 1, 1, 4, 1000, 1000, False), (1, 2, 1, 5, 50, 0, False),
    (3, 5, 3, 300, 32, 32, False), (1, 1, 1, 2, 1024, 512, True),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_norm_and_rotation_match_64_bits(shape):
    B, hq, hk, S, D, rot, inter = shape
    (xq, _, wq), (xk, _, wk) = make(1, B, hq, S, D), make(2, B, hk, S, D)
    got, cos, sin, at = run([(xq, None), (xk, None)], [wq, wk], rot, inter, start=3)
    for y, x, w in zip(got, (xq, xk), (wq, wk)):
        assert_within(y, norm_rope_reference(x, w, EPS, cos, sin, at, inter), bounds(x, w))


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_match_64_bits(shape):
    B, hq, hk, S, D, rot, inter = shape
    (xq, uq, wq), (xk, uk, wk) = make(3, B, hq, S, D), make(4, B, hk, S, D)
    got, cos, sin, at = run([(xq, uq), (xk, uk)], [wq, wk], rot, inter, grad=True)
    for (dx, dw), x, u, w in zip(got, (xq, xk), (uq, uk), (wq, wk)):
        want, bound = norm_rope_reference(x, w, EPS, cos, sin, at, inter, u), bounds(x, w, u)
        assert_within(dx, want[0], bound[0], "dx")
        assert_within(dw, want[1], bound[1], "dw")


# Eights that pass beside eights that are turned.
PARTIAL = [(1, 3, 1, 9, 80, 40, False), (2, 2, 1, 33, 96, 16, True), (1, 2, 2, 5, 128, 8, False), (1, 5, 1, 70, 64, 0, False),
           (1, 1, 1, 130, 24, 8, False), (1, 2, 1, 3, 512, 256, False), (2, 3, 1, 17, 256, 248, True)]


@pytest.mark.parametrize("shape", PARTIAL, ids=str)
def test_part_of_a_head_turned(shape):
    B, hq, hk, S, D, rot, inter = shape
    (xq, uq, wq), (xk, uk, wk) = make(11, B, hq, S, D), make(12, B, hk, S, D)
    got, cos, sin, at = run([(xq, None), (xk, None)], [wq, wk], rot, inter, start=2)
    for y, x, w in zip(got, (xq, xk), (wq, wk)):
        assert_within(y, norm_rope_reference(x, w, EPS, cos, sin, at, inter), bounds(x, w))
    got, cos, sin, at = run([(xq, uq), (xk, uk)], [wq, wk], rot, inter, grad=True)
    for (dx, dw), x, u, w in zip(got, (xq, xk), (uq, uk), (wq, wk)):
        want, bound = norm_rope_reference(x, w, EPS, cos, sin, at, inter, u), bounds(x, w, u)
        assert_within(dx, want[0], bound[0], "dx")
        assert_within(dw, want[1], bound[1], "dw")


@pytest.mark.parametrize("place", [{"order": (0, 1, 2, 3), "offset": 1}, {"order": TOKENS, "pad": 3}, {"order": (0, 1, 2, 3), "step": 2},
                                   {"order": (3, 2, 1, 0)}], ids=str)
def test_strides_and_orders_without_a_weight(place):
    x, u, _ = make(5, 2, 3, 10, 64)
    got, cos, sin, at = run([(x, u)], [None], 64, False, **place)
    assert_within(got[0], norm_rope_reference(x, None, EPS, cos, sin, at, False), bounds(x, None))
    got, cos, sin, at = run([(x, u)], [None], 64, False, grad=True, **place)
    want, bound = norm_rope_reference(x, None, EPS, cos, sin, at, False, u), bounds(x, None, u)
    assert_within(got[0][0], want[0], bound[0])
    assert_within(got[0][1], want[1], bound[1])


@pytest.mark.parametrize("D", [64, 20])
def test_positions_of_their_own_and_ones_the_tables_do_not_hold(D):
    x, u, w = make(6, 2, 3, 4, D)
    positions = np.array([[5, 0, 9, 9], [-1, 3, 10, 2_000_000_000]])
    cos, sin = rotation_tables(10, D)
    known = (positions >= 0) & (positions < 10)
    at = np.where(known, positions, 0)
    got, *_ = run([(x, u)], [w], D, False, positions=positions, rows=10)
    rows = np.broadcast_to(known[:, None], (2, 3, 4))
    assert_within(got[0][rows], norm_rope_reference(x, w, EPS, cos, sin, at, False)[rows], bounds(x, w)[rows])
    assert np.isnan(got[0][~rows]).all()
    got, *_ = run([(x, u)], [w], D, False, positions=positions, rows=10, grad=True)
    assert_within(got[0][0][rows], norm_rope_reference(x, w, EPS, cos, sin, at, False, u)[0][rows], bounds(x, w, u)[0][rows])
    assert np.isnan(got[0][0][~rows]).all()


def test_zero_rows_and_values_that_are_not_finite_stay_in_their_rows():
    x, u, w = make(7, 1, 2, 6, 64)
    x[0, 0, 1] = 0
    bad = x.copy()
    bad[0, 1, 2, 5] = np.nan
    bad[0, 1, 3, 5] = np.inf
    want = norm_rope_reference(x, w, EPS, *rotation_tables(6, 64), np.arange(6)[None], False)
    got, *_ = run([(bad, u)], [w], 64, False)
    fine = np.ones((1, 2, 6), bool)
    fine[0, 1, 2:4] = False
    assert_within(got[0][fine], want[fine], bounds(x, w)[fine])
    assert np.isnan(got[0][0, 1, 2]).all() and np.isnan(got[0][0, 1, 3]).any()


def test_gradients_match_differences_of_the_definition():
    """Central differences in 64 bits, off by O(step^2): 1e-6 of the magnitudes here."""
    x, u, w = make(8, 1, 2, 7, 32)
    got, cos, sin, at = run([(x, u)], [w], 32, True, grad=True)
    rng = np.random.default_rng(0)
    vx, vw = rng.standard_normal(x.shape), rng.standard_normal(w.shape)

    def value(dx, dw):
        return (norm_rope_reference(x + dx, w + dw, EPS, cos, sin, at, True) * u).sum()

    step = 1e-4
    want, bound = norm_rope_reference(x, w, EPS, cos, sin, at, True, u), bounds(x, w, u)
    for i, (v, ends) in enumerate(((vx, [value(s * step * vx, 0) for s in (1, -1)]), (vw, [value(0, s * step * vw) for s in (1, -1)]))):
        slope = (ends[0] - ends[1]) / (2 * step)
        assert abs((got[0][i] * v).sum() - slope) <= (bound[i] * abs(v)).sum() + 1e-6 * (abs(want[i]) * abs(v)).sum()


def test_no_rows_give_no_weight_gradient_and_refusals():
    x, u, w = make(9, 1, 2, 0, 16)
    got, *_ = run([(x, u)], [w], 16, False, rows=4, grad=True)
    assert not got[0][1].any()
    x, _, w = make(9, 1, 2, 4, 16)
    X, Y, W = Placed(x), Placed(shape=x.shape), DeviceArray.from_numpy(w)
    C, S = (Placed(t) for t in rotation_tables(4, 16))
    E, M = abi.TRS_E_INVALID_ARGUMENT, abi.TRS_E_SHAPE_MISMATCH

    def call(xs=(X,), ws=(W,), eps=EPS, c=C, s=S, start=0, outs=(Y,)):
        return norm_rope(list(xs), list(ws), eps, c, s, False, None, start, list(outs))

    assert call() == 0
    assert call(start=1) == E and call(start=-1) == E and call(eps=-1.0) == E and call(eps=float("inf")) == E
    assert call(outs=(X,)) == E
    assert call(outs=(Placed(shape=(1, 2, 4, 15)),)) == M
    assert call(xs=(Placed(shape=(2, 4, 16)),)) == E
    assert call(xs=(X, Placed(shape=(1, 2, 5, 16))), ws=(W, W), outs=(Y, Placed(shape=(1, 2, 5, 16)))) == M
    assert call(xs=(X, X), ws=(W, W), outs=(Y, Y)) == E
    big = [Placed(t) for t in rotation_tables(4, 18)]
    assert call(c=big[0], s=big[1]) == M
    assert call(xs=(Placed(shape=(1, 1, 1, 1025)),), outs=(Placed(shape=(1, 1, 1, 1025)),), ws=(None,)) == E

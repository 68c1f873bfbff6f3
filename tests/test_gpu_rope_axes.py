"""The rotation by positions of several axes, and its gradient, against 64 bits."""
import numpy as np
import pytest

import torch_rs
from attention_util import Placed, assert_within, ints, rotation_tables
from paged_util import rope, turned, turned_bound
from trs_backend import abi
from trs_backend.abi import check

pytestmark = pytest.mark.gpu
TOKENS = (0, 2, 1, 3)  # [batch, token, head, dim] in memory
F = torch_rs.nn.functional


def make(seed, B, H, S, D):
    return np.random.default_rng(seed).standard_normal((B, H, S, D)).astype(np.float32)


def run(xs, pairs, axes=1, pair_axes=None, positions=None, start=0, interleaved=False, inverse=False, rows=None, order=TOKENS, out_order=TOKENS, **place):
    B, _, S, _ = xs[0].shape
    rows = rows if rows is not None else (start + S if positions is None else int(np.max(positions)) + 1)
    cos, sin = rotation_tables(rows, 2 * pairs)
    C, N = Placed(cos, pad=2), Placed(sin, pad=2)
    X, outs = [Placed(x, order=order, **place) for x in xs], [Placed(shape=x.shape, order=out_order, pad=1) for x in xs]
    pos = None if positions is None else ints(positions)
    check(rope(X, C, N, interleaved, axes, pair_axes, pos, start, inverse, outs))
    got = [o.numpy() for o in outs]
    assert all(o.untouched() for o in outs)
    at = np.broadcast_to(start + np.arange(S), (axes, B, S)) if positions is None else positions
    for y, x in zip(got, xs):
        assert_within(y, turned(x, cos, sin, at, pair_axes, interleaved, inverse), turned_bound(x, pairs, interleaved))
    return got


#        B  Hq Hk  S    D  pairs axes interleaved
SHAPES = [
    (1, 1, 1, 1, 2, 1, 1, False), (2, 4, 2, 1, 128, 64, 3, False), (1, 3, 1, 33, 64, 32, 3, False), (2, 8, 2, 17, 128, 64, 3, True),
    (1, 2, 1, 70, 80, 40, 2, False), (1, 2, 1, 7, 96, 48, 4, True), (1, 1, 1, 20, 256, 128, 3, False), (1, 2, 2, 6, 64, 16, 2, False),
    (1, 2, 1, 6, 64, 16, 2, True), (1, 2, 1, 11, 6, 3, 2, False), (1, 1, 1, 5, 7, 2, 2, True), (1, 1, 1, 4, 1000, 500, 4, False),
    (1, 2, 1, 5, 50, 0, 1, False), (3, 5, 3, 300, 32, 16, 3, False), (1, 1, 1, 2, 1024, 256, 4, True), (1, 7, 5, 130, 24, 12, 3, False),
    (1, 13, 2, 3, 40, 8, 3, False), (2, 1, 6, 257, 72, 36, 2, True), (1, 64, 8, 2, 128, 64, 3, False),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("inverse", [False, True])
def test_rotation_matches_64_bits(shape, inverse):
    B, hq, hk, S, D, pairs, axes, inter = shape
    rng = np.random.default_rng(S)
    positions = rng.integers(0, 50, (axes, B, S))
    pair_axes = rng.integers(0, axes, pairs).tolist()  # any axis for any pair
    run([make(1, B, hq, S, D), make(2, B, hk, S, D)], pairs, axes, pair_axes, positions, interleaved=inter, inverse=inverse)
    sections = np.sort(pair_axes).tolist()  # and in runs
    run([make(3, B, hq, S, D)], pairs, axes, sections, positions, interleaved=inter, inverse=inverse)


@pytest.mark.parametrize("place", [{"order": (0, 1, 2, 3), "offset": 1}, {"order": TOKENS, "pad": 3}, {"order": (0, 1, 2, 3), "step": 2},
                                   {"order": (3, 2, 1, 0)}, {"order": (2, 0, 1, 3)}], ids=str)
@pytest.mark.parametrize("out_order", [(0, 1, 2, 3), TOKENS, (3, 0, 1, 2)], ids=str)
def test_strides_and_orders(place, out_order):
    x = [make(5, 2, 3, 10, 64), make(6, 2, 2, 10, 64)]
    run(x, 32, 1, None, None, start=3, out_order=out_order, **place)
    run(x, 24, 2, [0, 1] * 12, np.random.default_rng(0).integers(0, 9, (2, 2, 10)), out_order=out_order, interleaved=True, **place)


@pytest.mark.parametrize("D", [64, 20])
def test_a_pair_whose_position_the_tables_do_not_hold_is_nan(D):
    x = make(6, 2, 3, 4, D)
    positions = np.array([[[5, 0, 9, 9], [1, 3, 2, 2]], [[-1, 3, 10, 2_000_000_000], [9, -2_000_000_000, 0, 4]]])
    got = run([x], D // 2, 2, [0, 1] * (D // 4), positions, rows=10)[0]
    assert np.isnan(got[0, :, 0]).any() and not np.isnan(got[0, :, 0]).all() and not np.isnan(got[0, :, 1]).any()


def test_values_that_are_not_finite_stay_in_their_pairs():
    x = make(7, 1, 2, 6, 64)
    x[0, 1, 2, 5], x[0, 1, 3, 40] = np.nan, np.inf
    cos, sin = rotation_tables(6, 64)
    out = Placed(shape=x.shape)
    check(rope([Placed(x)], Placed(cos), Placed(sin), False, 1, None, None, 0, False, [out]))
    bad = ~np.isfinite(out.numpy())
    want = np.zeros(x.shape, bool)
    want[0, 1, 2, [5, 37]] = want[0, 1, 3, [8, 40]] = True
    assert (bad == want).all()


@pytest.mark.parametrize("shape", [(2, 3, 5, 64, 32), (1, 2, 4, 10, 3)], ids=str)
def test_an_output_may_be_its_inputs_own_view(shape):
    B, H, S, D, pairs = shape
    x = [make(8, B, H, S, D), make(9, B, H + 1, S, D)]
    cos, sin = rotation_tables(S, 2 * pairs)
    X = [Placed(t, order=TOKENS, pad=1) for t in x]
    check(rope(X, Placed(cos), Placed(sin), False, 1, None, None, 0, False, X))
    for p, t in zip(X, x):
        assert_within(p.numpy(), turned(t, cos, sin, np.broadcast_to(np.arange(S), (1, B, S)), None, False), turned_bound(t, pairs, False))
        assert p.untouched()


def test_the_inverse_is_the_gradient_by_differences():
    """The rotation is linear: differences of the definition in 64 bits are exact to their rounding."""
    x, up = make(10, 1, 2, 7, 32), make(11, 1, 2, 7, 32)
    positions = np.random.default_rng(1).integers(0, 30, (3, 1, 7))
    axes = [i % 3 for i in range(16)]
    cos, sin = rotation_tables(30, 32)
    back = run([up], 16, 3, axes, positions, inverse=True, rows=30)[0].astype(np.float64)
    rng = np.random.default_rng(2)
    for _ in range(4):
        d = rng.standard_normal(x.shape)
        ends = [(turned(x + s * d, cos, sin, positions, axes, False) * up).sum() for s in (1, -1)]
        assert abs((back * d).sum() - (ends[0] - ends[1]) / 2) <= (turned_bound(up, 16, False) * abs(d)).sum() + 1e-9


def test_through_torch_rs_with_its_gradient():
    q, k = make(12, 2, 4, 9, 16), make(13, 2, 2, 9, 16)
    positions = np.random.default_rng(3).integers(0, 20, (2, 2, 9))
    axes = [0] * 3 + [1] * 5
    cos, sin = rotation_tables(20, 16)
    Q, K, C, N = (torch_rs.tensor(t, device="cuda", requires_grad=g) for t, g in ((q, True), (k, True), (cos, False), (sin, False)))
    a, b = F.rope_axes(Q, K, C, N, positions=positions, pair_axes=axes)
    assert a._grad_fn_name == b._grad_fn_name == "RopeAxesBackward0"
    assert_within(a.numpy(), turned(q, cos, sin, positions, axes, False), turned_bound(q, 8, False))
    w = make(14, 2, 4, 9, 16), make(15, 2, 2, 9, 16)
    loss = (a * torch_rs.tensor(w[0], device="cuda")).sum() + (b * torch_rs.tensor(w[1], device="cuda")).sum()
    loss.backward()
    for x, u in ((Q, w[0]), (K, w[1])):
        assert_within(x.grad.numpy(), turned(u, cos, sin, positions, axes, False, True), turned_bound(u, 8, False))
    one = F.rope_axes(Q.detach(), None, C, N, start=4, interleaved=True)
    assert one._grad_fn_name is None
    assert_within(one.numpy(), turned(q, cos, sin, np.broadcast_to(4 + np.arange(9), (1, 2, 9)), None, True), turned_bound(q, 8, True))


def test_refusals_and_calls_without_elements():
    x = make(9, 1, 2, 4, 16)
    X, Y = Placed(x), Placed(shape=x.shape)
    C, S = (Placed(t) for t in rotation_tables(4, 16))
    E, M = abi.TRS_E_INVALID_ARGUMENT, abi.TRS_E_SHAPE_MISMATCH

    def call(xs=(X,), c=C, s=S, axes=1, pair_axes=None, start=0, outs=(Y,)):
        return rope(list(xs), c, s, False, axes, pair_axes, None, start, False, list(outs))

    assert call() == 0 and call(axes=4, pair_axes=[3] * 8) == 0
    assert call(start=1) == E and call(start=-1) == E and call(axes=0) == E and call(axes=5) == E and call(axes=2, pair_axes=[0] * 7 + [2]) == E
    assert call(xs=(X, Placed(x)), outs=(Y, X)) == E and call(xs=(X, X), outs=(Y, Y)) == E
    assert call(outs=(Placed(shape=(1, 2, 4, 15)),)) == M
    assert call(xs=(Placed(shape=(2, 4, 16)),)) == E
    assert call(xs=(X, Placed(shape=(1, 2, 5, 16))), outs=(Y, Placed(shape=(1, 2, 5, 16)))) == M
    big = [Placed(t) for t in rotation_tables(4, 18)]
    assert call(c=big[0], s=big[1]) == M
    assert call(xs=(Placed(shape=(1, 1, 1, 1025)),), outs=(Placed(shape=(1, 1, 1, 1025)),)) == E
    for shape in ((0, 2, 4, 16), (1, 0, 4, 16), (1, 2, 0, 16)):
        assert call(xs=(Placed(shape=shape),), outs=(Placed(shape=shape),)) == 0

"""Dropout from a counter-based generator: bit-exact against numpy's words, at odd
sizes, strides, orders and probabilities."""
import numpy as np
import pytest

from attention_util import Placed, dropout, dropout_reference
from helpers import assert_bitwise_equal
from trs_backend import abi
from trs_backend.abi import check

pytestmark = pytest.mark.gpu
BIG = (1 << 64) - 3


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 255, 1024, 4097, 100_003])
@pytest.mark.parametrize("p,seed,offset", [(0.1, 7, 0), (0.5, BIG, 12345678901), (0.999, 0, BIG)])
def test_flat(n, p, seed, offset):
    x = np.random.default_rng(n).standard_normal(n).astype(np.float32)
    X, Y = Placed(x, offset=n % 3), Placed(shape=(n,), offset=1)
    check(dropout(X, p, seed, offset, Y))
    assert_bitwise_equal(Y.numpy(), dropout_reference(x, p, seed, offset % 2**64))
    assert Y.untouched()


@pytest.mark.parametrize("shape,order,place", [
    ((6, 7, 8), (1, 0, 2), {}),           # rows of whole groups
    ((6, 7, 8), (1, 0, 2), {"pad": 3}),
    ((6, 7, 9), (1, 0, 2), {}),           # rows that groups straddle
    ((33, 65), (1, 0), {}),               # transposed
    ((5, 6, 7), (2, 0, 1), {"step": 2}),
    ((2, 1, 3, 1, 4), (4, 2, 0, 1, 3), {"offset": 5}),
])
@pytest.mark.parametrize("same", [True, False])
def test_strides_and_orders_keep_the_mask(shape, order, place, same):
    x = np.random.default_rng(1).standard_normal(shape).astype(np.float32)
    X = Placed(x, order=order, **place)
    Y = Placed(shape=shape, order=order if same else None, pad=0 if same else 1)
    check(dropout(X, 0.3, 99, 5, Y))
    assert_bitwise_equal(Y.numpy(), dropout_reference(x, 0.3, 99, 5))
    assert Y.untouched()


def test_a_broadcast_input():
    X = Placed(np.arange(1, 9, dtype=np.float32))
    X.layout = abi.layout_of((6, 8), (0, 1))
    Y = Placed(shape=(6, 8))
    check(dropout(X, 0.5, 3, 0, Y))
    assert_bitwise_equal(Y.numpy(), dropout_reference(np.tile(np.arange(1, 9, dtype=np.float32), (6, 1)), 0.5, 3, 0))


def test_probabilities_of_none_and_all_and_values_that_are_not_finite():
    x = np.array([1.0, -0.0, np.nan, np.inf, -np.inf, 3e38, 1e-45, 0.0] * 5, np.float32)
    for p in (0.0, 1.0, 1 - 2.0**-40, 0.5):
        X, Y = Placed(x), Placed(shape=x.shape)
        check(dropout(X, p, 11, 0, Y))
        assert_bitwise_equal(Y.numpy(), dropout_reference(x, p, 11, 0))


def test_in_place_and_a_second_call_continues_the_counters():
    x = np.random.default_rng(5).standard_normal(4000).astype(np.float32)
    X = Placed(x)
    check(dropout(X, 0.2, 1, 100, X))
    whole = dropout_reference(x, 0.2, 1, 100)
    assert_bitwise_equal(X.numpy(), whole)
    H, Y = Placed(x[2000:]), Placed(shape=(2000,))
    check(dropout(H, 0.2, 1, 100 + 500, Y))
    assert_bitwise_equal(Y.numpy(), whole[2000:])


def test_the_share_that_is_kept():
    """1e6 words: the share is within 5 standard deviations (0.0023) of 1 - p."""
    Y = Placed(shape=(1_000_000,))
    check(dropout(Placed(np.ones(1_000_000, np.float32)), 0.3, 42, 0, Y))
    assert abs((Y.numpy() != 0).mean() - 0.7) < 5 * np.sqrt(0.21 / 1e6)


def test_empty_and_refusals():
    X, Y = Placed(np.zeros((0, 4), np.float32)), Placed(shape=(0, 4))
    check(dropout(X, 0.5, 0, 0, Y))
    X, Y = Placed(np.ones((3, 4), np.float32)), Placed(shape=(3, 4))
    for p in (-0.1, 1.1, float("nan")):
        assert dropout(X, p, 0, 0, Y) == abi.TRS_E_INVALID_ARGUMENT
    assert dropout(X, 0.5, 0, 0, Placed(shape=(4, 3))) == abi.TRS_E_SHAPE_MISMATCH
    assert dropout(X, 0.5, 0, 0, Placed(shape=(12,))) == abi.TRS_E_SHAPE_MISMATCH
    Y.layout.stride[0] = 0
    assert dropout(X, 0.5, 0, 0, Y) == abi.TRS_E_INVALID_ARGUMENT
    T = Placed(shape=(3, 4))
    T.dev = X.dev
    T.layout.stride[0], T.layout.stride[1] = 1, 3
    assert dropout(X, 0.5, 0, 0, T) == abi.TRS_E_INVALID_ARGUMENT
    Y = Placed(shape=(3, 4))
    Y.dev = type("Null", (), {"ptr": None})()
    assert dropout(X, 0.5, 0, 0, Y) == abi.TRS_E_INVALID_ARGUMENT

"""Attention whose scores are large: sums beyond the range of the bf16 pieces, which hold
a score up to 2^47, against 64 bits.  The scale of most tests is ln 2, whose product
with log2(e) is 1 in fp32: scores of whole numbers are exact there, and so is what is
compared, but for the weights' and the sums' own rounding."""
import numpy as np
import pytest

from attention_util import EVERY, LEAST, U, Placed, assert_within, attention, attention_grad, ints, seen
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu
LN2 = np.float32(np.log(2))


def exact(q, k, v, window, sinks, scale, lengths=None):
    """{name: (value, bound)} of out and lse in 64 bits, for scores that fp32 holds exactly
    or all off alike: weights are off by the exponential and the sums, (n + 16) u."""
    B, H, sq, _ = q.shape
    G, sk = H // k.shape[1], k.shape[2]
    res = {"out": (np.zeros(q.shape), np.zeros(q.shape)), "lse": (np.full(q.shape[:3], -np.inf), np.zeros(q.shape[:3]))}
    for b in range(B):
        n = sk if lengths is None else lengths[b]
        mask = seen(sq, n, window, sinks)
        live = mask.any(1)
        for h in range(H):
            Q, K, V = (t.astype(np.float64) for t in (q[b, h][live], k[b, h // G, :n], v[b, h // G, :n]))
            s = np.where(mask[live], Q @ K.T * float(scale), -np.inf)
            top = s.max(1, keepdims=True)
            e = np.exp(s - top)
            P = e / e.sum(1, keepdims=True)
            lse = (top + np.log(e.sum(1, keepdims=True)))[:, 0]
            for name, value, bound in (("out", P @ V, 2 * (n + 16) * U * (P @ abs(V)) + n * LEAST),
                                       ("lse", lse, (n + 16) * U + 16 * U * abs(lse))):
                res[name][0][b, h, live], res[name][1][b, h, live] = value, bound
    return res


def exact_gradients(q, k, v, window, sinks, scale, up, lengths=None):
    """{name: (value, bound)} of dq, dk and dv for such scores.  A weight is read back from the
    row's logarithm, which is off by up to 2^-15 of itself however large it is; the rest are
    sums of magnitudes."""
    B, H, sq, D = q.shape
    G, sk = H // k.shape[1], k.shape[2]
    R = sq * G
    res = {n: (np.zeros(t.shape), np.zeros(t.shape)) for n, t in (("dq", q), ("dk", k), ("dv", v))}
    for b in range(B):
        n = sk if lengths is None else lengths[b]
        mask = seen(sq, n, window, sinks)
        live = mask.any(1)
        for h in range(H):
            kv = h // G
            Q, K, V, W = (t.astype(np.float64) for t in (q[b, h][live], k[b, kv, :n], v[b, kv, :n], up[b, h][live]))
            s = np.where(mask[live], Q @ K.T * float(scale), -np.inf)
            P = np.exp(s - s.max(1, keepdims=True))
            P /= P.sum(1, keepdims=True)
            o = P @ V
            dS = P * (W @ V.T - (W * o).sum(1, keepdims=True)) * float(scale)
            A = P * (abs(W) @ abs(V).T + (abs(W) * (P @ abs(V))).sum(1, keepdims=True)) * abs(float(scale))
            rel = (2 * n + 32) * U + 2.0 ** -15
            eS = A * (2 * rel + (2 * D + 32) * U) + LEAST * (1 + A / np.where(P > 0, P, 1))
            res["dq"][0][b, h, live] = dS @ K
            res["dq"][1][b, h, live] = eS @ abs(K) + (n + 16) * U * (A @ abs(K))
            res["dk"][0][b, kv, :n] += dS.T @ Q
            res["dk"][1][b, kv, :n] += eS.T @ abs(Q) + (R + 64) * U * (A.T @ abs(Q)) + R * LEAST
            res["dv"][0][b, kv, :n] += P.T @ W
            res["dv"][1][b, kv, :n] += rel * (P.T @ abs(W)) + (R + 64) * U * (P.T @ abs(W)) + LEAST * (R + abs(W).sum(0))
    return res


def values(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def forward(q, k, v, window, sinks, scale, lengths=None):
    out, rows = Placed(shape=q.shape), int(np.prod(q.shape[:3]))
    lse = DeviceArray(4 * rows)
    check(attention(*(Placed(t) for t in (q, k, v)), window, sinks, scale, out, lse, None if lengths is None else ints(lengths)))
    got = {"out": out.numpy(), "lse": lse.to_numpy(count=rows).reshape(q.shape[:3])}
    assert out.untouched()
    return got


def gradients(q, k, v, window, sinks, scale, up, lengths=None):
    P, out, lse = [Placed(t) for t in (q, k, v)], Placed(shape=q.shape), DeviceArray(4 * int(np.prod(q.shape[:3])))
    lens = None if lengths is None else ints(lengths)
    check(attention(*P, window, sinks, scale, out, lse, lens))
    grads = [Placed(shape=t.shape) for t in (q, k, v)]
    check(attention_grad(*P, window, sinks, scale, out, lse, Placed(up), *grads, lens))
    got = dict(zip(("dq", "dk", "dv"), (g.numpy() for g in grads)))
    assert all(g.untouched() for g in grads)
    return got


def compare(got, want):
    for name, value in got.items():
        assert_within(value, *want[name], what=name)


#        B  H hk  sq   sk  window sinks lengths
SHAPES = [
    (1, 2, 1, 100, 100, EVERY, 0, None),
    (1, 1, 1, 300, 300, 40, 3, None),
    (1, 1, 1, 1200, 1200, EVERY, 0, None),     # keys in parts
    (2, 4, 2, 90, 400, 200, 5, [400, 61]),     # the first queries of the second sequence see nothing
    (1, 2, 1, 3, 200, EVERY, 0, None),         # few rows
]
DIMS = (8, 32, 48, 64, 96, 128, 200)


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_finite_scores_far_below_zero(shape, D):
    """Every score of -2^50 (they weigh alike), and scores of which the largest, far below
    the others, weighs all."""
    B, H, hk, sq, sk, *mask = shape
    q, v = np.full((B, H, sq, D), 2.0 ** 24, np.float32), values(D, B, hk, sk, D)
    k = np.zeros((B, hk, sk, D), np.float32)
    k[..., 0] = -2.0 ** 26
    compare(forward(q, k, v, *mask[:2], LN2, mask[2]), exact(q, k, v, *mask[:2], LN2, mask[2]))
    k[..., 0] -= 2.0 ** 10 * np.arange(sk)
    compare(forward(q, k, v, *mask[:2], LN2, mask[2]), exact(q, k, v, *mask[:2], LN2, mask[2]))


def test_one_key_whatever_its_score():
    """A first query sees itself alone: its output is its value's, 64 products of -1e14 each."""
    q, k, v = np.full((1, 1, 70, 64), 1e7, np.float32), np.full((1, 1, 70, 64), -1e7, np.float32), values(0, 1, 1, 70, 64)
    got = forward(q, k, v, EVERY, 0, 0.125)
    assert np.array_equal(got["out"][0, 0, 0], v[0, 0, 0])
    want = exact(q, k, v, EVERY, 0, 0.125)  # all scores are the same sum
    compare({"out": got["out"]}, want)


@pytest.mark.parametrize("D", [32, 64, 96, 128])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_sums_that_leave_the_range_on_their_way(shape, D):
    """Half of a score's products are -2^45, the others 2^45: it is what is left, a small
    whole number, though the first half's sum is beyond the pieces' range."""
    B, H, hk, sq, sk, *mask = shape
    q, k, v = np.full((B, H, sq, D), 2.0 ** 22, np.float32), np.zeros((B, hk, sk, D), np.float32), values(D, B, hk, sk, D)
    k[:, :, ::2, : D // 2], k[:, :, ::2, D // 2:] = -2.0 ** 23, 2.0 ** 23
    # Both halves' sums are multiples of 2^45, so nothing is rounded.
    compare(forward(q, k, v, *mask[:2], LN2, mask[2]), exact(q, k, v, *mask[:2], LN2, mask[2]))
    up = values(D + 1, *q.shape)
    compare(gradients(q, k, v, *mask[:2], LN2, up, mask[2]), exact_gradients(q, k, v, *mask[:2], LN2, up, mask[2]))


@pytest.mark.parametrize("D", DIMS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_of_scores_far_below_zero(shape, D):
    """Scores of -2^50 that weigh alike, and ones of which the largest weighs all: a row's
    logarithm is no more exact than 2^27 there."""
    B, H, hk, sq, sk, *mask = shape
    q, v, up = np.full((B, H, sq, D), 2.0 ** 24, np.float32), values(D, B, hk, sk, D), values(D + 1, B, H, sq, D)
    k = np.zeros((B, hk, sk, D), np.float32)
    k[..., 0] = -2.0 ** 26
    compare(gradients(q, k, v, *mask[:2], LN2, up, mask[2]), exact_gradients(q, k, v, *mask[:2], LN2, up, mask[2]))
    k[..., 0] -= 2.0 ** 10 * np.arange(sk)
    compare(gradients(q, k, v, *mask[:2], LN2, up, mask[2]), exact_gradients(q, k, v, *mask[:2], LN2, up, mask[2]))


#          B  H hk  sq   sk   window sinks lengths
OFFSETS = [
    (1, 2, 1, 100, 100, EVERY, 0, None),
    (2, 4, 2, 90, 200, 60, 5, [200, 61]),
    (1, 1, 1, 420, 420, 50, 40, None),      # sinks' rows far past them
    (1, 3, 1, 5, 130, EVERY, 0, None),
]


@pytest.mark.parametrize("offset", [0, 300, 1e5, -1e5, 2.0 ** 20, 2.0 ** 25, -2.0 ** 30, 2.0 ** 40], ids=str)
@pytest.mark.parametrize("D", [32, 64, 128, 160, 256])
@pytest.mark.parametrize("shape", OFFSETS, ids=str)
def test_gradients_under_a_common_offset(shape, D, offset):
    """Scores of whole numbers with an offset that all of a row share, in two rows of three: it
    changes no weight.  Every score and sum is exact; differences are of at least a unit in
    the last place of the offset."""
    B, H, hk, sq, sk, *mask = shape
    step = max(1.0, abs(offset) * 2.0 ** -23)
    q, k = np.zeros((B, H, sq, D), np.float32), values(1, B, hk, sk, D)
    q[..., 0] = np.where(np.arange(sq) % 3, 2.0 ** 5, 0)
    q[..., 1] = np.exp2(np.floor(np.log2(step))) * (1 + np.arange(sq) % 2)
    k[..., 0], k[..., 1] = offset / 2.0 ** 5, -(np.arange(sk) * 7 % 4)
    v, up = values(2, *k.shape), values(3, *q.shape)
    compare(gradients(q, k, v, *mask[:2], LN2, up, mask[2]), exact_gradients(q, k, v, *mask[:2], LN2, up, mask[2]))


@pytest.mark.parametrize("D", [32, 64, 128, 200])
@pytest.mark.parametrize("std", [20.0, 200.0, 1e6])
def test_the_weights_of_a_row_sum_to_one_in_the_gradients(D, std):
    """Scores of any size, rounded as they may be: the gradients of the values add up to the
    upstream rows, here those whose logarithm is large."""
    q, k = (np.float32(std) * values(s, 1, 4, 150, D) for s in (5, 6))
    k, v, up = k[:, :2], values(7, 1, 2, 150, D), values(8, *q.shape)
    up[abs(forward(q, k, v, 70, 3, 0.2)["lse"]) <= 256] = 0
    assert up.any()
    dv = gradients(q, k, v, 70, 3, 0.2, up)["dv"].astype(np.float64)
    rows = up.reshape(1, 2, 300, D).astype(np.float64)
    # Weights of 150 keys and their sum, and sums over 300 rows.
    assert_within(dv.sum(2), rows.sum(2), (2 * 150 + 300 + 64) * U * abs(rows).sum(2), "dv")


@pytest.mark.parametrize("D", [64, 80, 128])
def test_a_sum_that_leaves_the_range_counts_in_every_block_of_keys(D):
    """Scores of 2^12 whose sums, of some keys of the first block alone, pass -2^49 on their way:
    these keys weigh as much as the others, whose gradients other blocks work out."""
    n = 300
    q, k = np.full((1, 2, n, D), 2.0 ** 22, np.float32), np.zeros((1, 1, n, D), np.float32)
    q[..., 32:] = 0
    q[..., 40], k[..., 40] = 2.0 ** 5, 2.0 ** 7
    k[:, :, :40:2, :16], k[:, :, :40:2, 16:32] = -2.0 ** 23, 2.0 ** 23
    v, up = values(D, *k.shape), values(D + 1, *q.shape)
    for sinks, window in ((0, EVERY), (30, 64)):
        compare(forward(q, k, v, window, sinks, LN2), exact(q, k, v, window, sinks, LN2))
        compare(gradients(q, k, v, window, sinks, LN2, up), exact_gradients(q, k, v, window, sinks, LN2, up))


@pytest.mark.parametrize("D", [16, 64, 128, 160])
def test_gradients_just_within_the_range(D):
    """dS K and dS^T Q that would leave fp32's range unscaled: by a scale of 2^-10 the gradients do not."""
    scale = np.float32(2.0 ** -10)
    q, k, v, up = (values(s, 1, 2, 80, D) for s in range(4))
    k, v = k[:, :1], np.float32(1e16) * v[:, :1]
    for side in (0, 1):
        big = [np.float32(1e12 if side == 0 else 1e-12) * k, np.float32(1e-12 if side == 0 else 1e12) * q]
        want = exact_gradients(big[1], big[0], v, 40, 2, scale, up)
        name = ("dq", "dk")[side]
        f = np.float32(2.0 ** 124 / abs(want[name][0]).max())  # sums of magnitudes stay within the range
        want = exact_gradients(big[1], big[0], v, 40, 2, scale, f * up)
        assert abs(want[name][0] / scale).max() > 3.5e38
        got = gradients(big[1], big[0], v, 40, 2, scale, f * up)
        # Scores are within 1/100 of 0; their rounding is far below the bound's weights'.
        assert_within(got[name], *want[name], what=name)


@pytest.mark.parametrize("D", [8, 32, 64, 80, 128, 200])
def test_weights_of_scores_beyond_the_range_sum_to_one_in_the_gradients(D):
    """The same of scores of about 1e17 either way, some rows' small: blocks on the fp32 instruction."""
    q, k = (np.float32(1e9) * values(s, 1, 4, 150, D) for s in (5, 6))
    q[:, :, ::7] *= np.float32(1e-19)
    k, v, up = k[:, :2], values(7, 1, 2, 150, D), values(8, *q.shape)
    dv = gradients(q, k, v, 70, 3, 0.2, up)["dv"].astype(np.float64)
    rows = up.reshape(1, 2, 300, D).astype(np.float64)
    assert_within(dv.sum(2), rows.sum(2), (2 * 150 + 300 + 64) * U * abs(rows).sum(2), "dv")

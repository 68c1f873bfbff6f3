"""Shared keys worked on for the whole batch at once where they, or queries, are not finite, and where the pool has not
all of their pages; tables wider than any sequence."""
import numpy as np
import pytest

from attention_util import EVERY, U, Placed, assert_within, attention_reference, ints, seen
from paged_util import BF16, F32, Cache, held, paged_attention
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])


def inputs(seed, B, H, HK, sq, n, D, kind, shared):
    rng = np.random.default_rng(seed)
    q = rng.standard_normal((B, H, sq, D)).astype(np.float32)
    k, v = (held(rng.standard_normal((B, HK, n, D)).astype(np.float32), kind) for _ in range(2))
    for x in (k, v):
        x[:, :, :shared] = x[:1, :, :shared]
    return q, k, v


def formula(q, k, v, window, sinks, scale, lengths):
    """(out, bound) in 64 bits of keys and values that need not be finite: what a query sees enters with IEEE's rules, what it
    does not see enters nowhere.  The bound is attention_reference's, of what is finite."""
    B, H, sq, D = q.shape
    G = H // k.shape[1]
    out, bound = np.zeros(q.shape), np.zeros(q.shape)
    for b, n in enumerate(lengths):
        m = seen(sq, n, window, sinks)
        live = m.any(1)
        m = m[live]
        if not live.any():
            continue
        for h in range(H):
            Q, K, V = (x.astype(np.float64) for x in (q[b, h][live], k[b, h // G, :n], v[b, h // G, :n]))
            K0, V0 = (np.where(np.isfinite(x), x, 0) for x in (K, V))
            s = Q @ K0.T * scale
            for j in np.flatnonzero(~np.isfinite(K).all(1)):
                s[:, j] = (Q * K[j]).sum(1) * scale
            s = np.where(m, s, -np.inf)
            with np.errstate(invalid="ignore"):
                e = np.exp(s - s.max(1, keepdims=True))
                P = e / e.sum(1, keepdims=True)
                o = P @ V0
                for j in np.flatnonzero(~np.isfinite(V).all(1)):
                    odd = ~np.isfinite(V[j])
                    o[np.ix_(m[:, j], odd)] += P[m[:, j], j][:, None] * V[j, odd]
            d = (D + 8) * U * np.where(m, abs(Q) @ abs(K0).T * abs(scale), 0).max(1, keepdims=True)
            out[b, h, live], bound[b, h, live] = o, (2 * d + (n + 16) * U) * (P @ abs(V0))
    return out, bound


def call(q, cache, shared, window, sinks, scale):
    out = Placed(shape=q.shape)
    check(paged_attention(Placed(q), cache, shared, window, sinks, scale, out))
    got = out.numpy()
    assert out.untouched()
    return got


# (batch - 1) * shared * key heads * dim * 4 (bfloat16) or 8 bytes are above 16 MiB in each: shared keys are a stage of their own.
#    B  H HK  sq  D page shared window sinks      (a stage's kernel goes by its rows and pairs)
SIZES = [
    (9, 8, 2, 1, 64, 16, 4100, EVERY, 0),        # few rows in both stages
    (9, 8, 2, 2, 64, 10, 4100, 1500, 7),         # pages that end inside a tile
    (9, 4, 2, 2, 200, 16, 1400, EVERY, 0),
    (17, 8, 2, 16, 64, 16, 4100, EVERY, 0),      # many rows of the shared keys
    (17, 8, 2, 16, 80, 16, 4100, 4000, 7),
    (17, 8, 2, 16, 33, 10, 4100, EVERY, 0),
    (20, 8, 4, 100, 32, 16, 1740, EVERY, 0),     # and of each sequence's own
    (20, 8, 4, 100, 32, 16, 1740, 900, 40),
]
BATCHES = pytest.mark.parametrize("size", SIZES, ids=str)


def lengths_of(B, sq, shared):
    """Sequences that end behind the shared keys, among them, ahead of them, and one without tokens."""
    ends = [shared + 560, shared - shared // 3 + 30, sq + 5, 0, shared + 1, shared // 3 + 2, max(sq // 2, 1), shared + 17, shared // 2]
    return [ends[i % 9] + (i // 9) % 3 * (ends[i % 9] > sq) for i in range(B)]


@KINDS
@BATCHES
@pytest.mark.parametrize("where", ["keys", "values"])
def test_shared_keys_and_values_that_are_not_finite(kind, size, where):
    """Seen by some sequences and hidden from others; padded queries hold NaN."""
    B, H, HK, sq, D, page, shared, window, sinks = size
    lengths = lengths_of(B, sq, shared)
    q, k, v = inputs(B + D, B, H, HK, sq, max(lengths), D, kind, shared)
    q = abs(q)
    third, last = shared // 3, HK - 1
    if where == "keys":
        k[:, 0, third, 3], k[:, last, 2 * third, 0] = np.nan, -np.inf  # a score of -inf has no weight
    else:
        v[:, 0, third, 3], v[:, last, 2 * third, D - 1], v[:, last, third + 1, 1] = np.nan, np.inf, -np.inf
    want = formula(q, k, v, window, sinks, D ** -0.5, lengths)
    odd = np.isnan(want[0]) | np.isinf(want[0])
    assert odd.any() and not odd.all()
    for b, n in enumerate(lengths):
        q[b, :, :max(sq - n, 0)] = np.nan
    cache = Cache(B, HK, page, D, lengths, kind, "heads", k, v, shared=shared)
    assert_within(call(q, cache, shared, window, sinks, D ** -0.5), *want)


@KINDS
@BATCHES
def test_shared_keys_that_nobody_sees_may_hold_anything(kind, size):
    """A window that begins behind them for every sequence, or ends ahead of them."""
    B, H, HK, sq, D, page, shared, window, sinks = size
    window, sinks = shared // 8, 3
    lengths = [shared - shared // 8 + 3 * i if i % 2 else sq + shared // 9 + i for i in range(B)]
    q, k, v = inputs(B + D + 1, B, H, HK, sq, max(max(lengths), shared), D, kind, shared)
    want = formula(q, k, v, window, sinks, D ** -0.5, lengths)
    lo = max(n for i, n in enumerate(lengths) if i % 2 == 0)
    hi = min(n - sq - window + 1 for i, n in enumerate(lengths) if i % 2)
    assert lo + 40 < hi
    for x, bad in ((k, np.nan), (v, np.inf)):
        x[:, :, lo:hi] = bad
        x[:, :, lo:hi:3] = -np.inf
    cache = Cache(B, HK, page, D, lengths, kind, "heads", k, v, shared=shared, width=-(-shared // page) + 1)
    assert_within(call(q, cache, shared, window, sinks, D ** -0.5), *want)


@KINDS
@pytest.mark.parametrize("size", SIZES + [(3, 4, 2, 1, 64, 16, 100, EVERY, 0), (3, 4, 2, 130, 64, 16, 100, 60, 0), (3, 4, 2, 2, 64, 10, 100, 60, 0)], ids=str)
def test_a_page_of_the_shared_keys_that_the_pool_does_not_have(kind, size):
    """Exactly the queries that see one of its keys are NaN."""
    B, H, HK, sq, D, page, shared, window, sinks = size
    lengths = lengths_of(B, sq, shared)
    q, k, v = inputs(B + D + 2, B, H, HK, sq, max(lengths), D, kind, shared)
    cache = Cache(B, HK, page, D, lengths, kind, "heads", k, v, shared=shared)
    gone = shared // 3 // page
    cache.table[0, gone] = cache.shape[0] if B % 2 else -7
    cache.table_dev = ints(cache.table)
    cache.struct.table = cache.table_dev.addr
    k[:, :, gone * page:(gone + 1) * page] = np.nan
    want = formula(q, k, v, window, sinks, D ** -0.5, lengths)
    odd = np.isnan(want[0])
    assert odd.any() and not odd.all()
    assert_within(call(q, cache, shared, window, sinks, D ** -0.5), *want)


#        B  H HK sq   D  page lengths               shared window sinks
WIDE = [
    (1, 8, 8, 1, 64, 16, [1000], 0, EVERY, 0),
    (8, 8, 2, 1, 128, 16, [2000 - 200 * i for i in range(8)], 0, 1024, 4),
    (1, 32, 8, 32, 64, 16, [500], 0, EVERY, 0),
    (2, 16, 4, 300, 80, 16, [900, 333], 0, 400, 3),
    (9, 8, 2, 1, 64, 16, [4300, 4200, 4150, 3000, 1500, 700, 20, 0, 4110], 4100, EVERY, 0),
]


@KINDS
@pytest.mark.parametrize("times", [8, 64])
@pytest.mark.parametrize("shape", WIDE, ids=str)
def test_tables_wider_than_any_sequence(kind, times, shape):
    """A server's table has room for its longest context, and nothing behind a sequence's last page."""
    B, H, HK, sq, D, page, lengths, shared, window, sinks = shape
    q, k, v = inputs(sq + D, B, H, HK, sq, max(lengths), D, kind, shared)
    cache = Cache(B, HK, page, D, lengths, kind, "heads", k, v, shared=shared, width=times * -(-max(lengths) // page))
    L = DeviceArray(4 * B * H * sq)
    out = Placed(shape=q.shape)
    check(paged_attention(Placed(q), cache, shared, window, sinks, D ** -0.5, out, L))
    want = attention_reference(q, k, v, window, sinks, D ** -0.5, lengths)
    assert_within(out.numpy(), *want["out"])
    assert_within(L.to_numpy(count=B * H * sq).reshape(B, H, sq), *want["lse"])

"""Attention over a paged cache, against 64 bits: pages that end inside a tile, ragged
lengths, windows, first tokens, prefixes that a batch shares, tokens and prompts."""
import numpy as np
import pytest

from attention_util import EVERY, Placed, assert_within, attention_reference, ints
from paged_util import BF16, F32, Cache, held, paged_attention
from trs_backend import abi
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu
TOKENS = (0, 2, 1, 3)
KINDS = pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])


def inputs(seed, B, H, HK, sq, most, D, kind, std=1.0):
    rng = np.random.default_rng(seed)
    q = (std * rng.standard_normal((B, H, sq, D))).astype(np.float32)
    k, v = (held(rng.standard_normal((B, HK, max(most, 1), D)).astype(np.float32), kind) for _ in range(2))
    return q, k, v


def share(k, v, shared):
    """Every sequence's first keys and values are the first one's."""
    for x in (k, v):
        x[:, :, :shared] = x[:1, :, :shared]


def run(q, k, v, lengths, page, kind, window=EVERY, sinks=0, shared=0, scale=None, form="heads", order=TOKENS, lse=True, damage=None, want=None, **kw):
    B, H, sq, D = q.shape
    cache = Cache(B, k.shape[1], page, D, lengths, kind, form, k, v, shared=shared, **kw)
    if damage is not None:
        damage(cache)
    scale = D ** -0.5 if scale is None else scale
    out = Placed(shape=q.shape, order=order)
    L = DeviceArray(max(4, 4 * B * H * sq)) if lse else None
    check(paged_attention(Placed(q, order=order), cache, shared, window, sinks, scale, out, L))
    got = {"out": out.numpy()}
    assert out.untouched()
    if lse:
        got["lse"] = L.to_numpy(count=B * H * sq).reshape(B, H, sq)
    n = [min(max(x, 0), cache.table.shape[1] * page) for x in lengths]
    if want is None:
        want = attention_reference(q, k, v, window, sinks, scale, n)
    for name, value in got.items():
        assert_within(value, *want[name], what=name)
    return got, want


#        B  H HK sq   D  page lengths            window sinks
SHAPES = [
    (1, 1, 1, 1, 1, 1, [1], EVERY, 0),
    (1, 1, 1, 1, 32, 16, [1], 1, 1),
    (1, 2, 1, 1, 64, 16, [33], 8, 2),
    (2, 4, 2, 1, 128, 16, [300, 17], EVERY, 0),
    (3, 8, 1, 2, 80, 8, [129, 2, 64], EVERY, 0),
    (1, 1, 1, 5, 7, 3, [5], EVERY, 0),
    (2, 8, 8, 1, 64, 10, [1000, 700], 512, 4),       # pages that end inside a tile
    (2, 32, 8, 1, 128, 48, [515, 31], EVERY, 0),
    (4, 8, 2, 1, 128, 16, [2000, 1, 0, 900], 300, 5),  # a sequence without tokens
    (1, 16, 1, 1, 96, 64, [777], EVERY, 0),          # as many rows as a tile
    (1, 17, 1, 1, 64, 16, [300], EVERY, 0),          # and one more
    (2, 20, 4, 3, 48, 16, [333, 100], 64, 70),
    (1, 4, 2, 33, 200, 16, [150], EVERY, 0),
    (1, 2, 1, 100, 256, 32, [130], 40, 6),
    (2, 2, 1, 40, 48, 16, [25, 40], 9, 2),           # more queries than keys: the first see nothing
    (1, 2, 2, 300, 64, 16, [300], EVERY, 0),         # a prompt
    (2, 4, 2, 200, 128, 16, [520, 333], EVERY, 0),   # a part of one over what the cache holds
    (1, 6, 2, 257, 128, 64, [600], 50, 3),
    (3, 6, 6, 130, 80, 16, [400, 130, 90], 64, 3),
    (1, 1, 1, 700, 32, 16, [700], 8, 1),
    (1, 4, 1, 500, 24, 24, [1000], 30, 70),
    (1, 5, 1, 140, 33, 16, [140], EVERY, 0),
    (2, 8, 2, 100, 96, 12, [100, 260], 128, 0),
    (1, 1, 1, 70, 129, 16, [170], 40, 6),
    (1, 3, 3, 90, 10, 100, [250], EVERY, 2),
    (40, 2, 1, 1, 64, 16, [7 * i % 300 for i in range(40)], EVERY, 0),
    (70, 4, 2, 1, 32, 16, [5 + i for i in range(70)], 20, 2),
]

# Pairs of a row and a key enough for tiles of 128 and 256 rows.
MANY = [
    (1, 64, 16, 1024, 16, 16, [1024], EVERY, 0),     # tiles of rows for every CU
    (2, 64, 8, 1000, 24, 32, [700, 1100], 600, 3),
    (1, 16, 4, 700, 64, 16, [1000], EVERY, 0),
    (2, 8, 2, 600, 128, 64, [1500, 900], EVERY, 0),
    (1, 8, 2, 1000, 33, 16, [1200], EVERY, 0),       # a dim that no vector divides
    (3, 6, 6, 700, 80, 16, [900, 700, 750], EVERY, 0),
    (1, 16, 4, 900, 96, 48, [1500], 600, 40),
    (1, 12, 4, 1000, 16, 10, [1000], EVERY, 2),      # pages that end inside a tile
    (1, 8, 2, 1300, 24, 12, [2000], 300, 70),
    (40, 8, 2, 30, 128, 16, [1000 - 20 * i for i in range(40)], EVERY, 0),  # 120 rows a sequence
    (4, 16, 2, 300, 64, 16, [0, 1000, 299, 5], EVERY, 0),
    (1, 5, 1, 1200, 128, 16, [1500], 1, 0),          # each query sees itself alone
    (2, 8, 2, 700, 256, 16, [1000, 1600], EVERY, 0),
    (1, 8, 2, 1000, 200, 16, [1300], 400, 3),
    (1, 16, 4, 800, 150, 24, [900], EVERY, 0),
    (1, 8, 2, 1100, 137, 10, [1200], 500, 0),
]

# Few rows over so many keys that a row has tens or hundreds of parts.
LONG = [
    (1, 1, 1, 1, 256, 8, [7000], EVERY, 0),
    (1, 8, 2, 2, 200, 128, [9001], EVERY, 0),
    (2, 4, 2, 1, 128, 16, [5000, 3], EVERY, 0),
    (3, 2, 1, 1, 64, 16, [8200, 0, 4100], 3000, 5),
    (1, 1, 1, 1, 8, 16, [9000], EVERY, 0),
    (1, 3, 1, 3, 33, 10, [6001], EVERY, 0),
    (8, 8, 8, 8, 100, 16, [2600 - 300 * i for i in range(8)], EVERY, 0),  # 512 rows
    (8, 8, 8, 9, 100, 16, [2600 - 300 * i for i in range(8)], EVERY, 0),  # and more
]


@KINDS
@pytest.mark.parametrize("shape", SHAPES + MANY + LONG, ids=str)
def test_attention_matches_64_bits(shape, kind):
    B, H, HK, sq, D, page, lengths, window, sinks = shape
    q, k, v = inputs(sq * 7 + D, B, H, HK, sq, max(lengths), D, kind)
    run(q, k, v, lengths, page, kind, window, sinks)


#        B  H HK sq   D  page lengths  shared window sinks
SHARED = [
    (2, 2, 1, 1, 64, 16, [40, 33], 32, EVERY, 0),
    (3, 4, 2, 1, 128, 16, [300, 281, 260], 256, EVERY, 0),
    (5, 8, 2, 1, 64, 16, [1100, 1050, 1001, 1010, 1090], 1000, EVERY, 0),   # the shared keys end inside a page
    (4, 4, 4, 1, 80, 8, [130, 100, 64, 20], 100, EVERY, 0),                 # sequences that end among the shared keys
    (3, 2, 1, 2, 32, 16, [50, 0, 17], 16, EVERY, 0),                        # and one without tokens
    (33, 8, 2, 1, 128, 16, [600 + i for i in range(33)], 576, EVERY, 0),    # many rows
    (20, 8, 1, 2, 64, 16, [700 + 3 * i for i in range(20)], 640, 500, 4),
    (64, 8, 2, 1, 128, 16, [300 + i for i in range(64)], 256, EVERY, 0),
    (6, 6, 2, 40, 48, 16, [300, 290, 280, 270, 260, 250], 200, EVERY, 0),   # prompts behind a shared one
    (40, 4, 1, 3, 96, 10, [200 + 7 * i for i in range(40)], 150, 64, 30),
    (70, 2, 1, 2, 256, 16, [100 + i for i in range(70)], 96, EVERY, 0),
    (2, 2, 2, 3, 33, 16, [200, 180], 150, 20, 10),                          # a window behind the shared keys: of these, the first alone
    (3, 3, 1, 1, 20, 16, [64, 64, 64], 64, EVERY, 0),                       # nothing of their own
    (2, 2, 1, 1, 64, 16, [64, 60], 1000, EVERY, 0),                         # more shared keys than the table has
    (1, 4, 1, 1, 64, 16, [100], 80, EVERY, 0),                              # one sequence
    (80, 8, 2, 1, 64, 16, [40 + i % 9 for i in range(80)], 32, EVERY, 0),
]

# Shared keys enough to be worked on for the whole batch at once, by few rows or by many.
TOGETHER = [
    (33, 8, 2, 1, 64, 16, [1100 + i for i in range(33)], 1024, EVERY, 0),
    (33, 8, 2, 1, 64, 16, [(1100 + i) * (i % 5 > 0) for i in range(33)], 1030, EVERY, 0),  # in a page's middle; sequences without tokens
    (3, 16, 8, 2, 128, 16, [2300, 2100, 2049], 2048, 700, 9),
    (17, 4, 4, 1, 80, 8, [1600 - 90 * i for i in range(17)], 1500, EVERY, 0),              # ones that end among the shared keys
    (33, 4, 2, 1, 33, 10, [2000 + 5 * i for i in range(33)], 2000, EVERY, 0),
    (9, 2, 2, 1, 256, 16, [2200 + i for i in range(9)], 2176, 1000, 0),
    (33, 8, 2, 8, 64, 16, [4200 + 3 * i for i in range(33)], 4096, EVERY, 0),
    (33, 8, 2, 8, 128, 16, [4200 + 3 * i for i in range(33)], 4096, 3000, 5),
    (20, 8, 4, 40, 48, 16, [1600 - 20 * i for i in range(20)], 1330, EVERY, 0),
    (20, 8, 4, 100, 32, 16, [1900 + i for i in range(20)], 1330, EVERY, 0),                # many rows of both kinds
    (12, 16, 2, 24, 256, 16, [2000 - i for i in range(12)], 1900, EVERY, 0),
    (24, 16, 2, 12, 96, 24, [2100] * 24, 2100, EVERY, 0),                                  # nothing of their own
    (34, 8, 2, 8, 20, 16, [4300 - 100 * i for i in range(34)], 4100, 2000, 40),
    (7, 2, 1, 2, 128, 16, [4700 + 30 * i for i in range(7)], 4600, EVERY, 0),              # a row's parts of both kinds by the tens
    (3, 1, 1, 1, 256, 16, [9100, 9050, 9040], 9030, EVERY, 0),
]


@KINDS
@pytest.mark.parametrize("shape", SHARED + TOGETHER, ids=str)
def test_keys_that_a_batch_shares(shape, kind):
    B, H, HK, sq, D, page, lengths, shared, window, sinks = shape
    q, k, v = inputs(sq + D + shared, B, H, HK, sq, max(lengths), D, kind)
    share(k, v, min(shared, k.shape[2]))
    run(q, k, v, lengths, page, kind, window, sinks, shared)


@KINDS
@pytest.mark.parametrize("form", ["heads", "tokens", "both", "odd"])
@pytest.mark.parametrize("order", [TOKENS, (0, 1, 2, 3), (1, 0, 2, 3)], ids=str)
def test_pools_and_queries_of_any_order(form, kind, order):
    for sq, D, page in ((1, 64, 16), (2, 48, 10), (150, 64, 16), (100, 20, 12)):
        q, k, v = inputs(sq, 2, 4, 2, sq, 200, D, kind)
        run(q, k, v, [200, 151], page, kind, 90, 3, form=form, order=order)
    for D, page in ((64, 16), (20, 12)):  # many rows
        q, k, v = inputs(D, 2, 16, 2, 400, 700, D, kind)
        run(q, k, v, [700, 651], page, kind, 500, 3, form=form, order=order)


@pytest.mark.parametrize("sq", [1, 100])
def test_a_query_without_a_unit_stride(sq):
    q, k, v = inputs(4, 1, 2, 1, sq, 120, 32, F32)
    cache = Cache(1, 1, 16, 32, [120], F32, "heads", k, v)
    out = Placed(shape=q.shape)
    check(paged_attention(Placed(q, step=2), cache, 0, EVERY, 0, 0.2, out))
    assert_within(out.numpy(), *attention_reference(q, k, v, EVERY, 0, 0.2, [120])["out"])


# Heads, tokens and keys of few rows and of many.
SIZES = pytest.mark.parametrize("H,sq,most", [(4, 1, 290), (4, 3, 290), (4, 130, 290), (16, 520, 1100)])


@KINDS
@pytest.mark.parametrize("D", [64, 80, 20])
@SIZES
@pytest.mark.parametrize("shared", [0, 48])
def test_hidden_values_that_are_not_finite_do_not_reach_a_query(kind, D, H, sq, most, shared):
    """NaN and infinities before the window and behind a sequence; queries of padding hold NaN."""
    B, lengths, window, sinks = 2, [most, sq + 90], 60, 5
    if H > 4:
        window = 600
    q, k, v = inputs(8, B, H, 2, sq, most, D, kind)
    share(k, v, shared)
    want = attention_reference(q, k, v, window, sinks, D ** -0.5, lengths)
    for b, n in enumerate(lengths):
        low = n - sq - window + 1
        for x, bad in ((k, np.nan), (v, np.inf)):
            if low > max(sinks, shared):
                x[b, :, max(sinks, shared):low] = bad
                x[b, :, max(sinks, shared):low:2] = -np.inf if bad == np.inf else np.inf
            x[b, :, n:] = np.nan
    run(q, k, v, lengths, 16, kind, window, sinks, shared, want=want)


@KINDS
@SIZES
def test_padded_queries_that_hold_nan_give_zero(kind, H, sq, most):
    q, k, v = inputs(9, 3, H, 2, sq, most, 64, kind)
    lengths = [most, 0, max(sq // 2, 0)]
    for b, n in enumerate(lengths):
        q[b, :, :max(sq - n, 0)] = np.nan
    got, _ = run(q, k, v, lengths, 16, kind, want={"out": (np.where(np.isnan(q), 0, attention_reference(np.nan_to_num(q), k, v, EVERY, 0, 0.125, lengths)["out"][0]),
                                                          attention_reference(np.nan_to_num(q), k, v, EVERY, 0, 0.125, lengths)["out"][1])}, scale=0.125, lse=False)
    assert not np.isnan(got["out"]).any()


@KINDS
@pytest.mark.parametrize("H,sq,D,n,window", [(4, 1, 64, 200, 64), (4, 2, 20, 200, 64), (4, 130, 64, 200, 64), (4, 130, 200, 200, 64), (32, 400, 64, 700, 500),
                                             (32, 400, 20, 700, 500)])
@pytest.mark.parametrize("where", ["key", "value"])
def test_visible_values_that_are_not_finite_are_as_the_formula_has_them(kind, H, sq, D, n, window, where):
    """NaN where the formula gives it, the same infinities, and no other row touched."""
    q, k, v = inputs(10, 2, H, 2, sq, n, D, kind)
    q, G, lengths = abs(q), H // 2, [n, n - 20]
    want = attention_reference(q, k, v, window, 0, D ** -0.5, lengths)
    value, bound = (x.copy() for x in want["out"])
    x, bad = k if where == "key" else v, (n - 10, n - 30)
    x[0, 0, bad[0], 3], x[1, 1, bad[1], 3] = np.nan, (-np.inf if where == "key" else np.inf)
    place = [m - sq + np.arange(sq) for m in lengths]
    sees = [(place[b] >= j) & (place[b] - j < window) for b, j in enumerate(bad)]
    if where == "key":
        value[0, :G, sees[0]] = np.nan
        # A score of -inf has no weight: the same as without the key.
        rows = attention_without(q, k, v, 1, 1, bad[1], n - 20, D, window)
        value[1, G:, sees[1]], bound[1, G:, sees[1]] = rows[0][:, sees[1]].transpose(1, 0, 2), rows[1][:, sees[1]].transpose(1, 0, 2)
    else:
        value[0, :G, sees[0], 3] = np.nan
        value[1, G:, sees[1], 3] = np.inf
    run(q, k, v, lengths, 16, kind, window, 0, want={"out": (value, bound)}, lse=False)


def attention_without(q, k, v, b, head, key, n, D, window):
    """out and bound of one key head's rows with one key left out."""
    sq, G = q.shape[2], q.shape[1] // k.shape[1]
    rows = q[b, head * G:(head + 1) * G].astype(np.float64)
    K, V = (np.where(np.isfinite(x[b, head, :n]), x[b, head, :n], 0).astype(np.float64) for x in (k, v))
    s = rows @ K.T * D ** -0.5
    p = (n - sq + np.arange(sq))[:, None]
    j = np.arange(n)[None]
    s = np.where((j <= p) & (p - j < window) & (j != key), s, -np.inf)
    e = np.exp(s - s.max(-1, keepdims=True))
    P = e / e.sum(-1, keepdims=True)
    d = (D + 8) * 2.0 ** -24 * (abs(rows) @ abs(K).T * D ** -0.5).max(-1, keepdims=True)
    return P @ V, (2 * d + (n + 16) * 2.0 ** -24) * (P @ abs(V))


@KINDS
@pytest.mark.parametrize("H,sq,most,window", [(4, 1, 200, 60), (4, 130, 200, 60), (32, 400, 700, 300)])
@pytest.mark.parametrize("shared", [0, 32])
def test_a_page_that_the_pool_does_not_have_makes_those_that_see_it_nan(kind, H, sq, most, window, shared):
    B, lengths = 3, [most, most - 10, most - 15]
    q, k, v = inputs(11, B, H, 2, sq, most, 64, kind)
    share(k, v, shared)
    bad = {0: 10, 1: 3, 2: 11}  # page 3 of the second: before every window of one token, not of a prompt

    def damage(cache):
        for b, i in bad.items():
            cache.table[b, i] = (cache.shape[0], -5, 2 ** 31 - 1)[b]
        cache.table_dev = ints(cache.table)
        cache.struct.table = cache.table_dev.addr

    value, bound = attention_reference(q, k, v, window, 0, 0.125, lengths)["out"]
    for b, n in enumerate(lengths):
        p = n - sq + np.arange(sq)
        first, last = 16 * bad[b], 16 * bad[b] + 15
        value[b][:, (p >= first) & (p - window < last)] = np.nan
    run(q, k, v, lengths, 16, kind, window, 0, shared, scale=0.125, damage=damage, want={"out": (value, bound)}, lse=False)


@KINDS
@pytest.mark.parametrize("H,sq,D", [(4, 1, 64), (4, 3, 96), (4, 150, 64), (4, 150, 200), (64, 300, 64)])
@pytest.mark.parametrize("size", [1e-20, 30.0, 1e4])
def test_scores_of_any_size(kind, H, sq, D, size):
    q, k, v = inputs(12, 2, H, 2, sq, 360, D, kind, std=size)
    run(q, k, v, [360, 300], 16, kind, 128, 2)


@KINDS
@pytest.mark.parametrize("H,sq", [(4, 1), (4, 100), (64, 300)])
def test_values_of_any_size(kind, H, sq):
    """Keys beyond the products' pieces, and values near the least and the largest floats."""
    q, k, v = inputs(13, 1, H, 2, sq, 450, 64, kind)
    run(q * np.float32(1e-30), held(k * np.float32(1e30), kind), v, [450], 16, kind)
    run(q, k, held(v * np.float32(1e-36), kind), [450], 16, kind)
    run(q, k, held(v * np.float32(1e34), kind), [450], 16, kind)


@KINDS
def test_lengths_beyond_the_table_and_below_zero(kind):
    q, k, v = inputs(14, 3, 2, 1, 2, 64, 64, kind)
    run(q, k, v, [1000, -3, 5], 16, kind, width=4)


@KINDS
@pytest.mark.parametrize("H,sq", [(4, 1), (64, 900)])
def test_offsets_past_32_bits(kind, H, sq):
    """Pools that reach past 2^32 bytes and 2^31 entries, in one buffer that is mostly untouched."""
    D, page, HK = 64, 16, 2
    q, k, v = inputs(15, 1, H, HK, sq, 160, D, kind)
    size = 2 if kind == BF16 else 4
    cache = Cache(1, HK, page, D, [160], kind, "heads", k, v, extra=0)
    count, step = cache.shape[0], (1 << 32) // size // 4  # a GiB a page: offsets to 10 GiB
    step = step // (HK * page * D) * (HK * page * D)
    big = [DeviceArray(size * (step * (count - 1) + HK * page * D)) for _ in range(2)]
    for which, d in enumerate(big):
        host = np.ascontiguousarray(cache.view(which))
        for i in range(count):
            check(abi.lib.trs_memcpy_h2d(d.addr + size * step * i, host[i].ctypes.data, host[i].nbytes))
    cache.struct.k, cache.struct.v = big[0].addr, big[1].addr
    cache.struct.lk.stride[0] = cache.struct.lv.stride[0] = step
    out = Placed(shape=q.shape)
    check(paged_attention(Placed(q), cache, 0, EVERY, 0, 0.125, out))
    assert_within(out.numpy(), *attention_reference(q, k, v, EVERY, 0, 0.125, [160])["out"])


@KINDS
def test_without_memory_for_parts(kind):
    """The parts of long sequences are for speed alone."""
    for B, sq, shared in ((2, 1, 0), (2, 1, 320), (1, 200, 0), (33, 1, 880), (33, 40, 870), (2, 700, 0)):
        q, k, v = inputs(16, B, 8, 2, sq, 900, 64, kind)
        share(k, v, shared)
        Q = Placed(q)
        out = Placed(shape=q.shape)
        lengths = [900 - i for i in range(B)]
        cache = Cache(B, 2, 16, 64, lengths, kind, "heads", k, v, shared=shared)
        check(abi.lib.trs_debug_fail_allocs_after(0))
        try:
            rc = paged_attention(Q, cache, shared, EVERY, 0, 0.125, out)
        finally:
            check(abi.lib.trs_debug_fail_allocs_after(-1))
        check(rc)
        assert_within(out.numpy(), *attention_reference(q, k, v, EVERY, 0, 0.125, lengths)["out"])


@KINDS
def test_the_same_bits_each_time(kind):
    for B, sq, shared in ((5, 1, 0), (40, 1, 256), (40, 1, 1000), (40, 20, 1000), (2, 150, 0), (2, 800, 0), (1, 1, 0)):
        q, k, v = inputs(17, B, 8, 2, sq, 1100, 128, kind)
        share(k, v, shared)
        cache = Cache(B, 2, 16, 128, [1100 - 2 * i for i in range(B)], kind, "heads", k, v, shared=shared)
        Q, outs = Placed(q), []
        for _ in range(3):
            out = Placed(shape=q.shape)
            check(paged_attention(Q, cache, shared, EVERY, 0, 0.1, out))
            outs.append(out.numpy().view(np.uint32))
        assert np.array_equal(outs[0], outs[1]) and np.array_equal(outs[0], outs[2])


def test_refusals_and_calls_without_elements():
    q, k, v = inputs(18, 2, 4, 2, 3, 20, 16, F32)
    cache = Cache(2, 2, 4, 16, [20, 9], F32, "heads", k, v)
    Q, out = Placed(q), Placed(shape=q.shape)
    E, M = abi.TRS_E_INVALID_ARGUMENT, abi.TRS_E_SHAPE_MISMATCH

    def call(q=Q, cache=cache, shared=0, window=EVERY, sinks=0, scale=1.0, out=out):
        return paged_attention(q, cache, shared, window, sinks, scale, out)

    assert call() == 0
    assert call(window=0) == E and call(sinks=-1) == E and call(shared=-1) == E and call(scale=float("nan")) == E
    assert call(out=Q) == E and call(out=Placed(shape=q.shape, step=2)) == E and call(out=Placed(shape=(2, 4, 3, 15))) == M
    assert call(q=Placed(shape=(2, 3, 3, 16)), out=Placed(shape=(2, 3, 3, 16))) == M
    assert call(q=Placed(shape=(2, 4, 3, 8)), out=Placed(shape=(2, 4, 3, 8))) == M
    assert call(q=Placed(shape=(4, 3, 16))) == E
    big = Placed(shape=(2, 4, 3, 257))
    assert call(q=big, out=Placed(shape=big.shape), cache=Cache(2, 2, 4, 257, [20, 9])) == E
    for field, value in (("type", -1), ("table", None), ("lengths", None), ("v", None), ("table_width", -1)):
        broken = Cache(2, 2, 4, 16, [20, 9], F32, "heads", k, v)
        setattr(broken.struct, field, value)
        assert call(cache=broken) == E, field
    wide = Cache(2, 2, 4, 16, [20, 9], F32, "heads", k, v)
    wide.struct.table_width = 1 << 40
    assert call(cache=wide) == -2
    for shape in ((0, 4, 3, 16), (2, 0, 3, 16), (2, 4, 0, 16)):
        assert call(q=Placed(shape=shape), out=Placed(shape=shape), cache=Cache(shape[0], 2, 4, 16, [20, 9][:shape[0]])) == 0
    empty = Cache(2, 2, 4, 16, [5, 0], width=0)
    assert call(cache=empty) == 0
    assert not out.numpy().any()

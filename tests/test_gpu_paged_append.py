"""Keys and values appended to a paged cache: what is written, where, and that nothing else is."""
import numpy as np
import pytest

from attention_util import Placed, assert_within, ints, rotation_tables
from paged_util import BF16, F32, Cache, append, held, turned, turned_bound
from trs_backend import abi
from trs_backend.abi import check

pytestmark = pytest.mark.gpu
TOKENS = (0, 2, 1, 3)


def rows(seed, B, H, T, D):
    return np.random.default_rng(seed).standard_normal((B, H, T, D)).astype(np.float32)


def run(B, HK, T, D, page, lengths, kind=F32, form="heads", pairs=None, axes=1, pair_axes=None, positions=None, interleaved=False, query=0, table_rows=None,
        order=TOKENS, damage=None, **kw):
    """Appends to a pool that holds something everywhere, and compares all of it."""
    k, v = rows(1, B, HK, T, D), rows(2, B, HK, T, D)
    cache = Cache(B, HK, page, D, lengths, kind, form, **kw)
    rng = np.random.default_rng(3)
    for i, h in enumerate(cache.host):
        before = rng.standard_normal(h.shape).astype(np.float32)
        h[...] = before if kind == F32 else (before.view(np.uint32) >> 16).astype(np.uint16)
    cache.dev = [type(cache.dev[0]).from_numpy(h) for h in cache.host]
    cache.struct.k, cache.struct.v = cache.dev[0].addr, cache.dev[-1].addr
    if damage is not None:
        damage(cache)
    old = cache.fetch()
    memory = [h.copy() for h in cache.host]
    capacity = cache.table.shape[1] * page
    n = [max(x, 0) for x in lengths]
    place = np.array([[n[b] - T + t for t in range(T)] for b in range(B)]).reshape(B, T)
    at = np.broadcast_to(np.maximum(place, 0), (axes, B, T)) if positions is None else positions
    pairs = D // 2 if pairs is None else pairs
    cos, sin = rotation_tables((table_rows or max(int(np.max(at, initial=0)) + 1, 1)), 2 * pairs)
    C, S = (None, None) if pairs == 0 else (Placed(cos, pad=1), Placed(sin, pad=1))
    q = rows(4, B, query, T, D) if query else None
    Q, QO = (Placed(q, order=order), Placed(shape=q.shape, order=TOKENS, pad=2)) if query else (None, None)
    check(append(cache, Placed(k, order=order), Placed(v, order=order), Q, QO, C, S, interleaved, axes, pair_axes,
                 None if positions is None else ints(positions)))
    got = cache.fetch()
    want_k, bound_k = (turned(k, cos, sin, at, pair_axes, interleaved), turned_bound(k, pairs, interleaved)) if pairs else (k.astype(np.float64), np.zeros(k.shape))
    # A rounding to bfloat16 is off by half a step, 2^-8 of what it rounds, which is off by the bound itself, or half of the least step.
    if kind == BF16:
        bound_k = bound_k + 2.0 ** -8 * (abs(want_k) + bound_k) + 2.0 ** -134
    want = [p.astype(np.float64) for p in old]
    bounds = [np.zeros(p.shape) for p in old]
    for b in range(B):
        for t in range(T):
            p = place[b, t]
            if not 0 <= p < capacity:
                continue
            page_id = cache.table[b, p // page]
            if not 0 <= page_id < cache.shape[0]:
                continue
            want[0][page_id, :, p % page], bounds[0][page_id, :, p % page] = want_k[b, :, t], bound_k[b, :, t]
            want[1][page_id, :, p % page] = held(v[b, :, t], kind)
    for g, w, e in zip(got, want, bounds):
        assert_within(g, w, e)
    # What lies between the views' elements is as it was.
    for i, m in enumerate(memory):
        mine, his = cache.host[i].copy(), m.copy()
        views = [x for x in range(2) if x % len(memory) == i]
        for which in views:
            for flat in (mine, his):
                view = np.lib.stride_tricks.as_strided(flat[cache.offsets[which]:], cache.shape, tuple(s * flat.itemsize for s in cache.strides))
                view[...] = 0
        assert np.array_equal(mine, his)
    if query:
        y = QO.numpy()
        assert_within(y, turned(q, cos, sin, at, pair_axes, interleaved) if pairs else q, turned_bound(q, pairs, interleaved) if pairs else np.zeros(q.shape))
        assert QO.untouched()
    return got


#        B HK  T   D  page lengths
SHAPES = [
    (1, 1, 1, 2, 1, [1]), (1, 2, 1, 64, 16, [1]), (3, 2, 1, 128, 16, [17, 16, 33]), (2, 8, 1, 128, 16, [512, 100]), (2, 3, 5, 80, 8, [5, 21]),
    (1, 2, 40, 64, 16, [40]), (2, 2, 33, 32, 10, [40, 33]), (1, 1, 7, 7, 3, [9]), (1, 2, 3, 256, 64, [70]), (1, 1, 300, 48, 48, [301]),
    (4, 1, 2, 10, 5, [2, 6, 11, 15]), (1, 5, 65, 96, 128, [200]), (2, 1, 1, 1024, 4, [3, 9]), (1, 3, 2, 1, 2, [3]),
]


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_keys_and_values_stand_in_their_pages(shape, kind):
    B, HK, T, D, page, lengths = shape
    run(B, HK, T, D, page, lengths, kind, pairs=0)
    run(B, HK, T, D, page, lengths, kind, query=2 * HK)
    if D >= 8:
        pairs = D // 4
        axes = np.random.default_rng(D).integers(0, 3, pairs)
        positions = np.random.default_rng(T).integers(0, 40, (3, B, T))
        run(B, HK, T, D, page, lengths, kind, pairs=pairs, axes=3, pair_axes=axes.tolist(), positions=positions, interleaved=True, query=HK)


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("form", ["heads", "tokens", "both", "odd"])
@pytest.mark.parametrize("order", [TOKENS, (0, 1, 2, 3), (3, 1, 0, 2)], ids=str)
def test_pools_and_inputs_of_any_order(form, kind, order):
    run(2, 3, 6, 64, 16, [20, 38], kind, form, order=order, query=3)
    run(2, 2, 3, 20, 7, [20, 3], kind, form, order=order, query=2, pairs=5)


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("D", [64, 12])
def test_padding_lengths_beyond_the_table_and_bad_pages(kind, D):
    # Sequences shorter than the call's tokens, none at all, a negative length, and one beyond the table's row.
    run(5, 2, 6, D, 4, [3, 0, -5, 1000, 6], kind, query=2, width=4)
    # Tokens of which the table's row holds some, or just all, and a full row, which keeps what it has.
    run(4, 2, 6, D, 4, [18, 16, 17, 2 ** 31 - 1], kind, width=4, pairs=0)
    run(2, 2, 1, D, 4, [16, 17], kind, query=2, width=4)

    def damage(cache):  # pages that the pool does not have
        cache.table[0, 1], cache.table[1, 0], cache.table[1, 2] = cache.shape[0], -7, 2 ** 31 - 1
        cache.table_dev = ints(cache.table)
        cache.struct.table = cache.table_dev.addr

    run(2, 2, 9, D, 4, [9, 12], kind, query=2, damage=damage)


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
def test_positions_that_the_tables_do_not_hold(kind):
    run(2, 2, 4, 32, 8, [4, 14], kind, table_rows=10, query=2)
    run(2, 2, 4, 32, 8, [4, 14], kind, table_rows=10, query=2, axes=2, pair_axes=[0, 1] * 8, positions=np.array([[[0, 1, -1, 9], [10, 2, 2, 2]], [[9, 9, 9, 9], [0, 11, -2 ** 31, 2 ** 31 - 1]]]))


def test_values_round_to_the_nearest_even():
    bits = np.array([0x3F808000, 0x3F818000, 0x3F807FFF, 0x3F808001, 0x7F7FFFFF, 0xFF7FFFFF, 0x7F800000, 0xFF800000, 0x00000001, 0x00018000, 0x80008000, 0x00000000,
                     0x80000000, 0x477FE001, 0x00008001, 0x7F7F8000], np.uint32)
    v = bits.view(np.float32).reshape(1, 1, 1, 16)
    cache = Cache(1, 1, 4, 16, [1], BF16)
    check(append(cache, Placed(v), Placed(v)))
    got = cache.fetch()
    for pool in got:
        assert np.array_equal(pool[cache.table[0, 0], 0, 0].view(np.uint32), held(v, BF16).reshape(-1).view(np.uint32))
    nan = np.full((1, 1, 1, 16), np.nan, np.float32)
    check(append(cache, Placed(nan), Placed(nan)))
    assert np.isnan(cache.fetch()[0][cache.table[0, 0], 0, 0]).all()


def test_the_query_may_be_turned_in_place():
    k, v, q = rows(1, 1, 2, 3, 64), rows(2, 1, 2, 3, 64), rows(3, 1, 4, 3, 64)
    cos, sin = rotation_tables(8, 64)
    cache, Q = Cache(1, 2, 4, 64, [8]), Placed(q, order=TOKENS)
    check(append(cache, Placed(k), Placed(v), Q, Q, Placed(cos), Placed(sin)))
    assert_within(Q.numpy(), turned(q, cos, sin, np.array([[[5, 6, 7]]]), None, False), turned_bound(q, 32, False))


def test_refusals_and_calls_without_elements():
    k, v, q = (Placed(rows(i, 2, 2, 3, 16)) for i in range(3))
    cache = Cache(2, 2, 4, 16, [8, 5])
    E, M = abi.TRS_E_INVALID_ARGUMENT, abi.TRS_E_SHAPE_MISMATCH
    C, S = (Placed(t) for t in rotation_tables(8, 16))
    out = Placed(shape=(2, 2, 3, 16))
    assert append(cache, k, v, q, out, C, S) == 0
    assert append(cache, k, Placed(shape=(2, 2, 2, 16))) == M and append(cache, Placed(shape=(2, 1, 3, 16)), v) == M
    assert append(cache, Placed(shape=(2, 2, 3, 15)), v) == M and append(cache, Placed(shape=(2, 3, 16)), v) == E
    assert append(cache, k, v, None, out) == E and append(cache, k, v, q, None) == E and append(cache, k, v, q, k) == E
    assert append(cache, k, v, q, out, C, S, axes=0) == E and append(cache, k, v, q, out, C, S, axes=2, pair_axes=[2] * 8) == E
    big = [Placed(t) for t in rotation_tables(8, 18)]
    assert append(cache, k, v, None, None, *big) == M
    for field, value in (("type", 2), ("table", None), ("lengths", None), ("k", None), ("table_width", -1)):
        broken = Cache(2, 2, 4, 16, [8, 5])
        setattr(broken.struct, field, value)
        assert append(broken, k, v) == E, field
    same = Cache(2, 2, 4, 16, [8, 5])
    same.struct.v = same.struct.k
    assert append(same, k, v) == E
    twice = Cache(2, 2, 4, 16, [8, 5])
    twice.struct.lk.stride[0] = 1
    assert append(twice, k, v) == E
    strided = Cache(2, 2, 4, 16, [8, 5])
    strided.struct.lk.stride[3] = 2
    assert append(strided, k, v) == E
    for shape in ((0, 2, 3, 16), (2, 2, 0, 16)):
        e = Placed(shape=shape)
        assert append(Cache(shape[0], 2, 4, 16, [8, 5][:shape[0]]), e, e, e, Placed(shape=shape), C, S) == 0
    # A table without columns: nothing has a place.
    empty = Cache(2, 2, 4, 16, [0, 0], width=0)
    assert append(empty, k, v, q, out, C, S) == 0

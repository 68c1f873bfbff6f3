"""The paged cache's calls captured into graphs on the library's stream: replays see the lengths, tables and
tensors as they are then, and write to no memory that other calls have."""
import ctypes

import numpy as np
import pytest

from attention_util import EVERY, Placed, assert_within, attention_reference, ints, rotation_tables
from paged_util import BF16, F32, Cache, append, held, paged_attention, turned, turned_bound
from trs_backend import abi
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu
RELAXED = 2


def rows(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


class Graph:
    """The work that `calls` queue, captured; nothing of it runs before `replay`."""

    def __init__(self, calls):
        self.hip = abi.lib  # its symbols are found through the library that needs them
        stream = ctypes.c_void_p()
        check(abi.lib.trs_stream(ctypes.byref(stream)))
        self.stream, self.graph, self.run = stream, ctypes.c_void_p(), ctypes.c_void_p()
        self.ok(self.hip.hipStreamBeginCapture(stream, RELAXED))
        try:
            calls()
        finally:
            rc = self.hip.hipStreamEndCapture(stream, ctypes.byref(self.graph))
        self.ok(rc)
        self.ok(self.hip.hipGraphInstantiate(ctypes.byref(self.run), self.graph, None, None, ctypes.c_size_t(0)))

    @staticmethod
    def ok(rc):
        assert rc == 0, f"HIP error {rc}"

    def replay(self):
        self.ok(self.hip.hipGraphLaunch(self.run, self.stream))

    def close(self):
        check(abi.lib.trs_synchronize())
        self.ok(self.hip.hipGraphExecDestroy(self.run))
        self.ok(self.hip.hipGraphDestroy(self.graph))


def put(array, values):
    values = np.ascontiguousarray(values)
    check(abi.lib.trs_memcpy_h2d(array.addr, values.ctypes.data, values.nbytes))


# B HK H  sq shared: one token with and without parts, shared keys in both stages, prompts.
CASES = [(1, 2, 8, 1, 0), (5, 2, 8, 1, 0), (40, 2, 8, 1, 512), (33, 2, 4, 40, 840), (1, 2, 8, 700, 0)]


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
def test_replays_are_as_the_calls(kind):
    made = []
    for i, (B, HK, H, sq, shared) in enumerate(CASES):
        D, page, most = 64, 16, 900
        k, v = (held(rows(10 * i + j, B, HK, most, D), kind) for j in range(2))
        k[:, :, :shared], v[:, :, :shared] = k[:1, :, :shared], v[:1, :, :shared]
        q = rows(10 * i + 2, B, H, sq, D)
        cache = Cache(B, HK, page, D, [most] * B, kind, "heads", k, v, shared=shared)
        Q, out, eager = Placed(q), Placed(shape=q.shape), Placed(shape=q.shape)
        lse = [DeviceArray(4 * B * H * sq) for _ in range(2)]
        graph = Graph(lambda: check(paged_attention(Q, cache, shared, EVERY, 0, 0.125, out, lse[0])))
        made.append((graph, cache, Q, out, eager, lse, k, v, q, shared))
    rng = np.random.default_rng(0)
    for turn in range(4):
        # Memory of all the sizes that calls take and give back, held over the replays.
        mine = [(DeviceArray.from_numpy(np.full(n // 4, 7, np.float32)), n) for n in (1 << 16, 1 << 20, 1 << 22, 1 << 24, 1 << 25, 1 << 26)]
        for graph, cache, Q, out, eager, lse, k, v, q, shared in made:
            lengths = rng.integers(max(shared, 1), 901, q.shape[0])
            put(cache.lengths_dev, lengths.astype(np.int32))
            graph.replay()
            check(paged_attention(Q, cache, shared, EVERY, 0, 0.125, eager, lse[1]))
            got = out.numpy()
            assert np.array_equal(got.view(np.uint32), eager.numpy().view(np.uint32))
            a, b = (np.zeros(q.shape[:3], np.float32) for _ in range(2))
            for d, h in zip(lse, (a, b)):
                check(abi.lib.trs_memcpy_d2h(h.ctypes.data, d.addr, h.nbytes))
            assert np.array_equal(a, b)
            if turn == 3:
                assert_within(got, *attention_reference(q, k, v, EVERY, 0, 0.125, lengths.tolist())["out"])
        for graph, *_ in made:  # and one behind another, unwaited
            graph.replay()
        for d, n in mine:
            assert (d.to_numpy() == 7).all()
    for m in made:
        m[0].close()


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
def test_a_captured_step_serves_token_after_token(kind):
    """A token appended, its query turned, and attention, captured once and replayed with longer lengths."""
    B, HK, H, D, page, n = 3, 2, 4, 64, 16, 40
    k, v, q = rows(1, B, HK, n, D), rows(2, B, HK, n, D), rows(3, B, H, n, D)
    cos, sin = rotation_tables(n + 8, D)
    caches = [Cache(B, HK, page, D, [n + 4] * B, kind) for _ in range(2)]
    C, S = Placed(cos), Placed(sin)
    K, V, Q, T, out = (Placed(shape=(B, h, 1, D)) for h in (HK, HK, H, H, H))
    T2, out2 = Placed(shape=(B, H, 1, D)), Placed(shape=(B, H, 1, D))

    def step(cache, turned, o):
        check(append(cache, K, V, Q, turned, C, S))
        check(paged_attention(turned, cache, 0, EVERY, 0, 0.125, o))

    graph = Graph(lambda: step(caches[0], T, out))
    for t in range(n):
        for p, x in ((K, k), (V, v), (Q, q)):
            put(p.dev, np.concatenate([x[:, :, t].reshape(-1), np.zeros(8, np.float32)]))
        for c in caches:
            put(c.lengths_dev, np.array([t + 1, max(t - 2, 0), t + 4], np.int32))
        graph.replay()
        step(caches[1], T2, out2)
        # (The third sequence's first three places hold NaN, which its tokens see.)
        assert np.array_equal(out.numpy(), out2.numpy(), equal_nan=True) and np.array_equal(T.numpy(), T2.numpy())
    kt, qt = (turned(x[:1], cos, sin, np.arange(n)[None, None], None, False).astype(np.float32) for x in (k, q))
    assert_within(T.numpy()[:1], turned(q[:1, :, -1:], cos, sin, np.array([[[n - 1]]]), None, False), turned_bound(q[:1, :, -1:], D // 2, False))
    if kind == F32:
        # A score's turned operands are off by 3 half units each of their own, which is within what the bound allows for dim + 8 = 72.
        want, bound = attention_reference(qt[:, :, -1:], kt, v[:1], EVERY, 0, 0.125)["out"]
        assert_within(out.numpy()[:1], want, 2 * bound)
    for x, y in zip(caches[0].fetch(), caches[1].fetch()):
        assert np.array_equal(x, y, equal_nan=True)
    graph.close()


def test_a_captured_call_refuses_a_query_that_is_copied_first():
    q, k, v = rows(1, 1, 2, 1, 32), rows(2, 1, 2, 20, 32), rows(3, 1, 2, 20, 32)
    cache, out = Cache(1, 2, 16, 32, [20], F32, "heads", k, v), Placed(shape=q.shape)
    Q, strided = Placed(q), Placed(q, step=2)
    got = []

    def calls():
        got.append(paged_attention(strided, cache, 0, EVERY, 0, 0.125, out))
        got.append(paged_attention(Q, cache, 0, EVERY, 0, 0.125, out))

    graph = Graph(calls)
    assert got == [abi.TRS_E_INVALID_ARGUMENT, 0]
    graph.replay()
    assert_within(out.numpy(), *attention_reference(q, k, v, EVERY, 0, 0.125)["out"])
    graph.close()

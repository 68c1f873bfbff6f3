"""Captured calls of paged attention that find no memory, and captures in which nothing may be allocated: the capture goes
on, the block cache keeps its blocks, and replays give the formula's values."""
import ctypes

import numpy as np
import pytest

from attention_util import EVERY, Placed, assert_within, attention_reference
from paged_util import BF16, F32, Cache, held, paged_attention
from test_gpu_paged_graph import Graph, rows
from trs_backend import abi
from trs_backend.abi import check

pytestmark = pytest.mark.gpu
GLOBAL, THREAD_LOCAL, RELAXED = 0, 1, 2
ALLOCATION_FAILED = -1
KINDS = pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])


class Captured(Graph):
    """A graph captured in a mode of its own."""

    def __init__(self, calls, mode=RELAXED):
        self.hip = abi.lib
        self.stream, self.graph, self.run = ctypes.c_void_p(), ctypes.c_void_p(), ctypes.c_void_p()
        check(abi.lib.trs_stream(ctypes.byref(self.stream)))
        self.ok(self.hip.hipStreamBeginCapture(self.stream, mode))
        try:
            calls()
        finally:
            rc = self.hip.hipStreamEndCapture(self.stream, ctypes.byref(self.graph))
        self.ok(rc)
        self.ok(self.hip.hipGraphInstantiate(ctypes.byref(self.run), self.graph, None, None, ctypes.c_size_t(0)))


def stats():
    live, cached = ctypes.c_size_t(), ctypes.c_size_t()
    check(abi.lib.trs_memory_stats(ctypes.byref(live), ctypes.byref(cached)))
    return live.value, cached.value


class Case:
    """Inputs of a call whose parts take more memory than other tests' captured calls: so many key heads, and one worker a head at least."""

    def __init__(self, seed, B, H, HK, sq, D, n, kind, shared=0):
        k, v = (held(rows(seed + i, B, HK, n, D), kind) for i in range(2))
        k[:, :, :shared], v[:, :, :shared] = k[:1, :, :shared], v[:1, :, :shared]
        q = rows(seed + 2, B, H, sq, D)
        self.shared, self.scale = shared, D ** -0.5
        self.cache = Cache(B, HK, 16, D, [n - i for i in range(B)], kind, "heads", k, v, shared=shared)
        self.q, self.out = Placed(q), Placed(shape=q.shape)
        self.want = attention_reference(q, k, v, EVERY, 0, self.scale, [n - i for i in range(B)])["out"]

    def call(self):
        return paged_attention(self.q, self.cache, self.shared, EVERY, 0, self.scale, self.out)

    def replays_right(self, graph):
        before = Placed(shape=self.out.shape)
        for _ in range(3):
            check(abi.lib.trs_memcpy_d2d(self.out.dev.addr, before.dev.addr, 4 * self.out.size))
            graph.replay()
            assert_within(self.out.numpy(), *self.want)
            Placed(rows(1, 1 << 16)).numpy()  # other work between the replays


# Few rows and many, of one stage and of two.
SIZES = pytest.mark.parametrize("size", [(1, 8192, 8192, 1, 64, 40), (1, 512, 512, 70, 64, 260), (2, 4096, 4096, 1, 64, 40, 32)], ids=str)


def case_of(size, kind, seed=0):
    B, H, HK, sq, D, n, shared = (*size, 0)[:7]
    return Case(seed, B, H, HK, sq, D, n, kind, shared)


@KINDS
@SIZES
def test_a_captured_call_without_memory_for_parts_takes_none(kind, size):
    case = case_of(size, kind)
    before = stats()
    check(abi.lib.trs_debug_fail_allocs_after(0))
    try:
        graph = Captured(lambda: check(case.call()))
    finally:
        check(abi.lib.trs_debug_fail_allocs_after(-1))
    assert stats() == before
    case.replays_right(graph)
    graph.close()


def test_an_allocation_that_the_device_refuses_ends_no_capture_and_drops_no_block():
    case = Case(3, 2, 8, 2, 1, 64, 900, F32)
    check(case.call())  # blocks in the cache, the call's workspace among them
    check(abi.lib.trs_synchronize())
    before, got = stats(), []
    assert before[1] > 0

    def calls():
        p = ctypes.c_void_p()
        got.append(abi.lib.trs_alloc(1 << 52, ctypes.byref(p)))  # more than there is
        got.append(p.value)
        got.append(stats())
        check(case.call())

    graph = Captured(calls)
    assert got == [ALLOCATION_FAILED, None, before]
    case.replays_right(graph)
    graph.close()


def test_the_cache_is_not_emptied_in_a_capture():
    """Its blocks wait for the stream, which cannot be waited for: the call is refused, and the capture goes on."""
    case = Case(4, 2, 8, 2, 1, 64, 900, F32)
    check(case.call())
    check(abi.lib.trs_synchronize())
    before, got = stats(), []
    assert before[1] > 0

    def calls():
        got.append(abi.lib.trs_empty_cache())
        got.append(stats())
        check(case.call())

    graph = Captured(calls)
    assert got == [abi.TRS_E_INVALID_ARGUMENT, before]
    case.replays_right(graph)
    graph.close()
    check(abi.lib.trs_empty_cache())
    assert stats()[1] == 0


@pytest.mark.parametrize("mode", [GLOBAL, THREAD_LOCAL, RELAXED])
@KINDS
@SIZES
def test_captures_of_any_mode(kind, size, mode):
    """With no block of the workspace's size in the cache."""
    # One more head each time, so that no call before this one has had so large a workspace.
    B, H, HK, *rest = size
    more = 1 + mode + 3 * (kind == BF16)
    case = case_of((B, H + 8 * more, HK + 8 * more, *rest), kind)
    check(abi.lib.trs_empty_cache())
    graph = Captured(lambda: check(case.call()), mode)
    case.replays_right(graph)
    graph.close()


@pytest.mark.parametrize("mode", [GLOBAL, THREAD_LOCAL])
@KINDS
def test_captures_of_any_mode_after_the_same_call(kind, mode):
    case = Case(5 + mode, 3, 8, 2, 2, 80, 700, kind)
    check(case.call())
    graph = Captured(lambda: check(case.call()), mode)
    case.replays_right(graph)
    graph.close()

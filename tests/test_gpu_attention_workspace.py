"""The workspace of attention's gradients: its size where sinks are few, and a smaller one
where there is no memory for parts."""
import ctypes

import numpy as np
import pytest

from attention_util import Placed, assert_within, attention, attention_grad, attention_reference
from trs_backend import abi
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu


def operands(seed, B, H, hk, n, D):
    rng = np.random.default_rng(seed)
    return tuple(rng.standard_normal(s).astype(np.float32) for s in ((B, H, n, D), (B, hk, n, D), (B, hk, n, D), (B, H, n, D)))


def forward(q, k, v, window, sinks):
    P, out, lse = [Placed(t) for t in (q, k, v)], Placed(shape=q.shape), DeviceArray(4 * int(np.prod(q.shape[:3])))
    check(attention(*P, window, sinks, 0.2, out, lse))
    return P, out, lse


def facts(B, H, n):
    return 5 * (-(-B * H * n // 64) * 64)


@pytest.mark.parametrize("D", [64, 128, 160])
def test_few_sinks_take_little_memory(D):
    """64 key heads of 4 sinks: no more than 64 parts of these 4 keys, and 16 of all keys."""
    B, H, n, window, sinks = 1, 128, 700, 16, 4
    q, k, v, up = operands(1, B, H, 64, n, D)
    P, out, lse = forward(q, k, v, window, sinks)
    U, grads = Placed(up), [Placed(shape=t.shape) for t in (q, k, v)]
    check(abi.lib.trs_empty_cache())
    check(attention_grad(*P, window, sinks, 0.2, out, lse, U, *grads))
    live, cached = ctypes.c_size_t(), ctypes.c_size_t()
    check(abi.lib.trs_memory_stats(ctypes.byref(live), ctypes.byref(cached)))
    # At most as many of the near pairs' parts as fill a CU with two blocks or eight waves each.
    parts = 2 * 64 * n * D * max(1, 8 * 256 // (64 * (n // 16))) if D > 128 else 0
    assert cached.value <= 4 * (facts(B, H, n) + 2 * 64 * 64 * sinks * D + parts) + (2 << 20)
    want = attention_reference(q[:, :4], k[:, :2], v[:, :2], window, sinks, np.float32(0.2), up=up[:, :4])
    for name, g, heads in zip(("dq", "dk", "dv"), grads, (4, 2, 2)):
        assert_within(g.numpy()[:, :heads], *want[name], name)


@pytest.mark.parametrize("sinks", [0, 3, 150])
@pytest.mark.parametrize("D", [30, 64, 128, 160])
def test_gradients_without_memory_for_parts(D, sinks):
    B, H, hk, n, window = 2, 4, 2, 400, 40
    q, k, v, up = operands(2, B, H, hk, n, D)
    want = attention_reference(q, k, v, window, sinks, np.float32(0.2), up=up)
    P, out, lse = forward(q, k, v, window, sinks)
    U, grads = Placed(up), [Placed(shape=t.shape) for t in (q, k, v)]
    least = 4 * (facts(B, H, n) + 2 * B * hk * sinks * D)
    try:
        check(abi.lib.trs_debug_fail_allocs_above(least))
        done = attention_grad(*P, window, sinks, 0.2, out, lse, U, *grads)
        got = [g.numpy() for g in grads]
        check(abi.lib.trs_debug_fail_allocs_above(least - 1))
        refused = attention_grad(*P, window, sinks, 0.2, out, lse, U, *grads)
    finally:
        check(abi.lib.trs_debug_fail_allocs_above(0))
    assert (done, refused) == (0, -1)
    for name, g in zip(("dq", "dk", "dv"), got):
        assert_within(g, *want[name], name)

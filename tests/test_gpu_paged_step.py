"""The paged cache as a model uses it: prompts and tokens appended, then read, through
torch_rs and as consecutive calls, with prefixes that sequences share, and beside
other calls."""
import ctypes
import sys
from pathlib import Path

import numpy as np
import pytest

import torch_rs
from attention_util import EVERY, Placed, assert_within, attention_reference, ints, rotation_tables
from paged_util import BF16, F32, Cache, append, held, paged_attention, turned
from trs_backend import abi
from trs_backend.abi import check

pytestmark = pytest.mark.gpu
F = torch_rs.nn.functional
ROOT = Path(__file__).resolve().parent.parent


def rows(seed, *shape):
    return np.random.default_rng(seed).standard_normal(shape).astype(np.float32)


def device(x, grad=False):
    return torch_rs.tensor(x, device="cuda", requires_grad=grad)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_a_prompt_and_tokens_as_a_model_serves_them(dtype):
    """Two ragged prompts padded in front, then tokens one by one: each step's output against attention over all that was appended."""
    kind = BF16 if dtype == "bfloat16" else F32
    B, H, HK, D, page, lengths = 2, 4, 2, 32, 8, [21, 13]
    table = np.array([[7, 2, 9, 0, 4], [1, 8, 3, 6, 5]])
    cache = F.paged_cache(10, HK, page, D, dtype)
    assert cache.shape == (10, HK, page, D) and cache.dtype == dtype and cache.device == "cuda:0"
    cos, sin = rotation_tables(64, D)
    C, S = device(cos), device(sin)
    K, V = (np.zeros((B, HK, 40, D), np.float32) for _ in range(2))
    pages = F.index_buffer(table)
    with torch_rs.no_grad():
        for step, T in enumerate((21, 1, 1, 2, 1)):
            if step:
                lengths = [n + T for n in lengths]
            q, k, v = rows(step, B, H, T, D), rows(100 + step, B, HK, T, D), rows(200 + step, B, HK, T, D)
            place = np.array([[n - T + t for t in range(T)] for n in lengths])
            at = np.maximum(place, 0)[None]
            kt, qt = (turned(x, cos, sin, at, None, False).astype(np.float32) for x in (k, q))
            for b in range(B):
                for t in range(T):
                    if place[b, t] >= 0:
                        K[b, :, place[b, t]], V[b, :, place[b, t]] = held(kt[b, :, t], kind), held(v[b, :, t], kind)
            n = F.index_buffer(lengths)
            Q = F.paged_append(cache, pages, n, device(k), device(v), C, S, query=device(q))
            out = F.paged_attention(Q, cache, pages, n, window=20, sinks=2).numpy()
            want, bound = attention_reference(qt, K, V, 20, 2, D ** -0.5, lengths)["out"]
            # A key that rounds the other way moves each score by a step of bfloat16 in one entry; the rotation's own roundings are below the bound.
            slack = 0 if kind == F32 else 2.0 ** -8 * (abs(qt).max() * abs(K).max() * D ** -0.5) * abs(V).max() * 2.0 ** -4
            assert_within(out, want, 2 * bound + slack + 1e-6)


def test_appended_without_rotation_and_with_axes_through_torch_rs():
    B, H, HK, T, D = 1, 2, 1, 6, 16
    q, k, v = rows(1, B, H, T, D), rows(2, B, HK, T, D), rows(3, B, HK, T, D)
    cos, sin = rotation_tables(9, D)
    positions, axes = np.random.default_rng(0).integers(0, 9, (3, B, T)), [0, 1, 2, 0, 1, 2, 0, 1]
    cache = F.paged_cache(2, HK, 4, D)
    assert F.paged_append(cache, [[1, 0]], [6], device(k), device(v)) is None
    got = F.paged_attention(device(q), cache, [[1, 0]], [6]).numpy()
    assert_within(got, *attention_reference(q, k, v, EVERY, 0, D ** -0.5)["out"])
    Q = F.paged_append(cache, [[1, 0]], [6], device(k), device(v), device(cos), device(sin), query=device(q), positions=positions, pair_axes=axes, interleaved=True)
    kt, qt = (turned(x, cos, sin, positions, axes, True).astype(np.float32) for x in (k, q))
    want, bound = attention_reference(qt, kt, v, EVERY, 0, D ** -0.5)["out"]
    assert_within(F.paged_attention(Q, cache, [[1, 0]], [6]).numpy(), want, 2 * bound + 1e-6)
    # The same as the two calls apart.
    apart = F.rope_axes(device(q), device(k), device(cos), device(sin), positions=positions, pair_axes=axes, interleaved=True)
    assert np.array_equal(apart[0].numpy(), Q.numpy())


def test_refusals_through_torch_rs():
    x, one = device(rows(1, 1, 2, 3, 8)), device(rows(2, 1, 1, 3, 8))
    cache = F.paged_cache(4, 1, 4, 8)
    with pytest.raises(RuntimeError, match="no gradient"):
        F.paged_attention(device(rows(1, 1, 2, 3, 8), True), cache, [[0]], [3])
    with pytest.raises(RuntimeError, match="no gradient"):
        F.paged_append(cache, [[0]], [3], device(rows(1, 1, 1, 3, 8), True), one)
    with torch_rs.no_grad():
        F.paged_attention(device(rows(1, 1, 2, 3, 8), True), cache, [[0]], [3])
    with pytest.raises(RuntimeError, match="table has shape"):
        F.paged_attention(x, cache, [0], [3])
    with pytest.raises(RuntimeError, match="lengths have shape"):
        F.paged_attention(x, cache, [[0]], [3, 4])
    with pytest.raises(RuntimeError, match="positions have shape"):
        F.paged_append(cache, [[0]], [3], one, one, device(rows(1, 4, 4)), device(rows(1, 4, 4)), positions=[[0, 1]])
    with pytest.raises(RuntimeError, match="positions have shape"):
        F.rope_axes(x, None, device(rows(1, 4, 4)), device(rows(1, 4, 4)), positions=5)
    with pytest.raises(RuntimeError, match="axes for 3 pairs"):
        F.rope_axes(x, None, device(rows(1, 4, 4)), device(rows(1, 4, 4)), pair_axes=[0, 0, 0])
    with pytest.raises(RuntimeError, match="4 dims"):
        F.rope_axes(device(rows(1, 3, 8)), None, device(rows(1, 4, 4)), device(rows(1, 4, 4)))
    with pytest.raises(RuntimeError, match="at least one page"):
        F.paged_cache(0, 1, 4, 8)
    with pytest.raises(ValueError, match="shared"):
        F.paged_attention(x, cache, [[0]], [3], shared=-1)


def test_a_shared_prefix_through_torch_rs_is_as_each_sequence_alone():
    B, H, HK, D, page, shared = 3, 4, 2, 16, 4, 10
    prefix_k, prefix_v = rows(1, 1, HK, shared, D), rows(2, 1, HK, shared, D)
    cache = F.paged_cache(12, HK, page, D)
    # The first two pages are shared; the third, which the prefix half fills, is each sequence's own.
    table = np.array([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 6, 7]])
    for b in range(B):
        F.paged_append(cache, table[b:b + 1], [shared], device(prefix_k), device(prefix_v))
    k, v, q = rows(3, B, HK, 3, D), rows(4, B, HK, 3, D), rows(5, B, H, 1, D)
    F.paged_append(cache, table, [shared + 3] * B, device(k), device(v))
    alone = F.paged_attention(device(q), cache, table, [shared + 3] * B).numpy()
    together = F.paged_attention(device(q), cache, table, [shared + 3] * B, shared=shared).numpy()
    K, V = (np.concatenate((np.repeat(p, B, 0), x), 2) for p, x in ((prefix_k, k), (prefix_v, v)))
    want = attention_reference(q, K, V, EVERY, 0, D ** -0.5)["out"]
    assert_within(alone, *want)
    assert_within(together, *want)


def test_a_token_of_the_example_block_is_as_in_the_whole_prompt():
    sys.path.insert(0, str(ROOT / "examples"))
    from attention_block import AttentionBlock

    block = AttentionBlock(width=96, heads=4, kv_heads=2, dim=24, window=16, sinks=2, positions=64)
    x = rows(1, 2 * 40, 96)
    with torch_rs.no_grad():
        whole = block(device(x), 2).numpy().reshape(2, 40, 96)
        cache = F.paged_cache(2 * 6, 2, 8, 24)
        table = np.arange(12).reshape(2, 6)[:, ::-1]
        got = [block.serve(device(np.ascontiguousarray(x.reshape(2, 40, 96)[:, :33].reshape(-1, 96))), cache, table, [33, 33]).numpy().reshape(2, 33, 96)]
        for t in range(33, 40):
            got.append(block.serve(device(np.ascontiguousarray(x.reshape(2, 40, 96)[:, t])), cache, table, [t + 1] * 2).numpy().reshape(2, 1, 96))
    # Sums of the same products in another order: no value above 8 here, and some hundred terms at 2^-24 each.
    assert abs(np.concatenate(got, 1) - whole).max() < 1e-4


@pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])
def test_two_callers_at_once(kind):
    """Threads with caches of their own: the library's stream orders their work."""
    import threading

    results = {}

    def work(i):
        B, H, HK, D = 4, 8, 2, 64
        k, v = (held(rows(10 * i + j, B, HK, 300, D), kind) for j in range(2))
        q = rows(10 * i + 2, B, H, 1, D)
        cache = Cache(B, HK, 16, D, [300, 200, 100, 50], kind, "heads", k, v, seed=i)
        ok = True
        for _ in range(20):
            out = Placed(shape=q.shape)
            check(paged_attention(Placed(q), cache, 0, EVERY, 0, 0.125, out))
            got = out.numpy()
            want, bound = attention_reference(q, k, v, EVERY, 0, 0.125, [300, 200, 100, 50])["out"] if i not in results else results[i]
            results[i] = want, bound
            ok = ok and bool((abs(got - want) <= bound).all())
        results[i, "ok"] = ok

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert all(results[i, "ok"] for i in range(3))


def test_steps_in_order_without_waiting():
    """Appends and attention queued one behind another: each sees what those before it wrote, and only that."""
    B, H, HK, D, page = 2, 4, 2, 64, 16
    k, v, q = rows(1, B, HK, 30, D), rows(2, B, HK, 30, D), rows(3, B, H, 30, D)
    cache = Cache(B, HK, page, D, [30, 30], F32, extra=0)
    outs, keep = [], []
    for t in range(30):
        n = ints([t + 1, t + 1])
        cache.struct.lengths = n.addr
        K, V, Q, O = Placed(k[:, :, t:t + 1]), Placed(v[:, :, t:t + 1]), Placed(q[:, :, t:t + 1]), Placed(shape=(B, H, 1, D))
        check(append(cache, K, V))
        check(paged_attention(Q, cache, 0, EVERY, 0, 0.125, O))
        outs.append(O)
        keep += [n, K, V, Q]
    for t, o in enumerate(outs):
        assert_within(o.numpy(), *attention_reference(q[:, :, t:t + 1], k, v, EVERY, 0, 0.125, [t + 1] * B)["out"])


def test_the_librarys_memory_is_returned():
    live = ctypes.c_size_t()
    q, k, v = rows(1, 2, 8, 1, 64), rows(2, 2, 2, 900, 64), rows(3, 2, 2, 900, 64)
    cache = Cache(2, 2, 16, 64, [900, 800], F32, "heads", k, v)
    Q, out = Placed(q), Placed(shape=q.shape)
    check(abi.lib.trs_memory_stats(ctypes.byref(live), None))
    before = live.value
    for _ in range(5):
        check(paged_attention(Q, cache, 0, EVERY, 0, 0.125, out))
    check(abi.lib.trs_memory_stats(ctypes.byref(live), None))
    assert live.value == before

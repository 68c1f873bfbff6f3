"""Shared keys of which a window leaves few: a prefix that saves no reading does not change the call."""
import numpy as np
import pytest

from attention_util import Placed, assert_within, attention_reference, ints
from paged_util import BF16, F32, Cache, held, paged_attention
from trs_backend.abi import check

pytestmark = pytest.mark.gpu
KINDS = pytest.mark.parametrize("kind", [F32, BF16], ids=["f32", "bf16"])


@KINDS
@pytest.mark.parametrize("B,H,HK,sq,D,window,sinks", [(64, 8, 2, 1, 64, 16, 0), (33, 8, 2, 2, 128, 100, 4), (40, 8, 2, 30, 64, 64, 0)])
def test_shared_keys_that_a_window_hides_change_nothing(kind, B, H, HK, sq, D, window, sinks):
    """A prefix of 8192 keys of which a query sees at most some hundred saves no reading: the call is the one without it, bit for bit."""
    shared, page = 8192, 16
    lengths = [shared + 1 + 7 * i if i % 3 else shared - 50 * i - 1 for i in range(B)]
    rng = np.random.default_rng(B + D)
    q = rng.standard_normal((B, H, sq, D)).astype(np.float32)
    k, v = (held(rng.standard_normal((B, HK, max(lengths), D)).astype(np.float32), kind) for _ in range(2))
    for x in (k, v):
        x[:, :, :shared] = x[:1, :, :shared]
    cache = Cache(B, HK, page, D, lengths, kind, "heads", k, v, shared=shared)
    cache.table[1:, :shared // page] = cache.table[:1, :shared // page]
    cache.table_dev = ints(cache.table)
    cache.struct.table = cache.table_dev.addr
    outs = [Placed(shape=q.shape) for _ in range(2)]
    for out, s in zip(outs, (0, shared)):
        check(paged_attention(Placed(q), cache, s, window, sinks, D ** -0.5, out))
    apart, together = (out.numpy() for out in outs)
    assert_within(apart, *attention_reference(q, k, v, window, sinks, D ** -0.5, lengths)["out"])
    assert np.array_equal(apart.view(np.uint32), together.view(np.uint32))

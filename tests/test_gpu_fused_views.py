"""Operands that are slices of one buffer, as a fused projection of queries, keys and values
leaves them: outputs between inputs are written, and what shares an element is refused."""
import ctypes

import numpy as np
import pytest

from attention_util import (assert_within, attention, attention_grad, attention_reference, norm_rope, norm_rope_reference, Placed,
                            rotation_tables, U)
from trs_backend import abi
from trs_backend.abi import DeviceArray, check, layout_of

pytestmark = pytest.mark.gpu


class Slice:
    """Heads `first` on of a [batch, token, heads, dim] buffer, as [batch, head, token, dim]."""

    def __init__(self, dev, whole, first, heads, dim=None, at=0):
        B, S, H, D = whole
        self.dev, self.whole, self.first, self.heads = dev, whole, first, heads
        self.layout = layout_of((B, heads, S, dim or D), (S * H * D, D, H * D, 1), first * D + at)

    @property
    def arg(self):
        return self.dev.ptr, ctypes.byref(self.layout)

    def numpy(self):
        return self.dev.to_numpy(count=int(np.prod(self.whole))).reshape(self.whole)[:, :, self.first: self.first + self.heads].transpose(0, 2, 1, 3)


def buffer(values):
    return DeviceArray.from_numpy(np.ascontiguousarray(values, dtype=np.float32))


@pytest.mark.parametrize("B, S, H, HK, D", [(2, 70, 4, 2, 64), (1, 33, 3, 1, 128), (2, 1, 2, 2, 30), (3, 5, 4, 1, 160)])
def test_attention_and_gradients_within_one_buffer(B, S, H, HK, D):
    """q, k, v, up, dq, dk and dv are heads of one buffer, and so is the output."""
    rng = np.random.default_rng(S)
    heads = [H, HK, HK, H, H, H, HK, HK]  # q, k, v, up, out, dq, dk, dv
    first = np.cumsum([0] + heads)
    host = np.full((B, S, first[-1], D), np.nan, np.float32)
    host[:, :, : first[4]] = rng.standard_normal((B, S, first[4], D))
    dev = buffer(host)
    q, k, v, up, out, dq, dk, dv = (Slice(dev, host.shape, f, n) for f, n in zip(first, heads))
    lse = DeviceArray(4 * B * H * S)
    check(attention(q, k, v, 20, 2, 0.2, out, lse))
    check(attention_grad(q, k, v, 20, 2, 0.2, out, lse, up, dq, dk, dv))
    want = attention_reference(*(t.numpy() for t in (q, k, v)), 20, 2, np.float32(0.2), up=up.numpy())
    for name, t in (("out", out), ("dq", dq), ("dk", dk), ("dv", dv)):
        assert_within(t.numpy(), *want[name], name)
    assert np.array_equal(dev.to_numpy(count=host.size).reshape(host.shape)[:, :, : first[4]], host[:, :, : first[4]])


@pytest.mark.parametrize("D", [64, 20])
def test_norms_of_heads_into_slices_of_one_buffer(D):
    B, S, H, HK = 2, 9, 4, 2
    rng = np.random.default_rng(D)
    host = rng.standard_normal((B, S, 2 * (H + HK), D)).astype(np.float32)
    dev = buffer(host)
    q, k, yq, yk = (Slice(dev, host.shape, f, n) for f, n in ((0, H), (H, HK), (H + HK, H), (2 * H + HK, HK)))
    cos, sin = rotation_tables(S, D)
    C, Sn = Placed(cos), Placed(sin)
    check(norm_rope([q, k], [None, None], 1e-6, C, Sn, False, None, 0, [yq, yk]))
    at = np.broadcast_to(np.arange(S), (B, S))
    for x, y in ((q, yq), (k, yk)):
        x = x.numpy()
        # The bound of the tests of this operator: the mean's halves, then five roundings.
        r = 1 / np.sqrt((x.astype(np.float64) ** 2).mean(-1, keepdims=True) + 1e-6)
        bound = (D / 2 + 12) * U * 2 * abs(x).max(-1, keepdims=True) * r * np.ones(D)
        assert_within(y.numpy(), norm_rope_reference(x, None, 1e-6, cos, sin, at, False), bound)
    assert np.array_equal(dev.to_numpy(count=host.size).reshape(host.shape)[:, :, : H + HK], host[:, :, : H + HK])


def test_slices_that_share_an_element_are_refused():
    B, S, D = 2, 8, 16
    dev, E = buffer(np.zeros((B, S + 1, 12, D))), abi.TRS_E_INVALID_ARGUMENT
    whole = (B, S, 12, D)

    def call(out_first, at=0, dim=D):
        q, k, v = Slice(dev, whole, 0, 4, dim), Slice(dev, whole, 4, 2, dim), Slice(dev, whole, 6, 2, dim)
        return attention(q, k, v, 4, 0, 1.0, Slice(dev, whole, out_first, 4, dim, at))

    assert call(8) == 0
    assert call(7) == E  # a head of the values
    assert call(0) == E
    assert call(8, -1) == E  # one element of them
    assert call(8, 1) == E    # the next token's first query
    assert call(8, 1, D - 1) == 0  # narrower heads: none
    other = Slice(dev, whole, 8, 4)
    other.layout = layout_of((B, 4, S, D), (S * 12 * D, D, 6 * D, 1), 8 * D)  # tokens at another pitch
    assert attention(Slice(dev, whole, 0, 4), Slice(dev, whole, 4, 2), Slice(dev, whole, 6, 2), 4, 0, 1.0, other) == E


def test_gradients_that_share_an_element_are_refused():
    B, S, D = 1, 6, 16
    dev, whole = buffer(np.zeros((B, S, 20, D))), (B, S, 20, D)
    q, k, v, up, out = (Slice(dev, whole, f, n) for f, n in ((0, 4), (4, 2), (6, 2), (8, 4), (12, 4)))
    lse = DeviceArray(4 * 4 * S)
    check(attention(q, k, v, 4, 0, 1.0, out, lse))
    apart = [Placed(shape=(B, n, S, D)) for n in (4, 2, 2)]
    assert attention_grad(q, k, v, 4, 0, 1.0, out, lse, up, *apart) == 0
    for i, (first, n) in enumerate(((15, 4), (16, 2), (17, 2))):
        grads = list(apart)
        grads[i] = Slice(dev, whole, first, n)
        expected = abi.TRS_E_INVALID_ARGUMENT if first < 16 else 0
        assert attention_grad(q, k, v, 4, 0, 1.0, out, lse, up, *grads) == expected
    two = [apart[0], Slice(dev, whole, 16, 2), Slice(dev, whole, 17, 2)]  # dk's last head is dv's first
    assert attention_grad(q, k, v, 4, 0, 1.0, out, lse, up, *two) == abi.TRS_E_INVALID_ARGUMENT

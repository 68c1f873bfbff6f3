"""Gradients of sequences of their own lengths: heads of every width, rows and sinks in
parts, and calls without elements through autograd."""
import numpy as np
import pytest

import torch_rs
from attention_util import EVERY, Placed, assert_within, attention, attention_grad, attention_reference, ints
from trs_backend.abi import DeviceArray, check

pytestmark = pytest.mark.gpu

#        B  H hk  sq   sk    D  window sinks lengths
SHAPES = [
    (3, 4, 2, 90, 90, 160, 20, 3, [90, 1, 40]),
    (4, 2, 1, 40, 130, 200, EVERY, 0, [130, 0, 39, 33]),
    (2, 2, 2, 300, 300, 256, 17, 20, [300, 171]),
    (2, 3, 1, 70, 70, 129, 30, 5, [64, 70]),
    (2, 2, 1, 900, 900, 64, 300, 4, [900, 333]),      # the rows of a key tile in parts
    (3, 1, 1, 1500, 1500, 32, 40, 70, [1500, 2, 801]),  # and the sinks'
    (2, 4, 1, 700, 700, 96, 16, 130, [700, 129]),       # sinks of two blocks
    (2, 1, 1, 1200, 1200, 128, EVERY, 0, [1, 1200]),
    (2, 1, 1, 900, 900, 192, 24, 40, [900, 450]),
    (2, 2, 1, 333, 333, 50, 64, 2, [333, 20]),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_of_sequences_of_their_own_lengths(shape):
    B, H, hk, sq, sk, D, window, sinks, lengths = shape
    rng = np.random.default_rng(sum(shape[:6]))
    q, k, v, up = (rng.standard_normal(s).astype(np.float32) for s in ((B, H, sq, D), (B, hk, sk, D), (B, hk, sk, D), (B, H, sq, D)))
    want = attention_reference(q, k, v, window, sinks, np.float32(0.2), lengths, up)
    for b, n in enumerate(lengths):  # what no query sees is not read
        k[b, :, n:] = v[b, :, n:] = np.nan
    P, lens = [Placed(t) for t in (q, k, v)], ints(lengths)
    out, lse = Placed(shape=q.shape), DeviceArray(4 * B * H * sq)
    check(attention(*P, window, sinks, 0.2, out, lse, lens))
    assert_within(out.numpy(), *want["out"], "out")
    grads = [Placed(shape=t.shape) for t in (q, k, v)]
    check(attention_grad(*P, window, sinks, 0.2, out, lse, Placed(up), *grads, lens))
    for name, g in zip(("dq", "dk", "dv"), grads):
        assert_within(g.numpy(), *want[name], name)
        assert g.untouched()


@pytest.mark.parametrize("shape", [(0, 2, 3, 16), (2, 2, 0, 16)], ids=str)
def test_calls_without_elements_have_gradients(shape):
    F = torch_rs.nn.functional
    q, k, v = (torch_rs.zeros(shape, device="cuda", requires_grad=True) for _ in range(3))
    w = torch_rs.ones(16, device="cuda", requires_grad=True)
    table = torch_rs.ones((4, 8), device="cuda")
    nq, nk = F.head_norm_rope(q, k, w, None, table, table)
    F.dropout(F.window_attention(nq, nk, v, window=2), 0.5, seed=1).sum().backward()
    for t in (q, k, v):
        assert t.grad.shape == shape
    assert not w.grad.numpy().any()

"""The attention block's operators through torch_rs: autograd, the example's block
against 64 bits, and serving against the prompt."""
import importlib.util
from pathlib import Path

import numpy as np
import pytest

import torch_rs
from attention_util import EVERY, attention_reference, assert_within, dropout_reference, norm_rope_reference
from helpers import assert_bitwise_equal

pytestmark = pytest.mark.gpu
F = torch_rs.nn.functional


def example():
    spec = importlib.util.spec_from_file_location("attention_block", Path(__file__).resolve().parent.parent / "examples" / "attention_block.py")
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    return mod


def leaf(a, grad=True):
    return torch_rs.tensor(np.asarray(a, np.float32), device="cuda", requires_grad=grad)


def test_dropout_by_seed_and_its_gradient():
    x = np.random.default_rng(0).standard_normal((6, 10, 8)).astype(np.float32)
    up = np.random.default_rng(1).standard_normal((10, 6, 8)).astype(np.float32)
    X = leaf(x)
    y = F.dropout(X.permute(1, 0, 2), 0.3, seed=5, offset=9)
    assert y._grad_fn_name == "DropoutBackward0"
    assert_bitwise_equal(y.numpy(), dropout_reference(x.transpose(1, 0, 2), 0.3, 5, 9))
    (y * leaf(up, False)).sum().backward()
    assert_bitwise_equal(X.grad.numpy(), dropout_reference(up, 0.3, 5, 9).transpose(1, 0, 2))
    assert F.dropout(X, 0.3, False, seed=5) is X and F.dropout(X, 0.0, seed=5) is X
    assert not F.dropout(X, 1.0, seed=5).numpy().any()
    with pytest.raises(RuntimeError, match="through the graph a second time|freed|Trying"):
        s = F.window_attention(leaf(np.ones((1, 1, 2, 4))), leaf(np.ones((1, 1, 2, 4))), leaf(np.ones((1, 1, 2, 4)))).sum()
        s.backward()
        s.backward()


def test_head_norm_rope_and_window_attention_through_autograd():
    rng = np.random.default_rng(2)
    B, S, H, HK, D = 2, 37, 4, 2, 32
    q, k, v = (rng.standard_normal((B, S, n, D)).astype(np.float32) for n in (H, HK, HK))
    wq, wk = ((1 + 0.1 * rng.standard_normal(D)).astype(np.float32) for _ in range(2))
    up = rng.standard_normal((B, H, S, D)).astype(np.float32)
    angle = np.outer(np.arange(50), 0.5 ** np.arange(D // 2))
    cos, sin = np.cos(angle).astype(np.float32), np.sin(angle).astype(np.float32)
    Q, K, V, WQ, WK = (leaf(t) for t in (q, k, v, wq, wk))
    positions = np.arange(S)[None] + np.array([[3], [7]])
    nq, nk = F.head_norm_rope(Q.permute(0, 2, 1, 3), K.permute(0, 2, 1, 3), WQ, WK, leaf(cos, False), leaf(sin, False), positions=positions)
    out = F.window_attention(nq, nk, V.permute(0, 2, 1, 3), window=11, sinks=2)
    assert out._grad_fn_name == "WindowAttentionBackward0" and nq._grad_fn_name == "HeadNormRopeBackward0"
    assert out.shape == (B, H, S, D) and out.permute(0, 2, 1, 3).is_contiguous()
    (out * leaf(up, False)).sum().backward()
    # The definition in 64 bits; fp32 in between costs a few parts in 1e6 of the largest entry.
    tq, tk = q.transpose(0, 2, 1, 3), k.transpose(0, 2, 1, 3)
    rq, rk = (norm_rope_reference(t, w, 1e-6, cos, sin, positions, False) for t, w in ((tq, wq), (tk, wk)))
    want = attention_reference(rq, rk, v.transpose(0, 2, 1, 3), 11, 2, 1 / np.sqrt(D), up=up)
    dq, dwq = norm_rope_reference(tq, wq, 1e-6, cos, sin, positions, False, want["dq"][0])
    dk, dwk = norm_rope_reference(tk, wk, 1e-6, cos, sin, positions, False, want["dk"][0])
    for got, exact in ((out.numpy(), want["out"][0]), (Q.grad.numpy(), dq.transpose(0, 2, 1, 3)), (K.grad.numpy(), dk.transpose(0, 2, 1, 3)),
                       (V.grad.numpy(), want["dv"][0].transpose(0, 2, 1, 3)), (WQ.grad.numpy(), dwq), (WK.grad.numpy(), dwk)):
        assert abs(got - exact).max() <= 2e-5 * abs(exact).max()


def test_gradients_of_one_operand_alone():
    rng = np.random.default_rng(3)
    q, k, v, up = (rng.standard_normal((1, 2, 20, 16)).astype(np.float32) for _ in range(4))
    want = attention_reference(q, k, v, EVERY, 0, 0.25, up=up)
    for at, name in enumerate(("dq", "dk", "dv")):
        leaves = [leaf(t, i == at) for i, t in enumerate((q, k, v))]
        (F.window_attention(*leaves) * leaf(up, False)).sum().backward()
        assert_within(leaves[at].grad.numpy(), *want[name])
        assert all(t.grad is None for i, t in enumerate(leaves) if i != at)
    assert F.window_attention(*(leaf(t, False) for t in (q, k, v))).requires_grad is False


def test_key_lengths_of_a_cache():
    rng = np.random.default_rng(4)
    q, k, v = (rng.standard_normal(s).astype(np.float32) for s in ((3, 4, 1, 64), (3, 2, 90, 64), (3, 2, 90, 64)))
    for lengths in ([90, 1, 40], F.index_buffer([90, 1, 40])):
        got = F.window_attention(leaf(q, False), leaf(k, False), leaf(v, False), window=16, sinks=1, key_lengths=lengths)
        assert_within(got.numpy(), *attention_reference(q, k, v, 16, 1, np.float32(1 / 8), [90, 1, 40])["out"])


def test_the_example_trains_and_serves():
    mod = example()
    block = mod.AttentionBlock(width=64, heads=4, kv_heads=2, dim=32, window=20, sinks=2, positions=100)
    x = np.random.default_rng(5).standard_normal((2 * 70, 64)).astype(np.float32)
    X = leaf(x)
    y = block(X, 2, p=0.25, seed=3, offset=11)
    y.sum().backward()
    # The forward pass in 64 bits.
    W = [w.numpy().astype(np.float64) for w in block.parameters()]
    cos, sin = block.cos.numpy(), block.sin.numpy()

    def heads(t, n):
        return t.reshape(2, 70, n, 32).transpose(0, 2, 1, 3)

    q, k, v = (heads(x.astype(np.float64) @ w, n) for w, n in zip(W[:3], (4, 2, 2)))
    at = np.broadcast_to(np.arange(70), (2, 70))
    q, k = norm_rope_reference(q, W[4], 1e-6, cos, sin, at, False), norm_rope_reference(k, W[5], 1e-6, cos, sin, at, False)
    o = attention_reference(q, k, v, 20, 2, 1 / np.sqrt(32))["out"][0].transpose(0, 2, 1, 3).reshape(140, 128) @ W[3]
    kept = dropout_reference(np.ones(o.shape, np.float32), 0.25, 3, 11)
    assert abs(y.numpy() - (x + o * kept)).max() <= 2e-5 * abs(o).max()
    for p in [X] + block.parameters():
        assert np.isfinite(p.grad.numpy()).all() and p.grad.numpy().any()
    with torch_rs.no_grad():
        whole = block(X, 2).numpy().reshape(2, 70, 64)
        _, keys, values = block.project(X, 2)
        last = block.token(leaf(x.reshape(2, 70, 64)[:, -1], False), keys, values, 69).numpy()
    assert abs(last - whole[:, -1]).max() <= 2e-5 * abs(whole).max()

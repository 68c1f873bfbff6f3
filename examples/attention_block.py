"""One attention block in torch_rs, trained a step and then asked for a token.

    python examples/attention_block.py [--tokens 1024] [--window 256] [--steps 3]

x [batch * tokens, width] -> queries, keys and values (one product each) -> the
norm of every head with the rotation by position -> attention over a sliding
window and the first tokens -> the output product -> dropout -> + x.  The step's
dropout masks come from (seed, offset) alone.  Serving computes the last token
of a sequence against the keys and values of all of them.
"""
from __future__ import annotations

import argparse
import math
import sys
from pathlib import Path

import numpy as np

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "pytorch-rs_amd"))

import torch_rs  # noqa: E402

F = torch_rs.nn.functional


class AttentionBlock:
    def __init__(self, width=512, heads=8, kv_heads=2, dim=64, window=256, sinks=4, positions=4096, seed=0):
        rng = np.random.default_rng(seed)
        self.heads, self.kv_heads, self.dim, self.window, self.sinks = heads, kv_heads, dim, window, sinks

        def weight(rows, cols):
            return torch_rs.tensor(rng.uniform(-1, 1, (rows, cols)).astype(np.float32) / math.sqrt(rows), device="cuda", requires_grad=True)

        self.wq, self.wk, self.wv = weight(width, heads * dim), weight(width, kv_heads * dim), weight(width, kv_heads * dim)
        self.wo = weight(heads * dim, width)
        self.nq, self.nk = (torch_rs.ones(dim, device="cuda", requires_grad=True) for _ in range(2))
        angle = np.outer(np.arange(positions), 10000.0 ** (-np.arange(dim // 2) / (dim // 2)))
        self.cos, self.sin = (torch_rs.tensor(f(angle).astype(np.float32), device="cuda") for f in (np.cos, np.sin))

    def parameters(self):
        return [self.wq, self.wk, self.wv, self.wo, self.nq, self.nk]

    def _heads(self, t, batch, heads):
        """[batch * tokens, heads * dim] as [batch, heads, tokens, dim], in place."""
        return t.reshape(batch, t.shape[0] // batch, heads, self.dim).permute(0, 2, 1, 3)

    def project(self, x, batch, start=0):
        """Rotated queries and keys, and values, of x [batch * tokens, width]."""
        q, k, v = (self._heads(x @ w, batch, n) for w, n in ((self.wq, self.heads), (self.wk, self.kv_heads), (self.wv, self.kv_heads)))
        q, k = F.head_norm_rope(q, k, self.nq, self.nk, self.cos, self.sin, start=start)
        return q, k, v

    def join(self, out, batch):
        """[batch, heads, tokens, dim] through the output product."""
        return out.permute(0, 2, 1, 3).reshape(batch * out.shape[2], self.heads * self.dim) @ self.wo

    def __call__(self, x, batch, p=0.0, seed=0, offset=0):
        q, k, v = self.project(x, batch)
        out = self.join(F.window_attention(q, k, v, window=self.window, sinks=self.sinks), batch)
        return x + F.dropout(out, p, p > 0, seed=seed, offset=offset)

    def token(self, x, keys, values, start, key_lengths=None):
        """One token a sequence, x [batch, width], over the rotated keys and the values that it sees, its own
        among them; `start` is its place."""
        batch = x.shape[0]
        q = self._heads(x @ self.wq, batch, self.heads)
        q = F.head_norm_rope(q, None, self.nq, None, self.cos, self.sin, start=start)
        return x + self.join(F.window_attention(q, keys, values, window=self.window, sinks=self.sinks, key_lengths=key_lengths), batch)


def main() -> int:
    ap = argparse.ArgumentParser(description=__doc__.split("\n\n")[0])
    ap.add_argument("--tokens", type=int, default=1024)
    ap.add_argument("--window", type=int, default=256)
    ap.add_argument("--steps", type=int, default=3)
    a = ap.parse_args()
    block = AttentionBlock(window=a.window, positions=a.tokens)
    rng = np.random.default_rng(1)
    x = rng.standard_normal((a.tokens, 512)).astype(np.float32)
    target = torch_rs.tensor(rng.standard_normal((a.tokens, 512)).astype(np.float32), device="cuda")
    X = torch_rs.tensor(x, device="cuda")
    for step in range(a.steps):
        diff = block(X, 1, p=0.1, seed=7, offset=step * (a.tokens * 512 // 4)) - target
        loss = (diff * diff).sum() * (1 / (a.tokens * 512))
        loss.backward()
        print(f"step {step}: loss {loss.item():.6f}")
        with torch_rs.no_grad():
            moved = [(w - w.grad * 0.5).detach().with_requires_grad(True) for w in block.parameters()]
        block.wq, block.wk, block.wv, block.wo, block.nq, block.nk = moved
    with torch_rs.no_grad():
        whole = block(X, 1).numpy()
        _, keys, values = block.project(X, 1)
        last = block.token(torch_rs.tensor(x[-1:], device="cuda"), keys, values, a.tokens - 1).numpy()
    print(f"last token alone against the whole prompt: {abs(last[0] - whole[-1]).max():.2e} apart")
    return 0


if __name__ == "__main__":
    sys.exit(main())

"""A transformer block's attention trained for a few steps, then run token by token.

    python examples/transformer_step.py [--steps 20] [--state-bits 8]

Training: products -> rotary positions (stored as bfloat16) -> causal attention
with shared key heads -> product -> mean square error, its gradients through all
of them, and an AdamW step over the four weights. Then the same weights answer
one token at a time: each token's query is turned by its own position and attends
the keys up to it, which gives the rows that the whole sequence gives.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ormi_amd import AdamW, RotaryTable, Tensor, attention, rotary  # noqa: E402


class AttentionBlock:
    """y = attention(rotary(x Wq), rotary(x Wk), x Wv) Wo, with kv_heads <= heads."""

    def __init__(self, width: int, heads: int, kv_heads: int, positions: int, rng, dtype: str = "bfloat16"):
        self.heads, self.kv_heads, self.features, self.dtype = heads, kv_heads, width // heads, dtype
        self.table = RotaryTable(self.features, positions)

        def weight(rows, cols):
            return Tensor((rng.standard_normal((rows, cols)) / np.sqrt(rows)).astype(np.float32), "hip", requires_grad=True)

        self.wq, self.wo = weight(width, width), weight(width, width)
        self.wk, self.wv = weight(width, kv_heads * self.features), weight(width, kv_heads * self.features)

    def parameters(self):
        return [self.wq, self.wk, self.wv, self.wo]

    def _heads(self, x: Tensor, w: Tensor, heads: int) -> Tensor:
        batch, length, width = x.shape
        return (x.reshape((batch * length, width)) @ w).reshape((batch, length, heads, self.features))

    def queries(self, x: Tensor, offset: int = 0) -> Tensor:
        return rotary(self._heads(x, self.wq, self.heads), self.table, offset=offset, dtype=self.dtype)

    def keys_values(self, x: Tensor):
        return (rotary(self._heads(x, self.wk, self.kv_heads), self.table, dtype=self.dtype),
                self._heads(x, self.wv, self.kv_heads).astype(self.dtype))

    def attend(self, q: Tensor, k: Tensor, v: Tensor, lengths: Tensor | None = None) -> Tensor:
        batch, length = q.shape[:2]
        y = attention(q, k, v, causal=True, lengths=lengths).astype("float32")
        return (y.reshape((batch * length, self.heads * self.features)) @ self.wo).reshape((batch, length, self.heads * self.features))

    def __call__(self, x: Tensor) -> Tensor:
        return self.attend(self.queries(x), *self.keys_values(x))


def train(block: AttentionBlock, x: np.ndarray, target: np.ndarray, steps: int, lr: float, state_bits: int = 32) -> list[float]:
    """The loss before each step."""
    optimizer = AdamW(block.parameters(), lr=lr, weight_decay=0.01, state_bits=state_bits)
    losses = []
    for _ in range(steps):
        error = block(Tensor(x, "hip")) - Tensor(target, "hip")
        loss = (error * error).mean()
        loss.backward()
        optimizer.step()
        losses.append(float(loss.numpy()))
        loss.zero_grad_graph()  # gradients point back at the nodes they came from: without it each step's graph stays
    return losses


def token_by_token(block: AttentionBlock, x: np.ndarray) -> np.ndarray:
    """The block's rows, one query at a time over the tokens' keys and values.

    Tensors are not written after they are made and the graph has no op that extends
    one, so all keys and values are made first; lengths hides those after the token.
    """
    batch, length, _ = x.shape
    k, v = block.keys_values(Tensor(x, "hip"))
    k.realize(), v.realize()
    rows = []
    for at in range(length):
        lengths = Tensor(np.full(batch, at + 1, np.int32), "hip", dtype="int32")  # what stands after the token does not count
        rows.append(block.attend(block.queries(Tensor(x[:, at:at + 1].copy(), "hip"), offset=at), k, v, lengths).numpy())
    return np.concatenate(rows, axis=1)


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    args.add_argument("--steps", type=int, default=20)
    args.add_argument("--state-bits", type=int, default=32, choices=(32, 8))
    args = args.parse_args()

    rng = np.random.default_rng(0)
    batch, length, width = 4, 256, 512
    x = rng.standard_normal((batch, length, width)).astype(np.float32)
    # What is learned: each token's answer is a turned copy of the token before it.
    turn = np.linalg.qr(rng.standard_normal((width, width)))[0].astype(np.float32)
    target = np.concatenate([np.zeros_like(x[:, :1]), x[:, :-1] @ turn], axis=1)

    block = AttentionBlock(width, heads=8, kv_heads=2, positions=length, rng=rng)
    losses = train(block, x, target, args.steps, lr=2e-3, state_bits=args.state_bits)
    print("loss", " ".join(f"{v:.4f}" for v in losses))
    whole, single = block(Tensor(x, "hip")).numpy(), token_by_token(block, x)
    print(f"token by token against the whole sequence: largest difference {np.abs(whole - single).max():.2e}"
          f" of values up to {np.abs(whole).max():.2f}")


if __name__ == "__main__":
    main()

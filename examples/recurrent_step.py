"""A recurrent block trained for a few steps on packed documents, then run token by token.

    python examples/recurrent_step.py [--steps 20] [--max-norm 1.0]

Training: product -> short causal convolution with silu -> gated linear recurrence
(its logits a product of the convolution's result) -> times a gate -> product -> mean
square error, its gradients through all of them, and an AdamW step with the gradients'
norm bounded. Then the same weights answer one token at a time, the convolution's
inputs and the recurrence's state carried from call to call.
"""
from __future__ import annotations

import argparse
import os
import sys

import numpy as np

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from ormi_amd import AdamW, Tensor, causal_conv, linear_recurrence  # noqa: E402


class RecurrentBlock:
    """y = (recurrence(u Wa, u) * gelu(x Wz)) Wo with u = silu(conv(x Wu)); (batch, length, width) in float32."""

    def __init__(self, width: int, inner: int, taps: int, rng, dtype: str = "bfloat16"):
        self.width, self.inner, self.dtype = width, inner, dtype

        def learned(values):
            return Tensor(values.astype(np.float32), "hip", requires_grad=True)

        def weight(rows, cols):
            return learned(rng.standard_normal((rows, cols)) / np.sqrt(rows))

        self.wu, self.wz, self.wa, self.wo = weight(width, inner), weight(width, inner), weight(inner, inner), weight(inner, width)
        self.taps, self.bias = learned(rng.standard_normal((inner, taps)) / np.sqrt(taps)), learned(np.zeros(inner))
        self.forget = learned(np.full(inner, 2.0))  # added to the logits: states that last for some tokens at the start

    def parameters(self):
        return [self.wu, self.wz, self.wa, self.wo, self.taps, self.bias, self.forget]

    def __call__(self, x: Tensor, state=(None, None), documents: Tensor | None = None):
        """(y, the state after the last token)."""
        batch, length, _ = x.shape
        inner = (batch, length, self.inner)
        flat = x.reshape((batch * length, self.width))
        u, inputs = causal_conv((flat @ self.wu).reshape(inner).astype(self.dtype), self.taps, self.bias, state[0], activation="silu", documents=documents)
        logits = (u.astype("float32").reshape((batch * length, self.inner)) @ self.wa + self.forget).reshape(inner)
        h, memory = linear_recurrence(logits, u, state[1], gate="logit", documents=documents)
        gated = h.astype("float32").reshape((batch * length, self.inner)) * (flat @ self.wz).gelu()
        return (gated @ self.wo).reshape((batch, length, self.width)), (inputs, memory)


def train(block: RecurrentBlock, x: np.ndarray, target: np.ndarray, documents: np.ndarray, steps: int, lr: float, max_norm: float) -> list[tuple]:
    """The loss before each step, and the norm of its gradients."""
    optimizer = AdamW(block.parameters(), lr=lr, weight_decay=0.01, max_norm=max_norm)
    history = []
    for _ in range(steps):
        y, _ = block(Tensor(x, "hip"), documents=Tensor(documents, "hip", dtype="int32"))
        error = y - Tensor(target, "hip")
        loss = (error * error).mean()
        loss.backward()
        optimizer.step()
        history.append((float(loss.numpy()), float(optimizer.norm.numpy())))
        loss.zero_grad_graph()  # gradients point back at the nodes they came from: without it each step's graph stays
    return history


def token_by_token(block: RecurrentBlock, x: np.ndarray) -> np.ndarray:
    """The block's rows, one token at a time."""
    state, rows = (None, None), []
    for at in range(x.shape[1]):
        y, state = block(Tensor(x[:, at:at + 1].copy(), "hip"), state)
        rows.append(y.numpy())
        state = tuple(t.detach() for t in state)  # the weights have gradients: a state as it is keeps every token's graph
    return np.concatenate(rows, axis=1)


def main() -> None:
    args = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    args.add_argument("--steps", type=int, default=20)
    args.add_argument("--max-norm", type=float, default=1.0)
    args = args.parse_args()

    rng = np.random.default_rng(0)
    batch, length, width = 4, 256, 256
    x = rng.standard_normal((batch, length, width)).astype(np.float32)
    documents = np.sort(rng.integers(0, 4, (batch, length))).astype(np.int32)
    # What is learned: each token's answer is a turned copy of the token before it in its document.
    turn = np.linalg.qr(rng.standard_normal((width, width)))[0].astype(np.float32)
    same = np.concatenate([np.zeros((batch, 1), bool), documents[:, 1:] == documents[:, :-1]], axis=1)
    target = np.concatenate([np.zeros_like(x[:, :1]), x[:, :-1] @ turn], axis=1) * same[..., None]

    block = RecurrentBlock(width, 2 * width, 4, rng)
    for loss, norm in train(block, x, target.astype(np.float32), documents, args.steps, 2e-3, args.max_norm):
        print(f"loss {loss:.4f}  gradient norm {norm:.3f}")
    whole, single = block(Tensor(x, "hip"))[0].numpy(), token_by_token(block, x)
    print(f"token by token against the whole sequence: largest difference {np.abs(whole - single).max():.2e}"
          f" of values up to {np.abs(whole).max():.2f}")


if __name__ == "__main__":
    main()

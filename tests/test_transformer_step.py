"""The operators together, as examples/transformer_step.py uses them: rotary
positions, attention with shared key heads and AdamW around plain products.

Tolerance: the block is about ten float32 products and sums in a row, each over at
most n = 96 terms (width, features, keys, batch times length); one of them is off
by at most n u of |A| |B|, which is at most sqrt(n) times its result for operands
without a common direction. 10 * 96 * 10 * 2^-24 = 6e-4 of a gradient's norm.
"""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

WIDTH, HEADS, KV_HEADS, BATCH, LENGTH = 64, 4, 2, 3, 32
BOUND = 10 * 96 * 10 * 2.0 ** -24


def _block(dtype):
    import transformer_step as example

    rng = np.random.default_rng(5)
    block = example.AttentionBlock(WIDTH, HEADS, KV_HEADS, LENGTH, rng, dtype=dtype)
    x = rng.standard_normal((BATCH, LENGTH, WIDTH)).astype(np.float32)
    target = rng.standard_normal((BATCH, LENGTH, WIDTH)).astype(np.float32)
    return example, block, x, target


def _plain(weights, x, target):
    """Loss, output and the weights' gradients in 64 bits, by the formulas."""
    wq, wk, wv, wo = weights
    d = WIDTH // HEADS
    half = d // 2
    angle = np.arange(LENGTH)[:, None] * 10000.0 ** (-2.0 * np.arange(half) / d)
    c, s = np.cos(angle)[None, :, None], np.sin(angle)[None, :, None]

    def turn(y, s):
        a, z = y[..., :half], y[..., half:]
        return np.concatenate([a * c - z * s, z * c + a * s], -1)

    q = turn((x @ wq).reshape(BATCH, LENGTH, HEADS, d), s)
    k = turn((x @ wk).reshape(BATCH, LENGTH, KV_HEADS, d), s)
    v = (x @ wv).reshape(BATCH, LENGTH, KV_HEADS, d)
    group = HEADS // KV_HEADS
    kh, vh = np.repeat(k, group, 2), np.repeat(v, group, 2)
    t = np.einsum("bihd,bjhd->bhij", q, kh) / np.sqrt(d)
    t = np.where(np.tril(np.ones((LENGTH, LENGTH), bool)), t, -np.inf)
    p = np.exp(t - t.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    o = np.einsum("bhij,bjhd->bihd", p, vh).reshape(BATCH, LENGTH, WIDTH)
    y = o @ wo
    error = y - target
    dy = 2 * error / error.size
    do = (dy @ wo.T).reshape(BATCH, LENGTH, HEADS, d)
    dp = np.einsum("bihd,bjhd->bhij", do, vh)
    dt = p * (dp - (p * dp).sum(-1, keepdims=True)) / np.sqrt(d)
    dq = turn(np.einsum("bhij,bjhd->bihd", dt, kh), -s)
    dk = turn(np.einsum("bhij,bihd->bjhd", dt, q).reshape(BATCH, LENGTH, KV_HEADS, group, d).sum(3), -s)
    dv = np.einsum("bhij,bihd->bjhd", p, do).reshape(BATCH, LENGTH, KV_HEADS, group, d).sum(3)
    grads = [np.einsum("blw,blc->wc", a, g.reshape(BATCH, LENGTH, -1)) for a, g in ((x, dq), (x, dk), (x, dv), (o, dy))]
    return (error * error).mean(), y, grads


def test_plain_gradients_against_differences():
    rng = np.random.default_rng(2)
    weights = [rng.standard_normal((WIDTH, c)) / 8 for c in (WIDTH, WIDTH // 2, WIDTH // 2, WIDTH)]
    x, target = rng.standard_normal((2, BATCH, LENGTH, WIDTH))
    grads = _plain(weights, x, target)[2]
    for i, g in enumerate(grads):
        step = rng.standard_normal(g.shape)
        h = 1e-5  # the difference's error: h^2 of the third derivative and 1e-16 / h of the loss
        up, down = ([w + e * h * step if j == i else w for j, w in enumerate(weights)] for e in (1, -1))
        slope = (_plain(up, x, target)[0] - _plain(down, x, target)[0]) / (2 * h)
        assert abs(slope - (g * step).sum()) <= 1e-7 * (1 + np.linalg.norm(step))


@pytest.mark.gpu
def test_gradients_of_the_block():
    from ormi_amd import Tensor

    _, block, x, target = _block("float32")
    error = block(Tensor(x, "hip")) - Tensor(target, "hip")
    loss = (error * error).mean()
    loss.backward()
    exact, _, grads = _plain([w.numpy().astype(np.float64) for w in block.parameters()], x.astype(np.float64), target.astype(np.float64))
    assert abs(float(loss.numpy()) - exact) <= BOUND * exact
    for w, g in zip(block.parameters(), grads):
        got = w.grad.numpy().astype(np.float64)
        assert np.linalg.norm(got - g) <= BOUND * np.linalg.norm(g)


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_training_lowers_the_loss(dtype, bits):
    example, block, x, target = _block(dtype)
    losses = example.train(block, x, target, steps=12, lr=3e-3, state_bits=bits)
    assert all(np.isfinite(losses)) and losses[-1] < losses[0]


@pytest.mark.gpu
def test_token_by_token_gives_the_whole_sequence():
    from ormi_amd import Tensor

    example, block, x, _ = _block("float32")
    whole, single = block(Tensor(x, "hip")).numpy(), example.token_by_token(block, x)
    assert np.linalg.norm(whole - single) <= 2 * BOUND * np.linalg.norm(whole)

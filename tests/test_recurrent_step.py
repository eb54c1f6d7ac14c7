"""The recurrent operators together, as examples/recurrent_step.py uses them: the
convolution, the recurrence and clipped AdamW around plain products.

Tolerance: the block is about ten float32 products and sums in a row, each over at
most n = 96 terms (channels, batch times length, a state's memory of some tens of
tokens); one of them is off by at most n u of |A| |B|, which is at most sqrt(n) times
its result for operands without a common direction. 10 * 96 * 10 * 2^-24 = 6e-4 of a
gradient's norm.
"""
import os
import sys

import numpy as np
import pytest

import recurrent_ref as ref

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))

WIDTH, INNER, TAPS, BATCH, LENGTH = 48, 64, 4, 3, 32
BOUND = 10 * 96 * 10 * 2.0 ** -24


def _block(dtype):
    import recurrent_step as example

    rng = np.random.default_rng(5)
    block = example.RecurrentBlock(WIDTH, INNER, TAPS, rng, dtype=dtype)
    x, target = rng.standard_normal((2, BATCH, LENGTH, WIDTH)).astype(np.float32)
    documents = np.sort(rng.integers(0, 3, (BATCH, LENGTH))).astype(np.int32)
    documents[0, -2:] = -1
    return example, block, x, target, documents


def _plain(weights, x, target, documents):
    """Loss, output and the weights' gradients in 64 bits, by the formulas."""
    from math import erf

    wu, wz, wa, wo, taps, bias, forget = weights
    cdf = lambda t: 0.5 * (1 + np.vectorize(erf)(t / np.sqrt(2)))  # noqa: E731
    p = x @ wu
    u = ref.conv(p, taps, bias, True, None, documents)[0]["y"]
    a = u @ wa + forget
    h = ref.recurrence(a, u, True, None, documents)[0]["y"]
    z = x @ wz
    gate = z * cdf(z)
    y = (h * gate) @ wo
    error = y - target
    dy = 2 * error / error.size
    dm = dy @ wo.T
    back = ref.recurrence(a, u, True, None, documents, dy=dm * gate)[0]
    du = back["dx"] + back["dg"] @ wa.T
    conv = ref.conv(p, taps, bias, True, None, documents, dy=du)[0]
    dz = dm * h * (cdf(z) + z * np.exp(-0.5 * z * z) / np.sqrt(2 * np.pi))
    outer = lambda a, g: np.einsum("blw,blc->wc", a, g)  # noqa: E731
    return (error * error).mean(), y, [outer(x, conv["dx"]), outer(x, dz), outer(u, back["dg"]), outer(h * gate, dy), conv["dw"], conv["db"],
                                       back["dg"].sum((0, 1))]


def _weights(block):
    return [w.numpy().astype(np.float64) for w in block.parameters()]


def test_plain_gradients_against_differences():
    rng = np.random.default_rng(2)
    weights = [rng.standard_normal(s) / 7 for s in ((WIDTH, INNER), (WIDTH, INNER), (INNER, INNER), (INNER, WIDTH), (INNER, TAPS), (INNER,), (INNER,))]
    x, target = rng.standard_normal((2, BATCH, LENGTH, WIDTH))
    documents = np.sort(rng.integers(0, 3, (BATCH, LENGTH)))
    grads = _plain(weights, x, target, documents)[2]
    for i, g in enumerate(grads):
        step = rng.standard_normal(g.shape)
        h = 1e-5  # the difference's error: h^2 of the third derivative and 1e-16 / h of the loss
        up, down = ([w + e * h * step if j == i else w for j, w in enumerate(weights)] for e in (1, -1))
        slope = (_plain(up, x, target, documents)[0] - _plain(down, x, target, documents)[0]) / (2 * h)
        assert abs(slope - (g * step).sum()) <= 1e-7 * (1 + np.linalg.norm(step))


@pytest.mark.gpu
def test_gradients_of_the_block(hip):
    from ormi_amd import Tensor, grad_norm

    _, block, x, target, documents = _block("float32")
    y, _ = block(Tensor(x, "hip"), documents=Tensor(documents, "hip", dtype="int32"))
    error = y - Tensor(target, "hip")
    loss = (error * error).mean()
    loss.backward()
    exact, _, grads = _plain(_weights(block), x.astype(np.float64), target.astype(np.float64), documents)
    norm = float(grad_norm([w.grad for w in block.parameters()]).numpy())
    assert abs(float(loss.numpy()) - exact) <= BOUND * exact
    for w, g in zip(block.parameters(), grads):
        got = w.grad.numpy().astype(np.float64)
        assert np.linalg.norm(got - g) <= BOUND * np.linalg.norm(g)
    assert abs(norm - np.sqrt(sum((g * g).sum() for g in grads))) <= BOUND * norm


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_training_runs(hip, dtype):
    """The first step's norm is that of the formula's gradients, within what the 16-bit sequences leave of them."""
    example, block, x, target, documents = _block(dtype)
    _, _, grads = _plain(_weights(block), x.astype(np.float64), target.astype(np.float64), documents)
    history = example.train(block, x, target, documents, steps=6, lr=3e-3, max_norm=0.1)
    assert np.isfinite(history).all() and all(n > 0 for _, n in history)
    # three roundings to the type on the way to y and four more back, each at most half a spacing of every term, of
    # which a state and its gradient add up a document's: LENGTH of them at most, without a common direction
    slack = BOUND + (0 if dtype == "float32" else 7 * ref.HALF[dtype])
    want = np.sqrt(sum((g * g).sum() for g in grads))
    assert abs(history[0][1] - want) <= slack * want * np.sqrt(LENGTH)
    assert all(np.isfinite(w.numpy()).all() for w in block.parameters())


@pytest.mark.gpu
def test_token_by_token_gives_the_whole_sequence(hip):
    from ormi_amd import Tensor

    example, block, x, _, _ = _block("float32")
    whole, single = block(Tensor(x, "hip"))[0].numpy(), example.token_by_token(block, x)
    assert np.linalg.norm(whole - single) <= 2 * BOUND * np.linalg.norm(whole)


@pytest.mark.gpu
def test_a_loop_reaches_a_steady_state(hip, ob):
    example, block, x, target, documents = _block("bfloat16")
    ob.empty_cache()
    mallocs = []
    for steps in (5, 40):
        example.train(block, x, target, documents, steps=steps, lr=1e-3, max_norm=1.0)
        ob.synchronize()
        mallocs.append(ob.allocator_stats()["device_mallocs"])
    assert mallocs[1] == mallocs[0]

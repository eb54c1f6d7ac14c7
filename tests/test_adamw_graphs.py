"""A training loop as documented holds no more memory after a hundred steps than
after a few: the optimizer lets go of the old leaves' gradients, and the loop
releases each step's graph."""
import os
import sys

import numpy as np
import pytest

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples"))


def test_a_step_clears_the_old_leaves(cpu, monkeypatch):
    """On the CPU device, with the step itself replaced by a plain one."""
    from ormi_amd import AdamW, Tensor, transformer

    def plain(params, grads, states, **options):
        return [Tensor(p.numpy() - 0.1 * g.numpy(), p.device, requires_grad=True) for p, g in zip(params, grads)], states

    monkeypatch.setattr(transformer, "adamw", plain)
    a, b = (Tensor(np.full((3, 4), x, np.float32), cpu, requires_grad=True) for x in (1.0, 2.0))
    opt = AdamW([a, b])
    loss = (a * 3.0).sum()
    loss.backward()
    old_a, old_b, kept = a._node, b._node, a.grad
    opt.step()
    assert old_a.grad is None and a._node is not old_a and b._node is old_b
    assert np.array_equal(kept.numpy(), np.full((3, 4), 3.0, np.float32))  # a gradient that is held stays
    assert np.allclose(a.numpy(), 0.7) and a.grad is None


# The allocator counts a cached block that serves a smaller request whole, so the bytes
# in use vary by what is cached; with an empty cache at the start a loop that keeps
# its graphs has to ask the device for memory again and again.
@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_the_example_reaches_a_steady_state(hip, ob, dtype):
    import transformer_step as example

    rng = np.random.default_rng(5)
    block = example.AttentionBlock(64, 4, 2, 32, rng, dtype=dtype)
    x, target = rng.standard_normal((2, 3, 32, 64)).astype(np.float32)
    ob.empty_cache()
    mallocs = []
    for steps in (5, 60):
        example.train(block, x, target, steps=steps, lr=1e-3)
        ob.synchronize()
        mallocs.append(ob.allocator_stats()["device_mallocs"])
    assert mallocs[1] == mallocs[0]


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_a_loop_that_releases_its_graphs(hip, ob, bits):
    from ormi_amd import AdamW, Tensor

    rng = np.random.default_rng(1)
    w = Tensor(rng.standard_normal((128, 128)).astype(np.float32), "hip", requires_grad=True)
    x = Tensor(rng.standard_normal((64, 128)).astype(np.float32), "hip")
    opt = AdamW([w], state_bits=bits)
    ob.empty_cache()
    mallocs = []
    for _ in range(60):
        y = (x @ w).gelu()
        loss = (y * y).mean()
        loss.backward()
        opt.step()
        loss.zero_grad_graph()
        ob.synchronize()
        mallocs.append(ob.allocator_stats()["device_mallocs"])
    assert mallocs[-1] == mallocs[4], mallocs

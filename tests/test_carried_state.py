"""States passed from call to call: what they keep alive, and detach()."""
import numpy as np
import pytest

import recurrent_ref as ref


def test_detach_is_a_leaf_of_the_same_buffer(cpu):
    from ormi_amd import Tensor

    a = Tensor(np.arange(6, dtype=np.float32).reshape(2, 3), cpu, requires_grad=True)
    b = a * 2.0
    d = b.detach()
    assert d.op.name == "LEAF" and not d.requires_grad and d.device is b.device and d._node.parents == []
    assert d._node.data.ptr == b._node.data.ptr and d.dtype == "float32" and np.array_equal(d.numpy(), b.numpy())
    (b * d).sum().backward()
    assert np.array_equal(a.grad.numpy(), 2 * d.numpy()) and d.grad is None  # d counts as a constant
    for view in (a.T, a.reshape((3, 2)), Tensor(np.ones((1, 3), np.float32), cpu).expand((4, 3))):
        d = view.detach()
        assert d.shape == view.shape and np.array_equal(d.numpy(), view.numpy())
        assert np.array_equal((d + 1.0).numpy(), view.numpy() + 1)
    for kind in ("int32", "bfloat16"):
        t = Tensor(np.ones((2, 2), np.float32), cpu, dtype=kind).detach()
        assert t.dtype == kind and (t.numpy() == 1).all()


def _tensors(rng, *shapes, grad=False, dtype="float32"):
    from ormi_amd import Tensor

    return [Tensor(rng.standard_normal(s).astype(np.float32), "hip", requires_grad=grad, dtype=dtype) for s in shapes]


def _live(ob):
    ob.synchronize()
    return ob.allocator_stats()["live_bytes"]


@pytest.mark.gpu
@pytest.mark.parametrize("learned", [False, True])
@pytest.mark.parametrize("read", ["each result", "the last result"])
def test_a_token_loop_keeps_no_token(hip, ob, learned, read):
    """As the functions' documentation says: states pass on as they are, or detached where gradients go."""
    from ormi_amd import causal_conv, linear_recurrence

    ob.empty_cache()
    rng = np.random.default_rng(1)
    taps, gain = _tensors(rng, (2048, 4), (2048,), grad=learned)
    state, kept, live = None, None, []
    for at in range(60):
        x, = _tensors(rng, (4, 1, 2048), dtype="bfloat16")
        u, kept = causal_conv(x, taps, None, kept, activation="silu")
        y, state = linear_recurrence(u.astype("float32") * gain, u, state, gate="logit")
        if read == "each result" or at % 20 == 19:
            y.numpy()
            state.realize(), kept.realize()
        if learned:
            state, kept = state.detach(), kept.detach()
        del x, u, y
        if at % 20 == 19:
            live.append(_live(ob))
    assert live[0] == live[1] == live[2]


@pytest.mark.gpu
def test_a_state_keeps_nothing_of_its_call(hip, ob):
    from ormi_amd import causal_conv, linear_recurrence

    rng = np.random.default_rng(2)
    base = _live(ob)
    g, x = _tensors(rng, (2, 4096, 512), (2, 4096, 512))
    y, state = linear_recurrence(g, x, gate="logit")
    z, kept = causal_conv(x, *_tensors(rng, (512, 3)))
    want, rows = state.numpy().copy(), kept.numpy().copy()
    del g, x, y, z
    # the two states, 4096 and 8192 bytes: the pool hands out blocks of at most twice a request's power of two
    assert _live(ob) - base <= 2 * (4 * 2 * 512 + 4 * 2 * 2 * 512)
    assert np.array_equal(state.numpy(), want) and np.array_equal(kept.numpy(), rows)


@pytest.mark.gpu
def test_a_detached_state_ends_the_gradient(hip):
    """Training in chunks: the second chunk's gradients are the formula's with the first's state as a constant."""
    from ormi_amd import Tensor, linear_recurrence, realize_all

    rng = np.random.default_rng(3)
    shape = (2, 70, 12)
    first, second = ([(rng.standard_normal(shape) + 2).astype(np.float32), *rng.standard_normal((2, *shape)).astype(np.float32)] for _ in range(2))
    leaves = [[Tensor(t, "hip", requires_grad=True) for t in part[:2]] for part in (first, second)]
    _, state = linear_recurrence(*leaves[0], gate="logit")
    y, _ = linear_recurrence(*leaves[1], state.detach(), gate="logit")
    (y * Tensor(second[2], "hip")).sum().backward()
    assert all(t.grad is None for t in leaves[0]) and state.grad is None
    realize_all(y, *(t.grad for t in leaves[1]))
    h0 = state.numpy()
    want, bound = ref.recurrence(second[0], second[1], True, h0, dy=second[2])
    for name, t in (("y", y), ("dg", leaves[1][0].grad), ("dx", leaves[1][1].grad)):
        ref.close(t.numpy(), want[name], bound[name], "float32", name)

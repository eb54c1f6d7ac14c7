"""The norm over a list of gradients, clipping, and the clipped AdamW step on the GPU.

Squares add up in 64 bits, so the norm is the exact one rounded once (n 2^-53 of it
apart), and the factor another rounding: clipped float32 values are within three half
spacings of the exact ones, and bit for bit the float32 products with the factor.
"""
import ctypes

import numpy as np
import pytest

from test_adamw import BLOCK, CALL, HYPER, SHAPES, encode, inputs, step32

F = np.float32
U = 2.0 ** -24


def tensor(a, dtype="float32"):
    from ormi_amd import Tensor

    return Tensor(a, "hip", dtype=dtype)


def exact_norm(grads):
    return float(np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads)))


def factor_of(grads, max_norm):
    n = exact_norm(grads)
    return F(1.0 if n <= max_norm else max_norm / n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("count", [1, 12, 130, 400])
def test_norm_and_clipping(hip, dtype, count):
    from ormi_amd import clip_grads, grad_norm

    shapes = [SHAPES[i % len(SHAPES)] for i in range(count)] + [(0,), (100003,)]
    grads = [tensor(np.asarray(np.random.default_rng(i).standard_normal(s), F), dtype) for i, s in enumerate(shapes)]
    host = [g.numpy() for g in grads]
    n = exact_norm(host)
    got = grad_norm(grads)
    assert got.shape == () and got.dtype == "float32" and abs(float(got.numpy()) - n) <= 1.01 * U * n
    for max_norm in (0.0, 0.25, n * 0.5, n * 2, np.inf):
        clipped, norm = clip_grads(grads, max_norm)
        assert float(norm.numpy()) == float(got.numpy())
        f = factor_of(host, max_norm)
        for c, g, h in zip(clipped, grads, host):
            assert c.dtype == dtype and c.shape == g.shape and np.array_equal(g.numpy(), h)
            # the factor may differ from numpy's by the sums' last bits of 64, which show as one float32 spacing
            options = [tensor(h * q, dtype).numpy() for q in (f, np.nextafter(f, F(0)), np.nextafter(f, F(2)))]
            assert any(np.array_equal(c.numpy(), o) for o in options)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1e-38, 1e-25, 1e20, 1e38])
def test_squares_neither_vanish_nor_overflow(hip, scale):
    from ormi_amd import clip_grads, grad_norm

    g = (np.random.default_rng(1).uniform(0.5, 1, 5000) * scale / 50).astype(F)
    n = exact_norm([g])
    assert abs(float(grad_norm([tensor(g)]).numpy()) - n) <= 1.01 * U * n
    (c,), _ = clip_grads([tensor(g)], 1e-3 * n)
    assert np.allclose(c.numpy(), g.astype(np.float64) * 1e-3, rtol=3 * U, atol=2e-45)


@pytest.mark.gpu
def test_norm_past_float32(hip):
    """A norm of more than float32 holds is infinite, and still clips: its factor is taken before the rounding."""
    from ormi_amd import clip_grads

    g = np.full(100, 3e38, F)
    (c,), norm = clip_grads([tensor(g)], 1.0)
    assert np.isinf(norm.numpy()) and np.allclose(c.numpy(), 0.1, rtol=1e-2)  # 1 / 3e39 is below the normal range: 7 bits


@pytest.mark.gpu
def test_values_that_are_not_finite(hip):
    from ormi_amd import clip_grads, grad_norm

    for bad in (np.inf, -np.inf, np.nan):
        a, b = np.ones(300, F), np.ones((3, 4), F)
        a[77] = bad
        (ca, cb), norm = clip_grads([tensor(a), tensor(b)], 1.0)
        assert np.array_equal(norm.numpy(), np.abs(bad), equal_nan=True) and np.array_equal(grad_norm([tensor(a)]).numpy(), np.abs(bad), equal_nan=True)
        if np.isnan(bad):
            assert np.isnan(ca.numpy()).all() and np.isnan(cb.numpy()).all()
        else:
            assert np.isnan(ca.numpy()[77]) and not np.delete(ca.numpy(), 77).any() and not cb.numpy().any()


@pytest.mark.gpu
def test_lists_without_elements_and_of_zeros(hip):
    from ormi_amd import clip_grads, grad_norm

    assert float(grad_norm([]).numpy()) == 0.0 and clip_grads([], 1.0)[0] == []
    z = [tensor(np.zeros(5, F)), tensor(np.zeros((0, 3), F))]
    clipped, norm = clip_grads(z, 0.0)
    assert float(norm.numpy()) == 0.0 and not clipped[0].numpy().any() and clipped[1].shape == (0, 3)


@pytest.mark.gpu
def test_views_shared_tensors_and_lazy_gradients(hip):
    """A transposed gradient, an expanded one, the same one twice, and one that is still to be computed; repeated calls give the same bits."""
    from ormi_amd import Tensor, clip_grads, grad_norm

    rng = np.random.default_rng(3)
    a, b = rng.standard_normal((37, 53)).astype(F), rng.standard_normal((1, 9)).astype(F)
    x, w = rng.standard_normal((6, 5)).astype(F), Tensor(rng.standard_normal((4, 5)).astype(F), "hip", requires_grad=True)
    (Tensor(x, "hip") @ w.T).sum().backward()
    at, bt = tensor(a), tensor(b)
    grads = [at.T, bt.expand((11, 9)), at, at, w.grad]
    host = [a.T, np.broadcast_to(b, (11, 9)), a, a, np.broadcast_to(x.sum(0, dtype=np.float64), (4, 5))]
    n = exact_norm(host)
    clipped, norm = clip_grads(grads, 0.5 * n)
    assert abs(float(norm.numpy()) - n) <= 20 * U * n  # the product's own roundings
    for c, h in zip(clipped, host):
        assert np.allclose(c.numpy(), 0.5 * h, rtol=30 * U, atol=30 * U)
    assert all(float(grad_norm(grads).numpy()) == float(norm.numpy()) for _ in range(3))


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [1e-3, 1e6])
def test_clipped_step_bit_for_bit(hip, bits, max_norm):
    from ormi_amd import AdamState, AdamState8, adamw, grad_norm

    host = inputs(SHAPES * 4, 4)
    T = tensor
    if bits == 32:
        states = [AdamState(T(m), T(v)) for _, _, m, v in host]
    else:
        states = [AdamState8.from_codes(p.shape, *encode(m.reshape(-1), 127, 2), *encode(v.reshape(-1), 255, 4)) for p, _, m, v in host]
    before = [[t.numpy() for t in s.values()] for s in states]
    new, moved = adamw([T(h[0]) for h in host], [T(h[1]) for h in host], states, step=3, max_norm=max_norm, **CALL)
    f = factor_of([h[1] for h in host], max_norm)
    assert float(grad_norm([T(h[1]) for h in host]).numpy()) > 1e-2
    for (p, g, _, _), q, s, (m, v) in zip(host, new, moved, before):
        want = step32(p, g * f, m, v, 3, **HYPER)
        assert np.array_equal(q.numpy(), want[0])
        if bits == 32:
            assert np.array_equal(s.m.numpy(), want[1]) and np.array_equal(s.v.numpy(), want[2])
        else:
            assert np.array_equal(s.parts[0].numpy().view(np.int8), encode(want[1].reshape(-1), 127, 2)[0])
    assert BLOCK == 256


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_clips_over_all_its_parameters(hip, bits):
    """Parameters whose step counts differ go in two calls; the norm is that of all of them."""
    from ormi_amd import AdamW, Tensor

    rng = np.random.default_rng(2)
    a, b, c = (Tensor(rng.standard_normal((30, 20)).astype(F), "hip", requires_grad=True) for _ in range(3))
    plain = [Tensor(t.numpy().copy(), "hip", requires_grad=True) for t in (a, b)]
    opt, twin = AdamW([a, b, c], lr=1e-2, state_bits=bits, max_norm=0.5), AdamW(plain, lr=1e-2, state_bits=bits)
    assert opt.norm is None
    for k in range(4):
        norms = []
        for x, y, optimizer in ((a, b, opt), (*plain, twin)):
            loss = (x * y if k != 1 else x * 1.0) - 1.0
            loss = (loss * loss).sum()
            loss.backward()
            used = [p for p in optimizer.params if p.grad is not None]
            norms.append(exact_norm([p.grad.numpy() for p in used]))
            if optimizer is twin:  # clipped by hand, the factor the device's
                f = factor_of([p.grad.numpy() for p in used], 0.5)
                for p in used:
                    p._node.grad = Tensor(p.grad.numpy() * f, "hip")._node
            optimizer.step()
            optimizer.zero_grad()
            loss.zero_grad_graph()
        assert abs(float(opt.norm.numpy()) - norms[0]) <= 1.01 * U * norms[0]
        for x, y in zip((a, b), plain):
            assert np.array_equal(x.numpy(), y.numpy()), k
    assert opt.steps == [4, 3, 0]


class Ref(ctypes.Structure):
    _fields_ = [("data", ctypes.c_void_p), ("out", ctypes.c_void_p), ("count", ctypes.c_int64), ("dtype", ctypes.c_int)]


def test_refusals(cpu, cabi):
    from ormi_amd import AdamState, AdamW, Tensor, adamw, clip_grads, grad_norm

    t = Tensor(np.zeros((2, 3), F), cpu)
    for call in (lambda: grad_norm([t]), lambda: clip_grads([t], 1.0)):
        with pytest.raises(RuntimeError, match="hip device"):
            call()
    for call in (lambda: grad_norm([np.zeros(3)]), lambda: clip_grads([None], 1.0)):
        with pytest.raises(TypeError):
            call()
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError):
            clip_grads([t], bad)
        with pytest.raises(ValueError):
            AdamW([t], max_norm=bad)
        with pytest.raises(ValueError):
            adamw([t], [t], [AdamState(t, t)], step=1, max_norm=bad)
    size, f = ctypes.c_size_t(), ctypes.c_double(1.0)
    for n, ref in [(-1, Ref(64, 64, 1, 0)), (1, None), (1, Ref(None, 64, 1, 0)), (1, Ref(64, 64, -1, 0)), (1, Ref(64, 64, 1, 1)), (1, Ref(64, 64, 1 << 38, 0))]:
        r = ctypes.byref(ref) if ref is not None else None
        assert cabi.ormi_hip_norm_workspace_size(r, n, ctypes.byref(size)) == 3, (n, ref)
        assert cabi.ormi_hip_norm(r, n, f, None, None, None, ctypes.c_size_t(0)) == 3
        assert cabi.ormi_hip_scale(r, n, ctypes.c_void_p(64)) == 3
    one = ctypes.byref(Ref(64, None, 1, 0))
    assert cabi.ormi_hip_scale(one, 1, ctypes.c_void_p(64)) == 3 and b"null tensor" in cabi.ormi_hip_last_error()
    assert cabi.ormi_hip_scale(ctypes.byref(Ref(64, 64, 1, 0)), 1, None) == 3 and b"null factor" in cabi.ormi_hip_last_error()
    assert cabi.ormi_hip_norm(one, 1, f, None, None, None, ctypes.c_size_t(0)) == 3 and b"workspace" in cabi.ormi_hip_last_error()
    assert cabi.ormi_hip_norm(one, 1, ctypes.c_double(-1.0), None, ctypes.c_void_p(64), ctypes.c_void_p(256), ctypes.c_size_t(256)) == 3
    assert cabi.ormi_hip_adamw_scaled(None, ctypes.c_void_p(64)) == 3 and cabi.ormi_hip_adamw_scaled(None, None) == 3

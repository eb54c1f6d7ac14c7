"""The AdamW step over many tensors on the GPU: bit for bit against the same
float32 operations in numpy (no fused multiply-adds on either side), which the
64-bit formula bounds; 8-bit moments; the optimizer; refusals."""
import ctypes

import numpy as np
import pytest

F = np.float32
BLOCK = 256


def step32(p, g, m, v, t, lr, b1, b2, eps, decay):
    """The kernel's operations, each rounded to float32."""
    m = m * F(b1) + g * F(1 - b1)
    v = v * F(b2) + (g * g) * F(1 - b2)
    rate = (m / F(1 - b1 ** t)) / (np.sqrt(v / F(1 - b2 ** t)) + F(eps))
    return p - F(lr) * (rate + F(decay) * p), m, v


def step64(p, g, m, v, t, lr, b1, b2, eps, decay):
    p, g, m, v = (x.astype(np.float64) for x in (p, g, m, v))
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    return p - lr * (m / (1 - b1 ** t) / (np.sqrt(v / (1 - b2 ** t)) + eps) + decay * p), m, v


def bounds(p, g, m, v, t, lr, b1, b2, eps, decay):
    """What float32 roundings may put between step32 and step64, for p, m and v:
    a few units of every term that is added."""
    u = 2.0 ** -24
    new, m1, v1 = step64(p, g, m, v, t, lr, b1, b2, eps, decay)
    root = np.sqrt(v1 / (1 - b2 ** t)) + eps
    em = 4 * u * (b1 * np.abs(m) + (1 - b1) * np.abs(g))
    rate = np.abs(m1) / (1 - b1 ** t) / root
    ep = 4 * u * np.abs(p) + lr * (em / (1 - b1 ** t) / root + 12 * u * rate + 4 * u * decay * np.abs(p))
    return ep, em, 6 * u * v1


def decode(codes, scales, top, root):
    w = np.abs(codes.astype(F)) * F(1.0 / top)
    w = w * w
    if root == 4:
        w = w * w
    return np.sign(codes.astype(F)) * (w * np.repeat(scales, BLOCK))


def encode(x, top, root):
    """(codes padded to whole blocks, scales) of flat float32 x."""
    blocks = np.pad(x, (0, -len(x) % BLOCK)).reshape(-1, BLOCK)
    scale = np.abs(blocks).max(1, keepdims=True, initial=0)
    unit = np.abs(blocks) / np.where(scale == 0, F(1), scale)
    unit = np.sqrt(unit) if root == 2 else np.sqrt(np.sqrt(unit))
    code = np.rint(unit * F(top))
    if root == 4:
        code = np.where(blocks > 0, np.maximum(code, 1), code)
    code = code * np.sign(blocks)
    return code.reshape(-1).astype(np.int8 if root == 2 else np.uint8), scale.reshape(-1)


SHAPES = [(1,), (3,), (4,), (255,), (256,), (257,), (33, 65), (2048,), (2049,), (5, 7, 11), (1024, 72), ()]
HYPER = dict(lr=3e-3, b1=0.9, b2=0.98, eps=1e-8, decay=0.05)
CALL = dict(lr=3e-3, betas=(0.9, 0.98), eps=1e-8, weight_decay=0.05)


def inputs(shapes, seed=0):
    rng = np.random.default_rng(seed)
    return [tuple(np.asarray(rng.standard_normal(s), F) * F(f) for f in (0.1, 0.02, 0.003)) + (np.asarray(rng.standard_normal(s), F) ** 2 * F(1e-4),)
            for s in shapes]


@pytest.mark.gpu
@pytest.mark.parametrize("count", [1, 12, 70])
def test_bits_and_formula(hip, count):
    from ormi_amd import AdamState, Tensor, adamw

    shapes = [SHAPES[i % len(SHAPES)] for i in range(count)]
    host = inputs(shapes, count)
    T = lambda x: Tensor(x, "hip")  # noqa: E731
    params, states = [T(h[0]) for h in host], [AdamState(T(h[2]), T(h[3])) for h in host]
    new, moved = adamw(params, [T(h[1]) for h in host], states, step=3, **CALL)
    for h, p, s, old in zip(host, new, moved, params):
        for got, want, exact, bound in zip((p, *s.values()), step32(*h, 3, **HYPER), step64(*h, 3, **HYPER), bounds(*h, 3, **HYPER)):
            assert got.shape == h[0].shape and np.array_equal(got.numpy(), want)
            assert (np.abs(want - exact) <= bound + 1e-37).all()
        assert np.array_equal(old.numpy(), h[0])  # what was passed in keeps its values


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("bits", [32, 8])
def test_16_bit_parameters_round_once(hip, dtype, bits):
    from ormi_amd import AdamState, AdamState8, Tensor, adamw

    for shape in [(257,), (40, 50)]:
        p, g, m, v = inputs([shape], 5)[0]
        pt, gt = Tensor(p, "hip", dtype=dtype), Tensor(g, "hip", dtype=dtype)
        if bits == 32:
            state = AdamState(Tensor(m, "hip"), Tensor(v, "hip"))
        else:
            state = AdamState8.from_codes(shape, *encode(m.reshape(-1), 127, 2), *encode(v.reshape(-1), 255, 4))
        before = [s.numpy() for s in state.values()]
        (new,), _ = adamw([pt], [gt], [state], step=7, **CALL)
        want = step32(pt.numpy(), gt.numpy(), *before, 7, **HYPER)[0]
        assert new.dtype == dtype and np.array_equal(new.numpy(), Tensor(want, "hip", dtype=dtype).numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("zero", [False, True])
def test_8_bit_states_bit_for_bit(hip, zero):
    from ormi_amd import AdamState8, Tensor, adamw

    host = inputs(SHAPES, 2)
    states, want = [], []
    for p, g, m, v in host:
        if zero:
            m, v = np.zeros_like(m), np.zeros_like(v)
        if p.ndim == 2:
            g[0] = 0  # elements whose moments stay zero beside others that do not
            m[0] = v[0] = 0
        mc, ms = encode(m.reshape(-1), 127, 2)
        vc, vs = encode(v.reshape(-1), 255, 4)
        states.append(AdamState8.zeros(p.shape) if zero else AdamState8.from_codes(p.shape, mc, ms, vc, vs))
        n = p.size
        want.append(step32(p.reshape(-1), g.reshape(-1), decode(mc, ms, 127, 2)[:n], decode(vc, vs, 255, 4)[:n], 1, **HYPER))
    new, moved = adamw([Tensor(h[0], "hip") for h in host], [Tensor(h[1], "hip") for h in host], states, step=1, **CALL)
    for h, p, s, (wp, wm, wv) in zip(host, new, moved, want):
        assert np.array_equal(p.numpy().reshape(-1), wp)
        parts = [t.numpy() for t in s.parts]
        for got, scale, x, top, root in ((parts[0], parts[1], wm, 127, 2), (parts[2], parts[3], wv, 255, 4)):
            codes, scales = encode(x, top, root)
            assert np.array_equal(got.view(codes.dtype), codes) and np.array_equal(scale, scales)
        n = h[0].size
        m, v = (t.numpy().reshape(-1) for t in s.values())
        assert np.array_equal(m, decode(parts[0].view(np.int8), parts[1], 127, 2)[:n])
        assert np.array_equal(v, decode(parts[2].view(np.uint8), parts[3], 255, 4)[:n])
        # a code's spacing: the second moment within 4 / 255 of the block's largest fourth root, and never lost
        assert ((v > 0) == (wv > 0)).all()
        block = np.repeat(parts[3], BLOCK)[:n]
        assert (np.abs(v ** 0.25 - wv ** 0.25) <= np.where(block > 0, 1.001 / 255, 0) * block ** 0.25 + 1e-12).all()


@pytest.mark.gpu
def test_values_that_are_not_finite_stay_in_their_block(hip):
    from ormi_amd import AdamState8, Tensor, adamw

    g = np.ones(600, F)
    g[300] = np.inf
    g[301] = np.nan
    (p,), (s,) = adamw([Tensor(np.ones(600, F), "hip")], [Tensor(g, "hip")], [AdamState8.zeros((600,))], step=1)
    m, v = (t.numpy() for t in s.values())
    assert np.isfinite(m[:256]).all() and np.isfinite(m[512:]).all() and np.isnan(m[256:512]).all()
    assert np.isfinite(v[:256]).all() and np.isnan(v[300]) and np.isfinite(p.numpy()[:256]).all()


@pytest.mark.gpu
def test_gradients_that_are_views(hip):
    """A transposed weight's gradient is a view: it is read in the parameter's order."""
    from ormi_amd import AdamState, Tensor, adamw

    rng = np.random.default_rng(1)
    x, w = rng.standard_normal((6, 5)).astype(F), rng.standard_normal((4, 5)).astype(F)
    wt = Tensor(w, "hip", requires_grad=True)
    (Tensor(x, "hip") @ wt.T).sum().backward()
    g = wt.grad.numpy()
    (new,), _ = adamw([wt], [wt.grad], [AdamState.zeros((4, 5))], step=1, **CALL)
    assert np.array_equal(new.numpy(), step32(w, g, np.zeros_like(w), np.zeros_like(w), 1, **HYPER)[0]) and new.requires_grad


@pytest.mark.gpu
@pytest.mark.parametrize("bits", [32, 8])
def test_optimizer_steps(hip, bits):
    """AdamW over several steps: tensors without a gradient keep value and step count; an old graph keeps its values."""
    from ormi_amd import AdamW, Tensor

    rng = np.random.default_rng(2)
    a, b, c = (Tensor(rng.standard_normal((30, 20)).astype(F), "hip", requires_grad=True) for _ in range(3))
    opt = AdamW([a, b, c], lr=1e-2, state_bits=bits)
    start, kept = a.numpy(), c.numpy()
    losses = []
    for k in range(20):
        loss = ((a * b if k != 1 else a) - 1.0)
        loss = (loss * loss).sum()
        old = a * 1.0
        loss.backward()
        losses.append(float(loss.numpy()))
        before = a.numpy()
        opt.step()
        assert a.grad is None and a.requires_grad and np.array_equal(old.numpy(), before)
        opt.zero_grad()
    assert losses[-1] < losses[2] and not np.array_equal(a.numpy(), start) and np.array_equal(c.numpy(), kept)
    assert opt.steps == [20, 19, 0]


def test_refusals(cpu, cabi):
    from ormi_amd import AdamState, AdamState8, AdamW, Tensor, adamw

    t = Tensor(np.zeros((2, 3), F), cpu)
    z = lambda s=(2, 3): AdamState(Tensor(np.zeros(s, F), cpu), Tensor(np.zeros(s, F), cpu))  # noqa: E731
    with pytest.raises(RuntimeError, match="hip device"):
        adamw([t], [t], [z()], step=1)
    with pytest.raises(RuntimeError, match="as many"):
        adamw([t], [], [z()], step=1)
    with pytest.raises(TypeError, match="all AdamState"):
        adamw([t, t], [t, t], [z(), AdamState8((2, 3), ())], step=1)
    with pytest.raises(TypeError):
        adamw([np.zeros(3)], [t], [z()], step=1)
    with pytest.raises(ValueError):
        AdamW([t], state_bits=16)
    with pytest.raises(ValueError):
        AdamState8.from_codes((2, 3), np.zeros(3, np.int8), np.zeros(1, F), np.zeros(256, np.uint8), np.zeros(1, F), cpu)
    assert cabi.ormi_hip_adamw(None) == 3 and b"null descriptor" in cabi.ormi_hip_last_error()

    class Desc(ctypes.Structure):
        _fields_ = [("n", ctypes.c_int), ("tensors", ctypes.c_void_p), ("bits", ctypes.c_int), ("step", ctypes.c_int64), ("lr", ctypes.c_double),
                    ("b1", ctypes.c_double), ("b2", ctypes.c_double), ("eps", ctypes.c_double), ("decay", ctypes.c_double)]

    good = dict(n=0, bits=32, step=1, lr=1e-3, b1=0.9, b2=0.999, eps=1e-8, decay=0.0)
    for bad in [dict(bits=16), dict(step=0), dict(b1=1.0), dict(b2=-0.1), dict(eps=-1.0), dict(n=1), dict(n=-1), dict(b1=float("nan"))]:
        d = Desc(**{**good, **bad})
        assert cabi.ormi_hip_adamw(ctypes.byref(d)) == 3, bad


@pytest.mark.gpu
def test_refusals_on_the_device(hip):
    from ormi_amd import AdamState, AdamState8, Tensor, adamw

    t = Tensor(np.zeros((2, 3), F), "hip")
    with pytest.raises(RuntimeError, match="another shape than its parameter"):
        adamw([t], [Tensor(np.zeros((3, 2), F), "hip")], [AdamState.zeros((2, 3))], step=1)
    with pytest.raises(RuntimeError, match="state of another shape"):
        adamw([t], [t], [AdamState.zeros((3, 2))], step=1)
    with pytest.raises(RuntimeError, match="state of another shape"):
        adamw([t], [t], [AdamState8.zeros((300,))], step=1)
    with pytest.raises(RuntimeError, match="step counts from 1"):
        adamw([t], [t], [AdamState.zeros((2, 3))], step=0)
    assert adamw([], [], [], step=1) == ([], [])

"""The short causal convolution on the GPU against the formula in 64 bits
(recurrent_ref.py, where the bounds are derived), the formula's gradients against
differences, and refusals."""
import ctypes

import numpy as np
import pytest

import recurrent_ref as ref
from test_recurrence import documents_of, tensor


def run(shape, width, dtype, activation, rng, *, bias=True, initial=False, documents=None, lengths=None, dy=True, dlast=False, fouled=False, wide=False):
    """The call with gradients and what they should be; fouled: what does not count holds NaN and infinities; wide: float32 gradients come in."""
    from ormi_amd import causal_conv, ormi_backend, realize_all

    batch, length, channels = shape
    x = rng.standard_normal(shape).astype(np.float32)
    w = rng.standard_normal(shape).astype(np.float32)
    if fouled:
        off = ~np.moveaxis(ref.rules(length, batch, documents, lengths)[0], 0, 1)[..., 0]
        x[off], w[off] = np.nan, np.inf
    weight = tensor(rng.standard_normal((channels, width)).astype(np.float32), grad=True)
    x, w = tensor(x, dtype, True), tensor(w, dtype)
    b = tensor(rng.standard_normal(channels).astype(np.float32), grad=True) if bias else None
    i = tensor(rng.standard_normal((batch, width - 1, channels)).astype(np.float32), dtype, True) if initial else None
    wl = tensor(rng.standard_normal((batch, width - 1, channels)).astype(np.float32), dtype) if dlast else None
    masks = {n: tensor(t, "int32") for n, t in (("documents", documents), ("lengths", lengths)) if t is not None}
    y, last = causal_conv(x, weight, b, i, activation=activation, **masks)
    assert y.dtype == dtype and last.dtype == dtype and last.shape == (batch, width - 1, channels)
    up = w.numpy()
    if fouled:  # the products with masked NaN stay out of the sum: the gradient is set by hand
        y._node.grad = w._node
        ormi_backend.compute_gradients(y._node)
    else:
        total = None
        if dy:
            total = (y * w * 1.5).sum() if wide else (y * w).sum()
            up = w.numpy() * np.float32(1.5) if wide else up
        if dlast:
            part = (last * wl).sum()
            total = part if total is None else total + part
        total.backward()
    learned = [x, weight] + ([b] if bias else []) + ([i] if initial else [])
    realize_all(y, last, *[t.grad for t in learned])
    want, bound = ref.conv(x.numpy(), weight.numpy(), b.numpy() if bias else None, activation == "silu", i.numpy() if initial else None,
                           documents, lengths, up if dy else None, wl.numpy() if dlast else None)
    assert np.array_equal(last.numpy(), want["last"].astype(np.float32))
    got = {"y": (y, dtype), "dx": (x.grad, dtype), "dw": (weight.grad, "float32")}
    if bias:
        got["db"] = (b.grad, "float32")
    if initial:
        got["dinitial"] = (i.grad, dtype)
    for name, (t, kind) in got.items():
        assert t.dtype == kind
        ref.close(t.numpy(), want[name], bound[name], kind, name)


DTYPES = ["float32", "bfloat16", "float16"]


@pytest.mark.gpu
@pytest.mark.parametrize("activation", [None, "silu"])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 4, 5, 8])
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 5), (3, 8, 64), (1, 255, 33), (2, 256, 8), (2, 600, 65)])
def test_forward_and_gradients(hip, shape, width, dtype, activation):
    rng = np.random.default_rng(sum(shape) + width)
    run(shape, width, dtype, activation, rng, initial=True, dlast=True)
    run(shape, width, dtype, activation, rng, bias=False, wide=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [2, 3, 4, 7])
@pytest.mark.parametrize("shape", [(2, 5, 9), (3, 130, 24), (2, 900, 35)])
def test_documents(hip, shape, width, dtype):
    rng = np.random.default_rng(shape[1])
    docs = documents_of(*shape[:2], min(shape[1], 7), rng)
    run(shape, width, dtype, "silu", rng, documents=docs, initial=True, dlast=True)
    docs[0] = -1  # a row without any token
    run(shape, width, dtype, None, rng, documents=docs, initial=True, dlast=True)
    run(shape, width, dtype, "silu", rng, documents=np.broadcast_to(np.arange(shape[1], dtype=np.int32), shape[:2]).copy())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 3, 4, 6])
@pytest.mark.parametrize("shape", [(5, 6, 9), (6, 300, 24)])
def test_lengths(hip, shape, width, dtype):
    rng = np.random.default_rng(shape[1])
    lengths = np.array([0, 1, shape[1], shape[1] // 2, shape[1] + 5, -3][:shape[0]], np.int32)
    run(shape, width, dtype, "silu", rng, lengths=lengths, initial=True, dlast=True)
    run(shape, width, dtype, "silu", rng, lengths=lengths, documents=documents_of(*shape[:2], 4, rng), initial=True, dlast=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", [3, 4, 8])
def test_what_does_not_count_may_hold_anything(hip, dtype, width):
    rng = np.random.default_rng(3)
    run((3, 900, 24), width, dtype, "silu", rng, lengths=np.array([0, 333, 900], np.int32), initial=True, fouled=True)
    run((3, 900, 24), width, dtype, "silu", rng, documents=documents_of(3, 900, 5, rng), initial=True, fouled=True)


@pytest.mark.gpu
@pytest.mark.parametrize("width", [2, 4, 8])
def test_nothing_passes_from_one_document_to_another(hip, width):
    from ormi_amd import causal_conv, realize_all

    rng = np.random.default_rng(5)
    x, w = rng.standard_normal((2, 2, 90, 12)).astype(np.float32)
    weight = rng.standard_normal((12, width)).astype(np.float32)
    docs = np.zeros((2, 90), np.int32)
    docs[:, 30:60], docs[:, 60:] = 1, 2
    clean, bound = ref.conv(x, weight, None, True, None, docs, None, w)
    x[:, 30:60:4] = np.nan
    w[:, 31:60:4] = np.inf
    xt = tensor(x, grad=True)
    y, _ = causal_conv(xt, tensor(weight), activation="silu", documents=tensor(docs, "int32"))
    (y * tensor(w)).sum().backward()
    realize_all(y, xt.grad)
    away = np.r_[0:30, 60:90]
    ref.close(y.numpy()[:, away], clean["y"][:, away], bound["y"][:, away], "float32")
    ref.close(xt.grad.numpy()[:, away], clean["dx"][:, away], bound["dx"][:, away], "float32")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width", [1, 2, 4, 5])
def test_calls_carry_on(hip, dtype, width):
    """A sequence cut into calls of 1 to 300 tokens, shorter than the width among them, gives the bits of one call."""
    from ormi_amd import causal_conv

    rng = np.random.default_rng(7)
    x = rng.standard_normal((2, 400, 20)).astype(np.float32)
    weight, bias = tensor(rng.standard_normal((20, width)).astype(np.float32)), tensor(rng.standard_normal(20).astype(np.float32))
    whole, end = causal_conv(tensor(x, dtype), weight, bias, activation="silu")
    state, at, rows = None, 0, []
    for n in (1, 1, 2, 1, 300, 3, 91, 1):
        y, state = causal_conv(tensor(x[:, at:at + n].copy(), dtype), weight, bias, state, activation="silu")
        rows.append(y.numpy())
        at += n
    assert np.array_equal(np.concatenate(rows, 1), whole.numpy()) and np.array_equal(state.numpy(), end.numpy())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_views_give_the_same_bits(hip, dtype):
    from ormi_amd import causal_conv, realize_all

    rng = np.random.default_rng(11)
    x, w = rng.standard_normal((2, 2, 300, 24)).astype(np.float32)
    weight = rng.standard_normal((24, 4)).astype(np.float32)

    def both(order, turned):
        back = np.argsort(order)
        held = tensor(np.ascontiguousarray(x.transpose(order)), dtype, True)
        wt = tensor(np.ascontiguousarray(w.transpose(order)), dtype).transpose(list(back))
        taps = tensor(np.ascontiguousarray(weight.T) if turned else weight, grad=True)
        y, last = causal_conv(held.transpose(list(back)), taps.T if turned else taps, activation="silu")
        (y * wt).sum().backward()
        realize_all(y, last, held.grad, taps.grad)
        return [y.numpy(), last.numpy(), held.grad.numpy().transpose(back), taps.grad.numpy().T if turned else taps.grad.numpy()]

    want = both((0, 1, 2), False)
    for order, turned in [((0, 1, 2), False), ((1, 0, 2), True), ((0, 2, 1), False), ((2, 1, 0), True)]:
        for a, b in zip(both(order, turned), want):
            assert np.array_equal(a, b), order


@pytest.mark.gpu
@pytest.mark.parametrize("width", [1, 2, 4, 8])
def test_gradient_through_the_kept_inputs_alone(hip, width):
    """Of two calls in a row, and of a call whose result nothing reads; inputs without a gradient get none."""
    from ormi_amd import causal_conv, realize_all

    rng = np.random.default_rng(17)
    run((2, 70, 20), width, "bfloat16", "silu", rng, initial=True, lengths=np.array([3, 70], np.int32), dy=False, dlast=True)
    x, w = rng.standard_normal((2, 2, 50, 10)).astype(np.float32)
    taps = tensor(rng.standard_normal((10, width)).astype(np.float32), grad=True)
    parts = [tensor(x[:, s].copy(), grad=True) for s in (slice(0, 2), slice(2, 50))]
    y0, kept = causal_conv(parts[0], taps)
    y1, _ = causal_conv(parts[1], taps, None, kept)
    ((y0 * tensor(w[:, :2].copy())).sum() + (y1 * tensor(w[:, 2:].copy())).sum()).backward()
    want, bound = ref.conv(x, taps.numpy(), None, False, dy=w)
    realize_all(taps.grad, *(p.grad for p in parts))
    ref.close(np.concatenate([p.grad.numpy() for p in parts], 1), want["dx"], bound["dx"] + 4 * ref.U * (np.abs(want["dx"]) + 8), "float32")
    ref.close(taps.grad.numpy(), want["dw"], bound["dw"] + 4 * ref.U * np.abs(want["dw"]), "float32")
    only = tensor(x)
    y, _ = causal_conv(only, taps)
    taps.zero_grad()
    (y * tensor(w)).sum().backward()
    assert only.grad is None
    ref.close(taps.grad.numpy(), want["dw"], bound["dw"], "float32")


@pytest.mark.gpu
def test_more_elements_than_2_to_the_31(hip, ob):
    """One tap of 2 and a bias of 1: each result is the same, each input's gradient too, at every offset; the weights'
    gradients are the number of tokens times exact values, which float32 holds."""
    from ormi_amd import causal_conv, realize_all

    tokens = 1 << 20
    shape = (2, tokens, 1040)
    x = tensor(np.full((1, 1, 1040), 0.75, np.float32), "bfloat16", True)
    taps = np.zeros((1040, 4), np.float32)
    taps[:, 2] = 2.0
    weight, bias = (tensor(t, grad=True) for t in (taps, np.ones(1040, np.float32)))
    many = x.expand(shape)
    y, last = causal_conv(many, weight, bias, tensor(np.full((2, 3, 1040), 0.75, np.float32), "bfloat16"))
    (y * tensor(np.full((1, 1, 1), 0.5, np.float32), "bfloat16").expand(shape)).sum().backward()
    realize_all(y, last, many.grad, weight.grad, bias.grad)
    assert (y.max(2).numpy() == 2.5).all() and ((-y).max(2).numpy() == -2.5).all() and (last.numpy() == 0.75).all()
    dx = many.grad.max(2).numpy()
    assert np.array_equal(dx, (-((-many.grad).max(2))).numpy())  # channels alike
    assert (dx[:, :-1] == 1.0).all() and (dx[:, -1] == 0.0).all()  # no token reads the last one as its third tap
    assert (weight.grad.numpy() == 2 * tokens * 0.375).all() and (bias.grad.numpy() == tokens).all()
    del y, last, many, x
    ob.empty_cache()


@pytest.mark.gpu
def test_large_activations_stay_finite(hip):
    from ormi_amd import causal_conv, realize_all

    x = np.array([-1e30, -1e4, -89.0, -20.0, 0.0, 20.0, 89.0, 1e4, 1e30], np.float32).reshape(1, -1, 1)
    xt, one = tensor(x, grad=True), tensor(np.ones((1, 1), np.float32))
    y, _ = causal_conv(xt, one, activation="silu")
    y.sum().backward()
    realize_all(y, xt.grad)
    with np.errstate(over="ignore"):
        s = 1 / (1 + np.exp(-x.astype(np.float64)))
    assert np.allclose(y.numpy(), x * s, rtol=1e-6, atol=1e-35) and np.allclose(xt.grad.numpy(), s * (1 + x * (1 - s)), rtol=2e-6, atol=1e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
@pytest.mark.parametrize("width", [1, 4])
def test_empty(hip, shape, width):
    """Without tokens the kept inputs are the initial ones, and the weights' gradients zero."""
    from ormi_amd import causal_conv, realize_all

    initial = np.arange(shape[0] * (width - 1) * shape[2], dtype=np.float32).reshape(shape[0], width - 1, shape[2])
    x, w, b, i = (tensor(t, grad=True) for t in (np.zeros(shape, np.float32), np.ones((shape[2], width), np.float32), np.ones(shape[2], np.float32), initial))
    y, last = causal_conv(x, w, b, i)
    ((y * 1.0).sum() + (last * 2.0).sum()).backward()
    realize_all(y, last, x.grad, w.grad, b.grad, i.grad)
    assert y.numpy().shape == shape
    if 0 in shape[:2]:
        assert not w.grad.numpy().any() and not b.grad.numpy().any()
    if shape[1] == 0:
        assert np.array_equal(last.numpy(), initial) and np.array_equal(i.grad.numpy(), np.full_like(initial, 2))


def test_formula_gradients_against_differences():
    rng = np.random.default_rng(1)
    shape, width = (2, 23, 3), 4
    docs = documents_of(2, 23, 3, rng)
    for silu in (False, True):
        x, w = rng.standard_normal((2, *shape))
        weight, bias, initial, wl = rng.standard_normal((3, width)), rng.standard_normal(3), *rng.standard_normal((2, 2, width - 1, 3))
        for masks in ({}, {"documents": docs}, {"lengths": np.array([2, 23])}):
            grads = ref.conv(x, weight, bias, silu, initial, dy=w, dlast=wl, **masks)[0]

            def loss(x, weight, bias, initial):
                v = ref.conv(x, weight, bias, silu, initial, **masks)[0]
                return (v["y"] * w).sum() + (v["last"] * wl).sum()

            for k, name in enumerate(("dx", "dw", "db", "dinitial")):
                at = [x, weight, bias, initial]
                step = rng.standard_normal(at[k].shape)
                h = 1e-5  # the difference's error: h^2 of the third derivative and 1e-15 / h of the loss
                up, down = ([t + (e * h * step if j == k else 0) for j, t in enumerate(at)] for e in (1, -1))
                slope = (loss(*up) - loss(*down)) / (2 * h)
                assert abs(slope - (grads[name] * step).sum()) <= 1e-6 * (1 + np.linalg.norm(grads[name]) * np.linalg.norm(step))


class Desc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("batch", ctypes.c_int), ("length", ctypes.c_int), ("channels", ctypes.c_int), ("width", ctypes.c_int),
                ("silu", ctypes.c_int), ("x", ctypes.c_void_p), ("x_strides", ctypes.c_int64 * 2), ("weight", ctypes.c_void_p), ("bias", ctypes.c_void_p),
                ("initial", ctypes.c_void_p), ("documents", ctypes.c_void_p), ("documents_sb", ctypes.c_int64), ("lengths", ctypes.c_void_p),
                ("out", ctypes.c_void_p), ("last", ctypes.c_void_p)]


class GradDesc(ctypes.Structure):
    _fields_ = [("forward", Desc), ("dout_dtype", ctypes.c_int), ("dout", ctypes.c_void_p), ("dout_strides", ctypes.c_int64 * 2), ("dlast", ctypes.c_void_p),
                ("dx", ctypes.c_void_p), ("dweight", ctypes.c_void_p), ("dbias", ctypes.c_void_p), ("dinitial", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


def test_refusals(cpu, cabi):
    from ormi_amd import Tensor, causal_conv

    t = lambda *s, dtype="float32": Tensor(np.zeros(s, np.float32), cpu, dtype=dtype)  # noqa: E731
    x, w = t(2, 5, 3), t(3, 4)
    for bad, match in [((t(5, 3), w), "batch, length, channels"), ((x, t(4, 3)), "weights .* of another shape"), ((x, t(3, 9)), "widths from 1 to 8"),
                       ((x, t(3, 0)), "widths from 1 to 8"), ((x, t(3)), "weights"), ((x, t(3, 4, dtype="bfloat16")), "weights .* as float32"),
                       ((x, w, t(4)), "bias .* of another shape"), ((x, w, None, t(2, 4, 3)), "initial .* of another shape"),
                       ((x, w, None, t(2, 3, 3, dtype="bfloat16")), "initial .* as float32"), ((t(2, 5, 3, dtype="int64"), w), "float32, bfloat16 or float16")]:
        with pytest.raises(RuntimeError, match=match):
            causal_conv(*bad)
    with pytest.raises(RuntimeError, match="documents .* as int32"):
        causal_conv(x, w, documents=t(2, 5))
    with pytest.raises(RuntimeError, match="lengths .* of another shape"):
        causal_conv(x, w, lengths=t(3, dtype="int32"))
    with pytest.raises(ValueError):
        causal_conv(x, w, activation="relu")
    with pytest.raises(TypeError):
        causal_conv(x, np.zeros((3, 4)))

    assert cabi.ormi_hip_conv(None) == 3 and b"null descriptor" in cabi.ormi_hip_last_error()
    assert cabi.ormi_hip_conv_grad(None) == 3 and cabi.ormi_hip_conv_grad_workspace_size(None, None) == 3
    good = dict(dtype=0, batch=1, length=4, channels=4, width=4, x=64, weight=64, out=64)
    for bad in [dict(dtype=1), dict(batch=-1), dict(length=-1), dict(channels=-1), dict(length=(1 << 30) + 1), dict(channels=(1 << 20) + 1), dict(x_strides=(ctypes.c_int64 * 2)(0, (1 << 20) + 1)),
                dict(x_strides=(ctypes.c_int64 * 2)(0, -1)), dict(width=0), dict(width=9), dict(x=None),
                dict(weight=None), dict(out=None)]:
        d = Desc(**{**good, **bad})
        assert cabi.ormi_hip_conv(ctypes.byref(d)) == 3, bad
    assert cabi.ormi_hip_conv_grad(ctypes.byref(GradDesc(forward=Desc(**good), dout=64, dout_dtype=3))) == 3


@pytest.mark.gpu
def test_refusals_on_the_device(hip, cabi):
    """More work-groups than a launch holds, and a workspace too small: refused before anything is read."""
    good = dict(dtype=0, length=4, channels=4, width=4, x=64, weight=64, out=64)
    d = Desc(**good, batch=1 << 24)
    assert cabi.ormi_hip_conv(ctypes.byref(d)) == 3 and b"too large" in cabi.ormi_hip_last_error()
    g = GradDesc(forward=Desc(**good, batch=2), dweight=64)
    size = ctypes.c_size_t()
    assert cabi.ormi_hip_conv_grad_workspace_size(ctypes.byref(g), ctypes.byref(size)) == 0 and size.value > 0
    assert cabi.ormi_hip_conv_grad(ctypes.byref(g)) == 3 and b"workspace" in cabi.ormi_hip_last_error()
    g.workspace, g.workspace_bytes = 256, size.value - 1
    assert cabi.ormi_hip_conv_grad(ctypes.byref(g)) == 3 and b"workspace" in cabi.ormi_hip_last_error()

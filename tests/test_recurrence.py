"""The gated linear recurrence on the GPU against the formula token by token in 64
bits (recurrent_ref.py, where the bounds are derived), the formula's gradients
against differences, and refusals."""
import ctypes

import numpy as np
import pytest

import recurrent_ref as ref

TYPES = [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16"), ("float16", "float32")]


def values(shape, logit, rng, size=1.0):
    """(gates, x) as float32: logits whose sigmoids span a few tokens' to a few hundred tokens' memory, or such values."""
    x = (rng.standard_normal(shape) * size).astype(np.float32)
    if logit:
        return (rng.standard_normal(shape) * 2 + 2).astype(np.float32), x
    g = 1 - np.exp(rng.uniform(np.log(3e-3), np.log(0.9), shape))
    return (g * np.where(rng.random(shape) < 0.1, -1, 1)).astype(np.float32), x  # gates may be negative


def documents_of(batch, length, count, rng, padding=3):
    docs = np.zeros((batch, length), np.int32)
    for b in range(batch):
        docs[b] = np.searchsorted(np.sort(rng.integers(0, max(length, 1), count)), np.arange(length), side="right")
        if b % 2 == 0 and padding:
            docs[b, length - min(padding, length):] = -1
        if length > 40:
            docs[b, 20:24] = -7  # tokens of no document inside
    return docs


def tensor(a, dtype="float32", grad=False):
    from ormi_amd import Tensor

    return Tensor(a, "hip", dtype=dtype, requires_grad=grad)


def run(shape, dtype, gate_dtype, logit, rng, *, initial=False, documents=None, lengths=None, dy=True, dlast=False, fouled=False):
    """The call with gradients and what they should be; fouled: what does not count holds NaN and infinities."""
    from ormi_amd import linear_recurrence, realize_all

    batch, length, channels = shape
    g, x = values(shape, logit, rng)
    w = rng.standard_normal(shape).astype(np.float32)
    if fouled:
        off = ~np.moveaxis(ref.rules(length, batch, documents, lengths)[0], 0, 1)[..., 0]
        for t, bad in ((g, np.nan), (x, np.inf), (w, np.nan)):
            t[off] = bad
    g, x, w = tensor(g, gate_dtype, True), tensor(x, dtype, True), tensor(w, dtype)
    h0 = tensor(rng.standard_normal((batch, channels)).astype(np.float32), grad=True) if initial else None
    wl = tensor(rng.standard_normal((batch, channels)).astype(np.float32)) if dlast else None
    masks = {n: tensor(t, "int32") for n, t in (("documents", documents), ("lengths", lengths)) if t is not None}
    y, last = linear_recurrence(g, x, h0, gate="logit" if logit else "value", **masks)
    assert y.dtype == dtype and last.dtype == "float32" and last.shape == (batch, channels)
    total = None
    if dy:
        total = (y * w).sum() if not fouled else None
    if dlast:
        part = (last * wl).sum()
        total = part if total is None else total + part
    if fouled:  # the products with masked NaN stay out of the sum: the gradients are set by hand
        y._node.grad = w._node
        from ormi_amd import ormi_backend

        ormi_backend.compute_gradients(y._node)
    else:
        total.backward()
    learned = [g, x] + ([h0] if initial else [])
    realize_all(y, last, *[t.grad for t in learned])
    want, bound = ref.recurrence(g.numpy(), x.numpy(), logit, h0.numpy() if initial else None, documents, lengths,
                                 w.numpy() if dy else None, wl.numpy() if dlast else None)
    got = {"y": (y, dtype), "last": (last, "float32"), "dg": (g.grad, gate_dtype), "dx": (x.grad, dtype)}
    if initial:
        got["dinitial"] = (h0.grad, "float32")
    for name, (t, kind) in got.items():
        assert t.dtype == kind
        ref.close(t.numpy(), want[name], bound[name], kind, name)
    return y, last


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1), (2, 3, 5), (3, 4, 64), (1, 5, 33), (2, 127, 8), (1, 128, 72), (2, 129, 65), (1, 1000, 40), (3, 517, 7)])
def test_forward_and_gradients(hip, shape, dtype, gate_dtype, logit):
    rng = np.random.default_rng(sum(shape) + logit)
    run(shape, dtype, gate_dtype, logit, rng, initial=True, dlast=True)
    run(shape, dtype, gate_dtype, logit, rng)


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES[:3])
@pytest.mark.parametrize("shape", [(1, 8200, 16), (2, 5003, 33)])
def test_long_sequences_are_split(hip, shape, dtype, gate_dtype, logit):
    rng = np.random.default_rng(shape[1])
    run(shape, dtype, gate_dtype, logit, rng, initial=True, dlast=True)
    run(shape, dtype, gate_dtype, logit, rng, documents=documents_of(*shape[:2], 6, rng), dlast=True)


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 5, 9), (3, 130, 24), (2, 700, 35)])
def test_documents(hip, shape, dtype, gate_dtype, logit):
    rng = np.random.default_rng(shape[1])
    docs = documents_of(*shape[:2], min(shape[1], 7), rng)
    run(shape, dtype, gate_dtype, logit, rng, documents=docs, initial=True, dlast=True)
    docs[0] = -1  # a row without any token
    run(shape, dtype, gate_dtype, logit, rng, documents=docs, initial=True, dlast=True)
    run(shape, dtype, gate_dtype, logit, rng, documents=np.broadcast_to(np.arange(shape[1], dtype=np.int32), shape[:2]).copy())


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("shape", [(5, 6, 9), (6, 300, 24), (5, 1500, 35)])
def test_lengths(hip, shape, dtype, gate_dtype, logit):
    rng = np.random.default_rng(shape[1])
    lengths = np.array([0, 1, shape[1], shape[1] // 2, shape[1] + 5, -3][:shape[0]], np.int32)
    run(shape, dtype, gate_dtype, logit, rng, lengths=lengths, initial=True, dlast=True)
    run(shape, dtype, gate_dtype, logit, rng, lengths=lengths, documents=documents_of(*shape[:2], 4, rng), initial=True, dlast=True)


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_what_does_not_count_may_hold_anything(hip, dtype, logit):
    rng = np.random.default_rng(3)
    shape = (3, 900, 24)
    run(shape, dtype, dtype, logit, rng, lengths=np.array([0, 333, 900], np.int32), initial=True, fouled=True)
    run(shape, dtype, dtype, logit, rng, documents=documents_of(3, 900, 5, rng), initial=True, fouled=True)


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
def test_nothing_passes_a_restart(hip, logit):
    """A document of NaN and infinite states leaves its neighbours' values and gradients as they are."""
    from ormi_amd import linear_recurrence, realize_all

    rng = np.random.default_rng(9)
    shape = (2, 1200, 12)
    g, x = values(shape, logit, rng)
    w = rng.standard_normal(shape).astype(np.float32)
    docs = np.zeros(shape[:2], np.int32)
    docs[:, 301:] = 1
    docs[:, 700:] = 2
    clean = ref.recurrence(g, x, logit, None, docs, None, w)
    x[:, 310:330] = np.inf
    x[:, 500:510] = np.nan
    w[:, 600:610] = np.nan
    gt, xt = tensor(g, grad=True), tensor(x, grad=True)
    y, _ = linear_recurrence(gt, xt, gate="logit" if logit else "value", documents=tensor(docs, "int32"))
    (y * tensor(w)).sum().backward()
    realize_all(y, gt.grad, xt.grad)
    away = np.r_[0:301, 700:1200]
    for t, name in ((y, "y"), (gt.grad, "dg"), (xt.grad, "dx")):
        ref.close(t.numpy()[:, away], clean[0][name][:, away], clean[1][name][:, away], "float32", name)
    assert not np.isfinite(y.numpy()[:, 330:700]).any()


@pytest.mark.gpu
def test_infinities_and_nan_stay_with_their_channel(hip):
    from ormi_amd import linear_recurrence

    x = np.ones((1, 600, 16), np.float32)
    g = np.full((1, 600, 16), 0.9, np.float32)
    x[0, 100, 3] = np.nan
    x[0, 200, 5] = np.inf
    g[0, 300, 7] = np.nan
    h = linear_recurrence(tensor(g), tensor(x))[0].numpy()[0]
    fine = [c for c in range(16) if c not in (3, 5, 7)]
    assert np.isfinite(h[:, fine]).all() and np.isfinite(h[:100]).all()
    assert np.isnan(h[100:, 3]).all() and not np.isfinite(h[200:, 5]).any() and np.isnan(h[300:, 7]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
def test_gates_at_their_limits(hip, logit):
    """Logits past the sigmoid's range and values of exactly 0 and 1."""
    from ormi_amd import linear_recurrence

    rng = np.random.default_rng(4)
    shape = (2, 400, 9)
    g = rng.choice([-np.inf, -1e30, -100.0, -88.0, 0.0, 20.0, 100.0, 1e30, np.inf] if logit else [0.0, 1.0, -1.0], shape).astype(np.float32)
    x = rng.standard_normal(shape).astype(np.float32)
    h0 = rng.standard_normal((2, 9)).astype(np.float32)
    y, last = linear_recurrence(tensor(g), tensor(x), tensor(h0), gate="logit" if logit else "value")
    with np.errstate(over="ignore"):
        want, bound = ref.recurrence(g, x, logit, h0)
    ref.close(y.numpy(), want["y"], bound["y"] + 1e-30, "float32")  # a logit of -88 counts as -87
    ref.close(last.numpy(), want["last"], bound["last"] + 1e-30, "float32")


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_calls_carry_on(hip, dtype, logit):
    """A sequence cut into calls of 1 to 300 tokens gives what one call gives, within the bounds of both."""
    from ormi_amd import linear_recurrence

    rng = np.random.default_rng(7)
    shape = (2, 700, 20)
    g, x = (tensor(t, dtype).numpy() for t in values(shape, logit, rng))
    want, bound = ref.recurrence(g, x, logit)
    state, at, rows = None, 0, []
    for n in (1, 1, 2, 4, 300, 128, 64, 199, 1):
        y, state = linear_recurrence(tensor(g[:, at:at + n].copy(), dtype), tensor(x[:, at:at + n].copy(), dtype), state, gate="logit" if logit else "value")
        rows.append(y.numpy())
        at += n
    ref.close(np.concatenate(rows, 1), want["y"], bound["y"], dtype)
    ref.close(state.numpy(), want["last"], bound["last"], "float32")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_views_give_the_same_bits(hip, dtype):
    """Transposed and expanded inputs and gradients, and the same call twice."""
    from ormi_amd import linear_recurrence, realize_all

    rng = np.random.default_rng(11)
    shape = (2, 300, 24)
    g, x = values(shape, False, rng)
    w = rng.standard_normal(shape).astype(np.float32)

    def both(order):
        back = np.argsort(order)
        held = [tensor(np.ascontiguousarray(t.transpose(order)), dtype, True) for t in (g, x)]
        wt = tensor(np.ascontiguousarray(w.transpose(order)), dtype).transpose(list(back))
        y, last = linear_recurrence(*(t.transpose(list(back)) for t in held))
        (y * wt).sum().backward()
        realize_all(y, last, *[t.grad for t in held])
        return [y.numpy(), last.numpy()] + [t.grad.numpy().transpose(back) for t in held]

    want = both((0, 1, 2))
    for order in [(0, 1, 2), (1, 0, 2), (0, 2, 1), (2, 1, 0)]:
        for a, b in zip(both(order), want):
            assert np.array_equal(a, b), order
    # one gate per channel, for all tokens: its gradient adds up
    one = tensor(g[:1, :1].copy(), dtype, True)
    xt = tensor(x, dtype)
    y, _ = linear_recurrence(one.expand(shape), xt)
    (y * tensor(w, dtype)).sum().backward()
    many, bound = ref.recurrence(np.broadcast_to(one.numpy(), shape), xt.numpy(), False, dy=tensor(w, dtype).numpy())
    total = many["dg"].sum((0, 1), keepdims=True)
    slack = bound["dg"].sum((0, 1), keepdims=True) + (ref.HALF[dtype] + 600 * ref.U) * np.abs(many["dg"]).sum((0, 1), keepdims=True)
    ref.close(one.grad.numpy(), total, slack, "float32")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 40000, 128), (3, 6000, 520), (8, 2000, 1000)])
@pytest.mark.parametrize("masked", [False, True])
def test_calls_give_the_same_bits(hip, shape, masked):
    """Tiles wait for one another in whatever order they run: no bit of any result depends on it."""
    from ormi_amd import linear_recurrence, realize_all

    rng = np.random.default_rng(21)
    g, x = values(shape, False, rng)
    g, x, w = tensor(np.abs(g), grad=True), tensor(x, "bfloat16", True), tensor(rng.standard_normal(shape).astype(np.float32), "bfloat16")
    masks = {"documents": tensor(documents_of(*shape[:2], 5, rng), "int32")} if masked else {}
    first = None
    for _ in range(6):
        for t in (g, x):
            t.zero_grad()
        y, last = linear_recurrence(g, x, **masks)
        total = (y * w).sum()
        total.backward()
        realize_all(y, last, g.grad, x.grad)
        got = [t.numpy() for t in (y, last, g.grad, x.grad)]
        total.zero_grad_graph()
        first = first or got
        assert all(np.array_equal(a, b) for a, b in zip(got, first))


@pytest.mark.gpu
def test_more_elements_than_2_to_the_31(hip, ob):
    """Gates of zero pass nothing on: each state is its input, each input's gradient the result's, at every offset."""
    from ormi_amd import linear_recurrence, realize_all

    shape = (2, (1 << 20) + 300, 1040)
    x, g = tensor(np.full((1, 1, 1040), 0.75, np.float32), "bfloat16", True), tensor(np.zeros((1, 1, 1040), np.float32), "bfloat16")
    many = x.expand(shape)
    y, last = linear_recurrence(g.expand(shape), many)
    (y * tensor(np.full((1, 1, 1), 0.5, np.float32), "bfloat16").expand(shape)).sum().backward()
    realize_all(y, last, many.grad)
    for t, value in ((y, 0.75), (many.grad, 0.5)):
        assert (t.max(2).numpy() == value).all() and ((-t).max(2).numpy() == -value).all()
    assert (last.numpy() == 0.75).all()
    del y, last, many, x, g
    ob.empty_cache()


@pytest.mark.gpu
def test_tokens_far_apart(hip, cabi):
    """Tokens 2^21 elements apart: more than a tile's offsets hold, so the call reads a copy; the entry itself refuses them."""
    from ormi_amd import causal_conv, linear_recurrence, realize_all

    rng = np.random.default_rng(19)
    held = (rng.integers(-4, 5, (3, 1 << 19, 4)) / 4).astype(np.float32)
    near = np.ascontiguousarray(held.transpose(1, 0, 2))
    taps = tensor(rng.standard_normal((4, 3)).astype(np.float32))
    results = []
    for far in (True, False):
        leaf = tensor(held if far else near, grad=True)
        x = leaf.transpose([1, 0, 2]) if far else leaf
        y, last = linear_recurrence(x, x)
        z, kept = causal_conv(x, taps)
        ((y * x).sum() + (z * x).sum()).backward()
        realize_all(y, last, z, kept, leaf.grad)
        results.append([t.numpy() for t in (y, last, z, kept)] + [leaf.grad.numpy().transpose(1, 0, 2) if far else leaf.grad.numpy()])
    assert all(np.array_equal(a, b) for a, b in zip(*results))
    d = Desc(dtype=0, gate_dtype=0, batch=1, length=4, channels=4, gates=64, x=64, out=64)
    for strides in ((0, (1 << 20) + 1), (0, -1)):
        d.x_strides = (ctypes.c_int64 * 2)(*strides)
        assert cabi.ormi_hip_recurrence(ctypes.byref(d)) == 3 and b"apart" in cabi.ormi_hip_last_error()


@pytest.mark.gpu
def test_gradient_reaches_through_the_last_state_alone_and_twice(hip):
    from ormi_amd import linear_recurrence, realize_all

    rng = np.random.default_rng(12)
    run((2, 200, 16), "bfloat16", "float32", True, rng, initial=True, dy=False, dlast=True)
    # one state feeds the next call: the gradient of two calls in a row is that of one
    shape = (2, 60, 10)
    g, x = values(shape, False, rng)
    w = rng.standard_normal(shape).astype(np.float32)
    parts = [[tensor(t[:, s].copy(), grad=True) for t in (g, x)] for s in (slice(0, 37), slice(37, 60))]
    y0, state = linear_recurrence(*parts[0])
    y1, last = linear_recurrence(*parts[1], state)
    ((y0 * tensor(w[:, :37].copy())).sum() + (y1 * tensor(w[:, 37:].copy())).sum()).backward()
    want, bound = ref.recurrence(g, x, False, dy=w)
    realize_all(*(t.grad for p in parts for t in p))
    for k, name in enumerate(("dg", "dx")):
        ref.close(np.concatenate([p[k].grad.numpy() for p in parts], 1), want[name], bound[name], "float32", name)
    # the result read twice and the state too
    gt, xt = tensor(g, grad=True), tensor(x, grad=True)
    y, last = linear_recurrence(gt, xt)
    wl = rng.standard_normal((2, 10)).astype(np.float32)
    ((y * tensor(w)).sum() + (last * tensor(wl)).sum() + (y * 2.0).sum() + (last * 3.0).sum()).backward()
    want, bound = ref.recurrence(g, x, False, dy=w + np.float32(2), dlast=wl + np.float32(3))
    more = ref.U * 4
    for t, name in ((gt, "dg"), (xt, "dx")):
        ref.close(t.grad.numpy(), want[name], bound[name] * 2 + more * np.abs(want[name]) + 1e-5, "float32", name)
    assert y.grad is not None and y.grad.shape == shape and np.allclose(y.grad.numpy(), w + 2)


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
def test_gradients_of_some_inputs_and_of_two_passes(hip, logit):
    """Only what asks for a gradient gets one; a second backward pass over new graphs of the same leaves adds to the first's."""
    from ormi_amd import linear_recurrence

    rng = np.random.default_rng(14)
    shape = (2, 300, 18)
    g, x = values(shape, logit, rng)
    w = rng.standard_normal(shape).astype(np.float32)
    want, bound = ref.recurrence(g, x, logit, np.zeros((2, 18)), dy=w)
    for which in range(3):
        leaves = [tensor(t, grad=k == which) for k, t in enumerate((g, x, np.zeros((2, 18), np.float32)))]
        for times in (1, 2):
            y, last = linear_recurrence(*leaves, gate="logit" if logit else "value")
            (y * tensor(w)).sum().backward()
            got = leaves[which].grad.numpy()
            name = ("dg", "dx", "dinitial")[which]
            ref.close(got, times * want[name], times * bound[name] + 2 * ref.U * np.abs(want[name]), "float32", name)
        assert all(t.grad is None for k, t in enumerate(leaves) if k != which)


@pytest.mark.gpu
def test_same_tensor_as_gates_and_inputs(hip):
    from ormi_amd import linear_recurrence

    rng = np.random.default_rng(13)
    x = rng.uniform(-0.9, 0.9, (2, 50, 6)).astype(np.float32)
    w = rng.standard_normal((2, 50, 6)).astype(np.float32)
    xt = tensor(x, grad=True)
    (linear_recurrence(xt, xt)[0] * tensor(w)).sum().backward()
    want, bound = ref.recurrence(x, x, False, dy=w)
    ref.close(xt.grad.numpy(), want["dg"] + want["dx"], bound["dg"] + bound["dx"] + 2 * ref.U * np.abs(want["dg"]), "float32")


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(0, 3, 4), (2, 0, 4), (2, 3, 0)])
def test_empty(hip, shape):
    from ormi_amd import linear_recurrence, realize_all

    h0 = np.arange(shape[0] * shape[2], dtype=np.float32).reshape(shape[0], shape[2])
    g, x, i = tensor(np.zeros(shape, np.float32), grad=True), tensor(np.zeros(shape, np.float32), grad=True), tensor(h0, grad=True)
    y, last = linear_recurrence(g, x, i)
    ((y * 1.0).sum() + (last * 2.0).sum()).backward()
    realize_all(y, last, g.grad, x.grad, i.grad)
    assert y.numpy().shape == shape and g.grad.numpy().shape == shape
    if shape[1] == 0:
        assert np.array_equal(last.numpy(), h0) and np.array_equal(i.grad.numpy(), np.full_like(h0, 2))


def test_formula_gradients_against_differences():
    rng = np.random.default_rng(1)
    shape = (2, 23, 3)
    docs = documents_of(2, 23, 3, rng)
    for logit in (False, True):
        g, x = (t.astype(np.float64) for t in values(shape, logit, rng))
        h0, wl = rng.standard_normal((2, 2, 3))
        w = rng.standard_normal(shape)
        for masks in ({}, {"documents": docs}, {"lengths": np.array([5, 23])}):
            grads = ref.recurrence(g, x, logit, h0, dy=w, dlast=wl, **masks)[0]

            def loss(g, x, h0):
                v = ref.recurrence(g, x, logit, h0, **masks)[0]
                return (v["y"] * w).sum() + (v["last"] * wl).sum()

            for k, name in enumerate(("dg", "dx", "dinitial")):
                at = [g, x, h0]
                step = rng.standard_normal(at[k].shape)
                h = 1e-5  # the difference's error: h^2 of the third derivative and 1e-15 / h of the loss
                up, down = ([t + (e * h * step if j == k else 0) for j, t in enumerate(at)] for e in (1, -1))
                slope = (loss(*up) - loss(*down)) / (2 * h)
                assert abs(slope - (grads[name] * step).sum()) <= 1e-6 * (1 + np.linalg.norm(grads[name]) * np.linalg.norm(step))


class Desc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("gate_dtype", ctypes.c_int), ("batch", ctypes.c_int), ("length", ctypes.c_int), ("channels", ctypes.c_int),
                ("logits", ctypes.c_int), ("gates", ctypes.c_void_p), ("gate_strides", ctypes.c_int64 * 2), ("x", ctypes.c_void_p),
                ("x_strides", ctypes.c_int64 * 2), ("initial", ctypes.c_void_p), ("documents", ctypes.c_void_p), ("documents_sb", ctypes.c_int64),
                ("lengths", ctypes.c_void_p), ("out", ctypes.c_void_p), ("last", ctypes.c_void_p), ("states", ctypes.c_void_p),
                ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]


class GradDesc(ctypes.Structure):
    _fields_ = [("forward", Desc), ("dout_dtype", ctypes.c_int), ("dout", ctypes.c_void_p), ("dout_strides", ctypes.c_int64 * 2),
                ("dlast", ctypes.c_void_p), ("dgates", ctypes.c_void_p), ("dx", ctypes.c_void_p), ("dinitial", ctypes.c_void_p)]


def test_refusals(cpu, cabi):
    from ormi_amd import Tensor, linear_recurrence

    t = lambda *s, dtype="float32": Tensor(np.zeros(s, np.float32), cpu, dtype=dtype)  # noqa: E731
    x = t(2, 5, 3)
    for bad, match in [((t(2, 5, 4), x), "gates of another shape"), ((t(2, 5), x), "another shape"), ((t(5, 3), t(5, 3)), "batch, length, channels"),
                       ((t(2, 5, 3, dtype="bfloat16"), x), "x's type or float32"), ((x, t(2, 5, 3, dtype="int64")), "float32, bfloat16 or float16"),
                       ((x, x, t(2, 4)), "initial .* of another shape"), ((x, x, t(2, 3, dtype="bfloat16")), "initial .* as float32")]:
        with pytest.raises(RuntimeError, match=match):
            linear_recurrence(*bad)
    with pytest.raises(RuntimeError, match="documents .* as int32"):
        linear_recurrence(x, x, documents=t(2, 5))
    with pytest.raises(RuntimeError, match="documents .* of another shape"):
        linear_recurrence(x, x, documents=t(5, dtype="int32"))
    with pytest.raises(RuntimeError, match="lengths .* of another shape"):
        linear_recurrence(x, x, lengths=t(3, dtype="int32"))
    with pytest.raises(ValueError):
        linear_recurrence(x, x, gate="tanh")
    with pytest.raises(TypeError):
        linear_recurrence(np.zeros((2, 5, 3)), x)

    assert cabi.ormi_hip_recurrence(None) == 3 and b"null descriptor" in cabi.ormi_hip_last_error()
    assert cabi.ormi_hip_recurrence_grad(None) == 3
    size = ctypes.c_size_t()
    assert cabi.ormi_hip_recurrence_workspace_size(None, ctypes.byref(size)) == 3
    good = dict(dtype=0, gate_dtype=0, batch=1, length=4, channels=4, gates=64, x=64, out=64)
    for bad in [dict(dtype=1), dict(gate_dtype=3), dict(dtype=3, gate_dtype=4), dict(batch=-1), dict(length=-1), dict(channels=-1), dict(length=(1 << 30) + 1),
                dict(channels=(1 << 20) + 1), dict(gates=None), dict(x=None), dict(out=None), dict(batch=1 << 24, channels=64)]:
        d = Desc(**{**good, **bad})
        assert cabi.ormi_hip_recurrence(ctypes.byref(d)) == 3, bad
    for bad in [dict(forward=Desc(**good)), dict(forward=Desc(**good, states=64), dout=64, dout_dtype=3)]:
        assert cabi.ormi_hip_recurrence_grad(ctypes.byref(GradDesc(**bad))) == 3, bad


@pytest.mark.gpu
def test_workspace_too_small(hip, cabi):
    d = Desc(dtype=0, gate_dtype=0, batch=1, length=4096, channels=4, gates=64, x=64, out=64)
    size = ctypes.c_size_t()
    assert cabi.ormi_hip_recurrence_workspace_size(ctypes.byref(d), ctypes.byref(size)) == 0 and size.value > 0
    assert cabi.ormi_hip_recurrence(ctypes.byref(d)) == 3 and b"workspace" in cabi.ormi_hip_last_error()
    d.workspace, d.workspace_bytes = 256, size.value - 1
    assert cabi.ormi_hip_recurrence(ctypes.byref(d)) == 3 and b"workspace" in cabi.ormi_hip_last_error()

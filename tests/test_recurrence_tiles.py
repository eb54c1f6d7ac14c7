"""The recurrence where each work-group goes through several tiles of 128 tokens, the
state in registers and the next tile's loads under way: what batches and channels
enough for the card select. Against the formula in 64 bits (recurrent_ref.py), whose
bounds count 80 joins: 2 of segments, 4 of waves and 4 of each tile before, at most 5
here."""
import ctypes

import numpy as np
import pytest

import recurrent_ref as ref
from test_recurrence import TYPES, Desc, documents_of, run, tensor, values

SHAPES = [(520, 300, 5), (130, 389, 197)]  # 520 chains of 64 channels each: 3 and 4 tiles, the last one in part
CODES = {"float32": 0, "bfloat16": 3, "float16": 4}


def unchained(cabi, shape, dtype, gate_dtype):
    """No workspace: no tile waits for another's."""
    size = ctypes.c_size_t(1)
    d = Desc(dtype=CODES[dtype], gate_dtype=CODES[gate_dtype], batch=shape[0], length=shape[1], channels=shape[2])
    assert cabi.ormi_hip_recurrence_workspace_size(ctypes.byref(d), ctypes.byref(size)) == 0
    return size.value == 0


def masks_of(shape, which, rng):
    masks = {}
    if "documents" in which:
        masks["documents"] = documents_of(*shape[:2], 5, rng)
        masks["documents"][3] = -1  # a row without any token
        masks["documents"][5] = np.arange(shape[1])  # one token each
    if "lengths" in which:
        masks["lengths"] = rng.integers(0, shape[1] + 1, shape[0]).astype(np.int32)
        masks["lengths"][:6] = 0, 1, shape[1], 128, 129, 256
    return masks


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES)
@pytest.mark.parametrize("masks", ["", "documents", "lengths", "documents and lengths"])
@pytest.mark.parametrize("shape", SHAPES[:1])
def test_forward_and_gradients(hip, cabi, shape, masks, dtype, gate_dtype, logit):
    assert unchained(cabi, shape, dtype, gate_dtype)
    rng = np.random.default_rng(len(masks) + logit)
    run(shape, dtype, gate_dtype, logit, rng, initial=True, dlast=True, **masks_of(shape, masks, rng))


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES[:3])
@pytest.mark.parametrize("masks", ["", "documents"])
def test_several_channel_blocks(hip, cabi, masks, dtype, gate_dtype, logit):
    assert unchained(cabi, SHAPES[1], dtype, gate_dtype)
    rng = np.random.default_rng(len(masks) + logit)
    run(SHAPES[1], dtype, gate_dtype, logit, rng, **masks_of(SHAPES[1], masks, rng))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,gate_dtype", TYPES[1:])
@pytest.mark.parametrize("masks", ["", "documents and lengths"])
def test_float32_gradients_come_in(hip, cabi, masks, dtype, gate_dtype):
    """A gradient that arrives in float32 beside 16-bit inputs: tiles are loaded when they are reached."""
    from ormi_amd import linear_recurrence, realize_all

    shape = SHAPES[0]
    assert unchained(cabi, shape, dtype, gate_dtype)
    rng = np.random.default_rng(7)
    held = masks_of(shape, masks, rng)
    g, x = values(shape, True, rng)
    w = rng.standard_normal(shape).astype(np.float32)
    g, x, w = tensor(g, gate_dtype, True), tensor(x, dtype, True), tensor(w)
    y, last = linear_recurrence(g, x, gate="logit", **{n: tensor(t, "int32") for n, t in held.items()})
    (y * w * 1.5).sum().backward()
    realize_all(y, last, g.grad, x.grad)
    want, bound = ref.recurrence(g.numpy(), x.numpy(), True, None, held.get("documents"), held.get("lengths"), w.numpy() * np.float32(1.5))
    for name, t, kind in (("y", y, dtype), ("last", last, "float32"), ("dg", g.grad, gate_dtype), ("dx", x.grad, dtype)):
        ref.close(t.numpy(), want[name], bound[name], kind, name)


@pytest.mark.gpu
@pytest.mark.parametrize("logit", [False, True])
@pytest.mark.parametrize("dtype,gate_dtype", TYPES[:3])
@pytest.mark.parametrize("masks", ["documents", "lengths"])
def test_what_does_not_count_may_hold_anything(hip, cabi, masks, dtype, gate_dtype, logit):
    shape = SHAPES[0]
    assert unchained(cabi, shape, dtype, gate_dtype)
    rng = np.random.default_rng(3)
    run(shape, dtype, gate_dtype, logit, rng, initial=True, fouled=True, **masks_of(shape, masks, rng))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_same_bits(hip, cabi, dtype):
    """Of two calls; and of a batch's first tile where it is called alone, whose tiles wait for one another."""
    from ormi_amd import linear_recurrence, realize_all

    shape = (520, 300, 5)
    rng = np.random.default_rng(9)
    g, x = values(shape, False, rng)
    w = rng.standard_normal(shape).astype(np.float32)

    def both(rows):
        gt, xt = tensor(g[rows].copy(), dtype, True), tensor(x[rows].copy(), dtype, True)
        y, last = linear_recurrence(gt, xt)
        total = (y * tensor(w[rows].copy(), dtype)).sum()
        total.backward()
        realize_all(y, last, gt.grad, xt.grad)
        got = [t.numpy().copy() for t in (y, last, gt.grad, xt.grad)]
        total.zero_grad_graph()
        return got

    whole = both(slice(None))
    assert all(np.array_equal(a, b) for a, b in zip(whole, both(slice(None))))
    assert np.array_equal(whole[0][17:18, :128], both(slice(17, 18))[0][:, :128])

"""Rotary positions on the GPU against the formula in 64 bits, and refusals.

The tables are float32 (half-spacing u of their values, at most the magnitude);
each result is two products and a sum, rounded once more to its type:
|error| <= 4 u (|a| + |b|) magnitude + half a spacing of the result.
"""
import math

import numpy as np
import pytest

U = 2.0 ** -24
HALF = {"float32": 2.0 ** -24, "bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}  # of 24, 8 and 11 significant bits


def frequencies(part, base=10000.0, scaling="none", factor=1.0, original=None, slow=1.0, fast=32.0):
    p = np.arange(part // 2)
    if scaling == "base" and part > 2:
        base *= factor ** (part / (part - 2))
    f = base ** (-2.0 * p / max(part, 1))
    if scaling == "linear":
        f /= factor
    if scaling == "parts":
        keep = np.clip((original * f / (2 * math.pi) - slow) / (fast - slow), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    return f


def turned(x, pos, part, pairs, inverse=False, magnitude=1.0, **scaling):
    x = x.astype(np.float64)
    angle = pos[..., None] * frequencies(part, **scaling)
    c, s = (f(angle)[:, :, None] * magnitude for f in (np.cos, np.sin))
    s = -s if inverse else s
    first, second = (slice(0, part // 2), slice(part // 2, part)) if pairs == "half" else (slice(0, part, 2), slice(1, part, 2))
    a, b = x[..., first], x[..., second]
    out, size = x.copy(), np.abs(x)
    out[..., first], out[..., second] = a * c - b * s, b * c + a * s
    size[..., first] = size[..., second] = (np.abs(a) + np.abs(b)) * magnitude
    return out, size


def assert_turned(got, want, dtype):
    exact, size = want
    bound = 4 * U * size + HALF[dtype] * np.abs(exact) + (2.0 ** -25 if dtype == "float16" else 1e-37)
    worst = float(np.max(np.abs(got.astype(np.float64) - exact) / bound, initial=0.0))
    assert worst <= 1.0, worst


@pytest.mark.gpu
@pytest.mark.parametrize("pairs", ["half", "interleaved"])
@pytest.mark.parametrize("dtype,out", [("float32", "float32"), ("float32", "bfloat16"), ("bfloat16", "bfloat16"), ("float16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("shape,part", [((1, 1, 1, 2), 2), ((2, 3, 5, 7), 4), ((2, 17, 4, 64), 64), ((1, 9, 6, 80), 48), ((3, 5, 9, 33), 22),
                                        ((2, 4, 3, 24), 8), ((1, 3, 2, 16), 0), ((2, 1, 33, 128), 128)])
def test_forward_and_gradient(hip, pairs, dtype, out, shape, part):
    from ormi_amd import RotaryTable, Tensor, realize_all, rotary

    rng = np.random.default_rng(part + shape[1])
    x = Tensor(rng.standard_normal(shape, dtype=np.float32), "hip", requires_grad=True, dtype=dtype)
    w = Tensor(rng.standard_normal(shape, dtype=np.float32), "hip", dtype=out)
    table = RotaryTable(part, 40, "hip")
    y = rotary(x, table, offset=11, pairs=pairs, dtype=out)
    (y * w).sum().backward()
    realize_all(y, x.grad)
    assert y.dtype == out and x.grad.dtype == dtype
    pos = np.broadcast_to(11 + np.arange(shape[1]), shape[:2])
    assert_turned(y.numpy(), turned(x.numpy(), pos, part, pairs), out)
    assert_turned(x.grad.numpy(), turned(w.numpy(), pos, part, pairs, inverse=True), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("scaling", [dict(), dict(scaling="linear", factor=4.0), dict(scaling="base", factor=8.0),
                                     dict(scaling="parts", factor=8.0, original=512), dict(base=500.0, magnitude=1.25)])
@pytest.mark.parametrize("per_batch", [False, True])
def test_positions_and_scaled_tables(hip, scaling, per_batch):
    from ormi_amd import RotaryTable, Tensor, rotary

    rng = np.random.default_rng(8)
    x = rng.standard_normal((3, 50, 2, 32), dtype=np.float32)
    pos = rng.integers(0, 30000, (3, 50) if per_batch else (50,)).astype(np.int32)
    table = RotaryTable(32, 30000, "hip", **scaling)
    got = rotary(Tensor(x, "hip"), table, Tensor(pos, "hip", dtype="int32")).numpy()
    assert_turned(got, turned(x, np.broadcast_to(pos, (3, 50)), 32, "half", **scaling), "float32")


@pytest.mark.gpu
@pytest.mark.parametrize("dim,part", [(64, 64), (40, 16), (33, 10)])
def test_views_give_the_same_bits(hip, dim, part):
    from ormi_amd import RotaryTable, Tensor, rotary

    x = np.random.default_rng(3).standard_normal((2, 6, 5, dim), dtype=np.float32)
    table = RotaryTable(part, 6, "hip")
    for dtype in ("float32", "bfloat16"):
        want = rotary(Tensor(x, "hip", dtype=dtype), table).numpy()
        for order in [(0, 2, 1, 3), (3, 1, 2, 0)]:
            held = Tensor(np.ascontiguousarray(x.transpose(order)), "hip", dtype=dtype)
            assert np.array_equal(rotary(held.transpose(order), table).numpy(), want)
    row = Tensor(np.ascontiguousarray(x[:1, :, :1]), "hip")
    wide = rotary(row.expand((2, 6, 5, dim)), table).numpy()
    assert np.array_equal(wide, np.broadcast_to(rotary(row, table).numpy(), wide.shape))


@pytest.mark.gpu
def test_gradient_through_broadcast_and_use_twice(hip):
    """The gradient of an expanded row adds up, and so does that of a tensor turned at two offsets."""
    from ormi_amd import RotaryTable, Tensor, rotary

    rng = np.random.default_rng(4)
    x = Tensor(rng.standard_normal((1, 4, 1, 8), dtype=np.float32), "hip", requires_grad=True)
    w = rng.standard_normal((2, 4, 3, 8), dtype=np.float32)
    table = RotaryTable(8, 64, "hip")
    wide = x.expand((2, 4, 3, 8))
    ((rotary(wide, table) + rotary(wide, table, offset=20)) * Tensor(w, "hip")).sum().backward()
    pos = np.broadcast_to(np.arange(4), (2, 4))
    want = turned(w, pos, 8, "half", inverse=True)[0] + turned(w, pos + 20, 8, "half", inverse=True)[0]
    assert np.allclose(x.grad.numpy(), want.sum((0, 2), keepdims=True), rtol=0, atol=64 * U * np.abs(w).sum())


@pytest.mark.gpu
def test_positions_outside_the_table_are_nan(hip):
    from ormi_amd import RotaryTable, Tensor, rotary

    x = np.ones((1, 4, 3, 8), np.float32)
    pos = Tensor(np.array([0, -1, 5, 2**31 - 1], np.int32), "hip", dtype="int32")
    got = rotary(Tensor(x, "hip"), RotaryTable(6, 5, "hip"), pos).numpy()
    assert np.isfinite(got[0, 0]).all() and np.isnan(got[0, 1:, :, :6]).all() and (got[..., 6:] == 1).all()


@pytest.mark.gpu
def test_empty(hip):
    from ormi_amd import RotaryTable, Tensor, rotary

    for shape in [(0, 2, 1, 8), (2, 0, 1, 8), (2, 2, 0, 8)]:
        assert rotary(Tensor(np.zeros(shape, np.float32), "hip"), RotaryTable(8, 4, "hip")).numpy().shape == shape


def test_refusals(cpu, cabi):
    from ormi_amd import RotaryTable, Tensor, rotary

    x = Tensor(np.zeros((1, 4, 2, 8), np.float32), cpu)
    table = RotaryTable(8, 6, cpu)
    with pytest.raises(RuntimeError, match="outside the tables"):
        rotary(x, table, offset=3)
    with pytest.raises(RuntimeError, match="outside the tables"):
        rotary(x, table, offset=-1)
    with pytest.raises(RuntimeError, match="more pairs"):
        rotary(x, RotaryTable(10, 6, cpu))
    with pytest.raises(RuntimeError, match="batch, length, heads, features"):
        rotary(Tensor(np.zeros((4, 2, 8), np.float32), cpu), table)
    with pytest.raises(RuntimeError, match="positions"):
        rotary(x, table, Tensor(np.zeros(3, np.int32), cpu, dtype="int32"))
    with pytest.raises(RuntimeError, match="int32"):
        rotary(x, table, Tensor(np.zeros(4, np.float32), cpu))
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        rotary(x, table, dtype="int64")
    with pytest.raises(ValueError):
        rotary(x, table, pairs="thirds")
    with pytest.raises(ValueError):
        rotary(x, table, Tensor(np.zeros(4, np.int32), cpu, dtype="int32"), offset=1)
    for bad in [dict(part=3), dict(part=-2), dict(positions=-1), dict(scaling="dynamic"), dict(scaling="parts"), dict(base=0.0)]:
        with pytest.raises(ValueError):
            RotaryTable(**{"part": 8, "positions": 6, "device": cpu, **bad})
    assert cabi.ormi_hip_rotary(None) == 3 and b"null descriptor" in cabi.ormi_hip_last_error()

"""Calls whose work-groups or threads would not fit one launch are cut into
launches that do, or refused before anything is read; none is cut short."""
import ctypes

import numpy as np
import pytest


class Rotary(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("out_dtype", ctypes.c_int), ("batch", ctypes.c_int), ("length", ctypes.c_int), ("heads", ctypes.c_int),
                ("dim", ctypes.c_int), ("part", ctypes.c_int), ("interleaved", ctypes.c_int), ("inverse", ctypes.c_int), ("x", ctypes.c_void_p),
                ("x_strides", ctypes.c_int64 * 4), ("out", ctypes.c_void_p), ("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p),
                ("table_rows", ctypes.c_int), ("positions", ctypes.c_void_p), ("positions_strides", ctypes.c_int64 * 2), ("offset", ctypes.c_int)]


def test_rotary_refuses_tokens_of_more_threads_than_a_launch(cabi):
    """2^20 heads of 2^20 features: 2^37 threads for one token. The pointers are not touched."""
    for heads, dim in [(1 << 20, 1 << 20), ((1 << 31) - 1, (1 << 31) - 1), (1 << 16, 1 << 18)]:
        d = Rotary(0, 0, 1, 1, heads, dim, 0, 0, 0, 64, (ctypes.c_int64 * 4)(0, 0, dim, 1), 64, None, None, 0, None, (ctypes.c_int64 * 2)(), 0)
        assert cabi.ormi_hip_rotary(ctypes.byref(d)) == 3 and b"heads * dim" in cabi.ormi_hip_last_error()


class AdamTensor(ctypes.Structure):
    _fields_ = [(n, ctypes.c_void_p) for n in ("p", "g", "out", "m", "v", "m_out", "v_out", "m_scale", "v_scale", "m_scale_out", "v_scale_out")] + [
        ("count", ctypes.c_int64), ("p_dtype", ctypes.c_int), ("g_dtype", ctypes.c_int)]


class Adam(ctypes.Structure):
    _fields_ = [("n", ctypes.c_int), ("tensors", ctypes.POINTER(AdamTensor)), ("bits", ctypes.c_int), ("step", ctypes.c_int64), ("lr", ctypes.c_double),
                ("b1", ctypes.c_double), ("b2", ctypes.c_double), ("eps", ctypes.c_double), ("decay", ctypes.c_double)]


def test_adamw_refuses_a_tensor_of_more_work_groups_than_a_launch(cabi):
    """2^24 work-groups of 256 threads and 2048 elements are 2^32 threads. The pointers are not touched."""
    for count in (((1 << 24) - 1) * 2048 + 1, 1 << 35, -1):
        t = AdamTensor(*[64] * 11, count, 0, 0)
        d = Adam(1, ctypes.pointer(t), 32, 1, 1e-3, 0.9, 0.999, 1e-8, 0.0)
        assert cabi.ormi_hip_adamw(ctypes.byref(d)) == 3 and b"count" in cabi.ormi_hip_last_error()


@pytest.mark.gpu
def test_the_gradient_of_more_rows_than_a_launch_takes(hip, ob):
    """2^28 queries and more of one feature over one key: 16 rows to a work-group would be 2^32 threads. The key's
    weight is 1, so dv is the number of rows and dq and dk are zero, all exactly."""
    from ormi_amd import Tensor, attention, realize_all

    rows = (1 << 28) + 64
    one = lambda x, **more: Tensor(np.full((1, 1, 1, 1), x, np.float32), "hip", dtype="bfloat16", **more)  # noqa: E731
    q, k, v = one(0.25, requires_grad=True), one(1.0, requires_grad=True), one(0.5, requires_grad=True)
    many = q.expand((1, rows, 1, 1))
    out = attention(many, k, v)
    (out * one(1.0).expand((1, rows, 1, 1))).sum().backward()
    size = (many.grad * many.grad).sum()
    realize_all(size, k.grad, v.grad)
    assert float(v.grad.numpy()[0, 0, 0, 0]) == 2.0 ** 28 and float(k.grad.numpy()[0, 0, 0, 0]) == 0.0 and float(size.numpy()) == 0.0
    del many, out, size, q, k, v
    ob.empty_cache()

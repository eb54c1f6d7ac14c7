"""Calls whose work-groups or threads would not fit one launch are cut into
launches that do, or refused before anything is read; none is cut short."""
import ctypes


class Rotary(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int), ("out_dtype", ctypes.c_int), ("batch", ctypes.c_int), ("length", ctypes.c_int), ("heads", ctypes.c_int),
                ("dim", ctypes.c_int), ("part", ctypes.c_int), ("interleaved", ctypes.c_int), ("inverse", ctypes.c_int), ("x", ctypes.c_void_p),
                ("x_strides", ctypes.c_int64 * 4), ("out", ctypes.c_void_p), ("cos", ctypes.c_void_p), ("sin", ctypes.c_void_p),
                ("table_rows", ctypes.c_int), ("positions", ctypes.c_void_p), ("positions_strides", ctypes.c_int64 * 2), ("offset", ctypes.c_int)]


def test_rotary_refuses_tokens_of_more_threads_than_a_launch(cabi):
    """2^20 heads of 2^20 features: 2^37 threads for one token. The pointers are not touched."""
    cabi.ormi_hip_rotary.argtypes = [ctypes.POINTER(Rotary)]
    for heads, dim in [(1 << 20, 1 << 20), ((1 << 31) - 1, (1 << 31) - 1), (1 << 16, 1 << 18)]:
        d = Rotary(0, 0, 1, 1, heads, dim, 0, 0, 0, 64, (ctypes.c_int64 * 4)(0, 0, dim, 1), 64, None, None, 0, None, (ctypes.c_int64 * 2)(), 0)
        assert cabi.ormi_hip_rotary(ctypes.byref(d)) == 3 and b"heads * dim" in cabi.ormi_hip_last_error()

"""Integer operands that are views (expanded, transposed) reach the kernels bit
for bit: document ids and code words past 2^24, which float32 does not hold,
rules of one value for the whole batch, and the C entry that copies a view."""
import ctypes

import numpy as np
import pytest

from attention_ref import assert_within, attention as ref

BIG = 1 << 24  # BIG and BIG + 1 are one float32


def ints(x):
    from ormi_amd import Tensor

    return Tensor(np.ascontiguousarray(x, dtype=np.int32), "hip", dtype="int32")


def operands(keys):
    rng = np.random.default_rng(keys)
    return [rng.standard_normal(s, dtype=np.float32) for s in ((2, keys, 2, 16), (2, keys, 1, 16), (2, keys, 1, 16))]


@pytest.mark.gpu
@pytest.mark.parametrize("view", ["expanded", "transposed"])
@pytest.mark.parametrize("keys", [30, 150])
def test_documents_that_are_views_keep_their_ids(hip, view, keys):
    from ormi_amd import Tensor, attention

    ids = np.where(np.arange(keys) < keys // 3, BIG, BIG + 1).astype(np.int32)
    if view == "expanded":
        host = np.stack([ids, ids])
        docs = ints(ids[None]).expand((2, keys))
    else:
        host = np.stack([ids, ids[::-1] + 1])
        docs = ints(host.T).transpose((1, 0))
    data = operands(keys)
    out = attention(*(Tensor(x, "hip") for x in data), causal=True, documents=docs)
    assert_within(out.numpy(), ref(*data, causal=True, documents=host)["out"], view)


@pytest.mark.gpu
def test_rules_of_one_value_for_the_batch(hip):
    from ormi_amd import Tensor, attention

    data = operands(40)
    t = [Tensor(x, "hip") for x in data]
    out = attention(*t, causal=True, prefix=ints([9]).expand((2,)), lengths=ints([33]).expand((2,)))
    want = ref(*data, causal=True, prefix=np.int32([9, 9]), lengths=np.int32([33, 33]))["out"]
    assert_within(out.numpy(), want, "prefix and lengths")


@pytest.mark.gpu
def test_code_words_that_are_views(hip):
    """A block whose words are one word expanded: 0x7f7e7d7c needs 31 bits."""
    from ormi_amd import AdamState8, Tensor

    bytes4 = np.uint8([0x7c, 0x7d, 0x7e, 0x7f])
    one = np.float32([0.5])
    want = AdamState8.from_codes((256,), np.tile(bytes4, 64).view(np.int8), one, np.tile(bytes4, 64), one).values()
    word = ints(bytes4.view(np.int32)).expand((64,))
    got = AdamState8((256,), (word, Tensor(one, "hip"), word, Tensor(one, "hip"))).values()
    for g, w in zip(got, want):
        assert np.array_equal(g.numpy(), w.numpy())


def copy_view(cabi, *args):
    cabi.ormi_hip_copy_view.argtypes = [ctypes.c_void_p, ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int, ctypes.POINTER(ctypes.c_int),
                                        ctypes.POINTER(ctypes.c_int64)]
    return cabi.ormi_hip_copy_view(*args)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", [np.uint8, np.uint16, np.uint32, np.uint64])
@pytest.mark.parametrize("shape,axes", [((), ()), ((7,), (0,)), ((5, 300), (1, 0)), ((3, 4, 5), (2, 0, 1)), ((2, 1, 3, 1, 2, 1, 2, 3), (7, 0, 6, 1, 5, 2, 4, 3))])
def test_a_view_is_copied_bit_for_bit(hip, cabi, kind, shape, axes):
    bits = np.random.default_rng(1).integers(0, np.iinfo(kind).max, shape, dtype=kind, endpoint=True)
    bits = np.asarray(bits, kind)
    view = bits.transpose(axes) if shape else bits
    want = np.ascontiguousarray(view)
    src, dst = ctypes.c_void_p(), ctypes.c_void_p()
    for p in (src, dst):
        assert cabi.ormi_hip_malloc(ctypes.byref(p), bits.nbytes) == 0
    assert cabi.ormi_hip_memcpy_h2d(src, bits.ctypes.data, bits.nbytes) == 0
    n = view.ndim
    strides = (ctypes.c_int64 * 8)(*(s // bits.itemsize for s in view.strides))
    assert copy_view(cabi, dst, src, bits.itemsize, n, (ctypes.c_int * 8)(*view.shape), strides) == 0, cabi.ormi_hip_last_error()
    got = np.empty_like(want)
    assert cabi.ormi_hip_memcpy_d2h(got.ctypes.data, dst, got.nbytes) == 0
    assert np.array_equal(got, want)
    for p in (src, dst):
        cabi.ormi_hip_free(p)


def test_the_copy_refuses(cabi):
    """Arguments are checked before the device is touched."""
    buf = (ctypes.c_char * 64)()
    shape, strides = (ctypes.c_int * 8)(2, 2), (ctypes.c_int64 * 8)(2, 1)
    for dst, src, size, ndim, sh, st, message in [
            (None, buf, 4, 2, shape, strides, b"null"), (buf, None, 4, 2, shape, strides, b"null"), (buf, buf, 3, 2, shape, strides, b"element size"),
            (buf, buf, 4, 9, shape, strides, b"dimensions"), (buf, buf, 4, -1, shape, strides, b"dimensions"), (buf, buf, 4, 2, None, strides, b"null"),
            (buf, buf, 4, 2, (ctypes.c_int * 8)(2, -1), strides, b"negative")]:
        assert copy_view(cabi, dst, src, size, ndim, sh, st) == 3 and message in cabi.ormi_hip_last_error(), message
    assert copy_view(cabi, None, None, 4, 2, (ctypes.c_int * 8)(2, 0), strides) == 0  # nothing to copy

"""Attention and its gradient on the GPU against the formula in 64 bits
(attention_ref.py derives the bounds), and its refusals."""
import ctypes
import math

import numpy as np
import pytest

from attention_ref import assert_within, attention as ref

DTYPES = ["float32", "bfloat16", "float16"]


def rounded(x, dtype):
    """x as the dtype holds it, in float32."""
    from ormi_amd import Tensor

    return Tensor(x, "hip", dtype=dtype).numpy()


def run(case, dtype, grad=True, wrap=lambda t: t):
    """(results by name, references by name) for a dict of host arrays and options."""
    from ormi_amd import Tensor, attention, realize_all

    data = {n: rounded(case[n], dtype) for n in ("q", "k", "v")}
    leaves = {n: Tensor(x, "hip", requires_grad=grad, dtype=dtype) for n, x in data.items()}
    rules = {n: Tensor(case[n], "hip", dtype=str(case[n].dtype)) for n in ("slopes", "documents", "prefix", "lengths") if n in case}
    options = {n: case[n] for n in ("causal", "scale", "cap") if n in case}
    out = attention(*(wrap(leaves[n]) for n in "qkv"), **options, **rules)
    got = {}
    host = {n: case[n] for n in ("slopes", "documents", "prefix", "lengths") if n in case}
    if grad:
        rng = np.random.default_rng(77)
        w = rounded(rng.standard_normal(out.shape, dtype=np.float32) * np.float32(case.get("dout", 1.0)), dtype)
        (out * Tensor(w, "hip", dtype=dtype)).sum().backward()
        grads = [leaves[n].grad for n in "qkv"]
        realize_all(out, *grads)
        got = {"d" + n: g.numpy() for n, g in zip("qkv", grads)}
        for n, g in zip("qkv", grads):
            assert g.dtype == dtype, n
    got["out"] = out.numpy()
    assert out.dtype == dtype
    return got, data, host, options, (w if grad else None)


def check(case, dtype, grad=True):
    got, data, host, options, w = run(case, dtype, grad)
    want = ref(data["q"], data["k"], data["v"], w, dtype=dtype, **options, **host)
    for n in want:
        assert_within(got[n], want[n], f"{n} ({dtype})")
    return got


def make(b, lq, lk, heads, kvh, d, seed=0, size=1.0, **options):
    rng = np.random.default_rng(seed)
    f = lambda *s: rng.standard_normal(s, dtype=np.float32) * np.float32(size)  # noqa: E731
    return {"q": f(b, lq, heads, d), "k": f(b, lk, kvh, d), "v": f(b, lk, kvh, d), **options}


def packed(b, lk, docs, tail, seed=3):
    rng = np.random.default_rng(seed)
    ids = np.zeros((b, lk), np.int32)
    for i in range(b):
        ids[i] = np.searchsorted(np.sort(rng.integers(0, lk, docs - 1)), np.arange(lk), side="right")
        if tail:
            ids[i, lk - tail:] = -1
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1, 1), (1, 2, 3, 1, 1, 7), (2, 33, 33, 2, 2, 64), (1, 64, 65, 4, 2, 33), (2, 130, 130, 6, 2, 128),
                                   (1, 129, 257, 3, 1, 80), (1, 40, 40, 2, 2, 256), (1, 70, 90, 1, 1, 130), (1, 5, 300, 8, 1, 96)])
@pytest.mark.parametrize("causal", [False, True])
def test_sizes(hip, dtype, shape, causal):
    check(make(*shape, seed=sum(shape), causal=causal), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rule", ["cap", "slopes", "cap_slopes", "prefix", "documents", "documents_bidirectional", "lengths", "lengths_causal"])
@pytest.mark.parametrize("dim", [64, 72, 256])
def test_rules(hip, dtype, rule, dim):
    c = make(2, 150, 150, 4, 2, dim, seed=dim)
    slopes = np.float32(2.0) ** -np.arange(1, 5, dtype=np.float32)
    if "cap" in rule:
        c.update(cap=3.0, causal=True)
    if "slopes" in rule:
        c.update(slopes=slopes)
    if rule == "prefix":
        c.update(causal=True, prefix=np.array([0, 97], np.int32))
    if "documents" in rule:
        c.update(documents=packed(2, 150, 4, 9), causal=rule == "documents")
    if "lengths" in rule:
        c.update(lengths=np.array([150, 151 - 64], np.int32), causal=rule == "lengths_causal")
    check(c, dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("queries,keys,heads,kvh,dim", [(1, 1, 4, 4, 64), (1, 700, 8, 2, 64), (1, 2049, 7, 1, 128), (3, 1000, 8, 1, 80), (2, 513, 4, 4, 256),
                                                        (1, 5000, 32, 8, 128)])
def test_single_tokens_over_a_cache(hip, dtype, queries, keys, heads, kvh, dim):
    """Few rows, many keys: the keys are split over work-groups and joined."""
    rng = np.random.default_rng(keys)
    lengths = rng.integers(queries, keys + 1, 3).astype(np.int32)
    check(make(3, queries, keys, heads, kvh, dim, seed=keys, causal=True, lengths=lengths), dtype, grad=False)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_long_rows_join_in_order(hip, dtype):
    """Rows that need several splits forward and backward (one key head, many rows)."""
    c = make(1, 600, 600, 8, 1, 64, seed=5, causal=True)
    a, b = check(c, dtype), run(c, dtype)[0]
    for n in a:
        assert np.array_equal(a[n], b[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_rows_that_see_nothing(hip, dtype, causal):
    """No key at all, a length below the queries' number, tokens of no document: zeros, and finite gradients."""
    c = make(4, 40, 50, 2, 1, 64, seed=9, causal=causal, lengths=np.array([0, 1, 25, 50], np.int32))
    got = check(c, dtype)
    assert not got["out"][0].any() and not got["dq"][0].any() and not got["dk"][0].any() and not got["dv"][0].any()
    docs = packed(4, 50, 3, 0)
    docs[1] = -1
    docs[2, ::3] = -7
    docs[3, 10:] = np.arange(40)
    got = check(make(4, 40, 50, 2, 1, 64, seed=10, causal=causal, documents=docs), dtype)
    assert not got["out"][1].any() and not got["dk"][1].any()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("form", [{}, {"cap": 3.0}, {"slopes": np.float32([0.5, 0.25])}])
@pytest.mark.parametrize("dim", [24, 64, 96, 128, 256])
def test_few_keys_leave_one_rounding(hip, dtype, form, dim):
    """Rows that see few keys keep what rounding leaves of their weights and score gradients: every value is one
    rounding to its type (h of it; half a step below its normal range) beside float32's sums and second-order terms,
    h of what all roundings to the type would allow, twice for weight and score gradient."""
    case = make(2, 16, 20, 2, 1, dim, seed=31, causal=True, **form)
    got, data, host, options, w = run(case, dtype)
    coarse = ref(data["q"], data["k"], data["v"], w, dtype=dtype, **options, **host)
    fine = ref(data["q"], data["k"], data["v"], w, dtype="float32", **options, **host)
    h = {"bfloat16": 2.0 ** -8, "float16": 2.0 ** -11}[dtype]
    least = {"bfloat16": 2.0 ** -134, "float16": 2.0 ** -25}[dtype]
    for n, (exact, bound) in fine.items():
        assert_within(got[n], (exact, bound + h * np.abs(exact) + 2 * h * coarse[n][1] + least), f"{n} ({dtype})")


@pytest.mark.gpu
def test_no_keys_and_no_queries(hip):
    from ormi_amd import Tensor, attention

    q = Tensor(np.ones((2, 3, 2, 8), np.float32), "hip", requires_grad=True)
    k = Tensor(np.ones((2, 0, 2, 8), np.float32), "hip", requires_grad=True)
    out = attention(q, k, k)
    out.sum().backward()
    assert not out.numpy().any() and not q.grad.numpy().any() and k.grad.shape == (2, 0, 2, 8)
    empty = attention(Tensor(np.ones((2, 0, 2, 8), np.float32), "hip"), q, q)
    assert empty.numpy().shape == (2, 0, 2, 8)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_past_the_length_are_not_read(hip, dtype):
    c = make(2, 3, 200, 4, 2, 64, seed=4, causal=True, lengths=np.array([77, 130], np.int32))
    want = check(dict(c), dtype)
    for n in "kv":
        c[n][0, 77:] = np.nan
        c[n][1, 130:] = np.inf
    got = run(c, dtype)[0]
    for n in want:
        assert np.array_equal(got[n], want[n]), n


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
@pytest.mark.parametrize("form", ["plain", "slopes", "cap"])
def test_masked_tokens_may_hold_anything(hip, dtype, dim, form):
    """Padding tokens (no document) whose q, k, v and dout are NaN or infinite: the others' results are those
    with zeros there, and theirs are zeros."""
    docs = packed(2, 140, 3, 13)
    docs[1, 50:55] = -2
    c = make(2, 140, 140, 4, 2, dim, seed=dim, causal=True, documents=docs)
    if form == "slopes":
        c["slopes"] = np.float32([0.5, 0.3, 0.2, 0.0])
    if form == "cap":
        c["cap"] = 4.0
    pad = docs < 0
    for n in "qkv":
        c[n][pad] = 0
    w = rounded(np.random.default_rng(3).standard_normal(c["q"].shape, dtype=np.float32), dtype)
    w[pad] = 0
    data = {n: rounded(c[n], dtype) for n in "qkv"}
    rules = {n: c[n] for n in ("causal", "documents", "slopes", "cap") if n in c}
    want = ref(data["q"], data["k"], data["v"], w, dtype=dtype, **rules)
    for n in "qkv":
        data[n][pad] = np.nan if n != "v" else np.inf
    w[pad] = np.nan
    from ormi_amd import Tensor, attention, realize_all

    leaves = {n: Tensor(x, "hip", requires_grad=True, dtype=dtype) for n, x in data.items()}
    given = {n: Tensor(v, "hip", dtype=str(v.dtype)) if isinstance(v, np.ndarray) else v for n, v in rules.items()}
    out = attention(leaves["q"], leaves["k"], leaves["v"], **given)
    (out * Tensor(w, "hip", dtype=dtype)).sum().backward()
    grads = [leaves[n].grad for n in "qkv"]
    realize_all(out, *grads)
    for n, t in zip(("out", "dq", "dk", "dv"), (out, *grads)):
        got = t.numpy()
        assert not got[pad].any(), n
        assert_within(got, want[n], f"{n} ({dtype})")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,keys,heads", [(90, 90, 2), (5, 700, 8)])
def test_later_tokens_reach_no_earlier_row(hip, dtype, rows, keys, heads):
    """A causal token that is NaN or infinite in v or k: rows before it are those without it (with few rows the
    keys are split over work-groups), rows from it on are not finite."""
    c = make(1, rows, keys, heads, 1, 64, seed=30, causal=True)
    at = keys - 3
    want = run(c, dtype, grad=False)[0]["out"]
    for n, bad in (("v", np.inf), ("v", np.nan), ("k", np.nan)):
        hurt = {**c, n: c[n].copy()}
        hurt[n][0, at] = bad
        got = run(hurt, dtype, grad=False)[0]["out"]
        data = {n: rounded(c[n], dtype) for n in "qkv"}
        exact, bound = ref(data["q"], data["k"], data["v"], dtype=dtype, causal=True)["out"]
        assert_within(got[:, :-3], (exact[:, :-3], bound[:, :-3]), n)
        assert not np.isfinite(got[:, -3:]).any()
    assert np.isfinite(want).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
def test_what_is_seen_is_not_hidden(hip, dtype, causal):
    """An infinity that a row sees stands in its feature and in no other; NaN everywhere stays NaN everywhere."""
    case = make(1, 300, 300, 2, 1, 64, seed=41, causal=causal)
    case["v"][0, 0, 0, 5] = np.inf
    got = run(case, dtype, grad=False)[0]["out"]
    assert (got[..., 5] == np.inf).all() and np.isfinite(np.delete(got, 5, axis=-1)).all()
    for name in "qkv":
        case[name] = np.full_like(case[name], np.nan)
    got = run(case, dtype)[0]
    assert all(np.isnan(np.asarray(g, np.float32)).all() for g in got.values())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("size,scale", [(30.0, 1.0), (1.0, -0.4), (1.0, 0.0), (0.01, None)])
def test_scores_large_reversed_and_flat(hip, dtype, size, scale):
    check(make(1, 100, 140, 2, 1, 64, seed=8, size=size, causal=True, scale=scale), dtype)


@pytest.mark.gpu
def test_small_losses_keep_float16_gradients(hip):
    """Gradients of a loss of 2^-13: the score gradients would be far below float16's normal range."""
    check(make(1, 200, 200, 2, 2, 64, seed=12, causal=True, dout=2.0 ** -13), "float16")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 24, 33])
def test_views_of_other_orders(hip, dtype, dim):
    """Heads before tokens, and features outermost, as transposed views."""
    c = make(2, 50, 50, 2, 2, dim, seed=2, causal=True)
    want = run(c, dtype)[0]
    for order in [(0, 2, 1, 3), (3, 1, 2, 0)]:
        turned = {**c, **{n: np.ascontiguousarray(c[n].transpose(order)) for n in "qkv"}}
        got = run(turned, dtype, wrap=lambda t: t.transpose(order))[0]
        assert np.array_equal(got["out"], want["out"])
        for n in ("dq", "dk", "dv"):
            assert np.array_equal(got[n].transpose(order), want[n]), n


@pytest.mark.gpu
def test_broadcast_keys_sum_their_gradients(hip):
    """Keys and values expanded over the batch: their gradients add up over it."""
    from ormi_amd import Tensor, attention

    c = make(3, 20, 30, 2, 2, 32, seed=6)
    k, v = (Tensor(c[n][:1], "hip", requires_grad=True) for n in "kv")
    q = Tensor(c["q"], "hip", requires_grad=True)
    out = attention(q, k.expand((3, 30, 2, 32)), v.expand((3, 30, 2, 32)))
    w = np.random.default_rng(1).standard_normal(out.shape, dtype=np.float32)
    (out * Tensor(w, "hip")).sum().backward()
    want = ref(c["q"], np.repeat(c["k"][:1], 3, 0), np.repeat(c["v"][:1], 3, 0), w)
    assert_within(out.numpy(), want["out"], "out")
    for name, t in (("dk", k), ("dv", v)):
        exact, bound = want[name]
        assert_within(t.grad.numpy(), (exact.sum(0, keepdims=True), bound.sum(0, keepdims=True) + 3 * 2.0 ** -24 * np.abs(exact).sum(0, keepdims=True)), name)


@pytest.mark.gpu
def test_gradient_against_differences(hip):
    """Central differences of the 64-bit formula's loss, at some elements of q, k and v."""
    c = make(1, 24, 24, 4, 2, 16, seed=21, causal=True, cap=2.0, slopes=np.float32([0.5, 0.25, 0.1, 0.0]), prefix=np.array([9], np.int32))
    got, data, host, options, w = run(c, "float32")
    rng = np.random.default_rng(5)
    for name in "qkv":
        for _ in range(6):
            at = tuple(int(rng.integers(n)) for n in data[name].shape)
            loss = []
            for step in (1e-4, -1e-4):
                moved = {n: data[n].astype(np.float64) for n in "qkv"}
                moved[name][at] += step
                loss.append((ref(moved["q"], moved["k"], moved["v"], **options, **host)["out"][0] * w).sum())
            slope = (loss[0] - loss[1]) / 2e-4
            # third derivatives of order 10 times step^2 / 6, 64-bit noise 1e-12 / step, float32 noise
            assert abs(got["d" + name][at] - slope) <= 1e-6 + 2e-5 * abs(slope), (name, at)


@pytest.mark.gpu
def test_gradient_of_only_some_operands(hip):
    from ormi_amd import Tensor, attention

    c = make(1, 40, 40, 2, 1, 32, seed=14, causal=True)
    full = run(c, "float32")[0]
    w = np.random.default_rng(77).standard_normal(c["q"].shape, dtype=np.float32)
    for name in "qkv":
        t = {n: Tensor(c[n], "hip", requires_grad=n == name) for n in "qkv"}
        (attention(t["q"], t["k"], t["v"], causal=True) * Tensor(w, "hip")).sum().backward()
        assert np.array_equal(t[name].grad.numpy(), full["d" + name]), name


@pytest.mark.gpu
def test_offsets_past_32_bits(hip, cabi):
    """A cache whose batches lie more than 2^32 bytes apart, and one whose tokens
    lie 2^31 bytes apart (read through a packed copy), by the C entry."""
    class Desc(ctypes.Structure):
        _fields_ = [("dtype", ctypes.c_int), ("batch", ctypes.c_int), ("queries", ctypes.c_int), ("keys", ctypes.c_int),
                    ("heads", ctypes.c_int), ("kv_heads", ctypes.c_int), ("dim", ctypes.c_int), ("q", ctypes.c_void_p),
                    ("k", ctypes.c_void_p), ("v", ctypes.c_void_p), ("q_strides", ctypes.c_int64 * 4), ("k_strides", ctypes.c_int64 * 4),
                    ("v_strides", ctypes.c_int64 * 4), ("scale", ctypes.c_float), ("cap", ctypes.c_float), ("causal", ctypes.c_int),
                    ("slopes", ctypes.c_void_p), ("documents", ctypes.c_void_p), ("documents_batch_stride", ctypes.c_int64),
                    ("prefix", ctypes.c_void_p), ("lengths", ctypes.c_void_p), ("out", ctypes.c_void_p), ("rest", ctypes.c_void_p), ("lse", ctypes.c_void_p),
                    ("workspace", ctypes.c_void_p), ("workspace_bytes", ctypes.c_size_t)]

    cabi.ormi_hip_attention.argtypes = [ctypes.POINTER(Desc)]
    cabi.ormi_hip_attention_workspace_size.argtypes = [ctypes.POINTER(Desc), ctypes.POINTER(ctypes.c_size_t)]
    c = make(2, 1, 3, 2, 1, 64, seed=1)
    want = ref(c["q"], c["k"], c["v"])["out"]

    def malloc(n):
        p = ctypes.c_void_p()
        assert cabi.ormi_hip_malloc(ctypes.byref(p), n) == 0
        return p

    small = [malloc(c["q"].nbytes), malloc(c["q"].nbytes)]
    assert cabi.ormi_hip_memcpy_h2d(small[0], c["q"].ctypes.data, c["q"].nbytes) == 0
    for batch_stride, token_stride in [((1 << 30) + 64, 64), (64, 1 << 29)]:
        reach = 4 * (batch_stride + 2 * token_stride + 64)
        big = malloc(reach)
        for name in "kv":
            src = c[name]
            # k and v share the block: v 64 floats after k in each row's reach when rows are far apart
            shift = 0 if name == "k" else 0
            block = big if name == "k" else malloc(reach)
            if name == "v":
                vbig = block
            for b in range(2):
                for j in range(3):
                    row = np.ascontiguousarray(src[b, j, 0])
                    at = block.value + 4 * (b * batch_stride + j * token_stride + shift)
                    assert cabi.ormi_hip_memcpy_h2d(ctypes.c_void_p(at), row.ctypes.data, row.nbytes) == 0
        strides = (ctypes.c_int64 * 4)(batch_stride, token_stride, 64, 1)
        d = Desc(0, 2, 1, 3, 2, 1, 64, small[0], big, vbig, (ctypes.c_int64 * 4)(128, 128, 64, 1), strides, strides, 1 / 8, 0.0, 0, None, None, 0,
                 None, None, small[1], None, None, None, 0)
        n = ctypes.c_size_t()
        assert cabi.ormi_hip_attention_workspace_size(ctypes.byref(d), ctypes.byref(n)) == 0
        ws = malloc(max(n.value, 1))
        d.workspace, d.workspace_bytes = ws, n.value
        assert cabi.ormi_hip_attention(ctypes.byref(d)) == 0, cabi.ormi_hip_last_error()
        out = np.empty(c["q"].shape, np.float32)
        assert cabi.ormi_hip_memcpy_d2h(out.ctypes.data, small[1], out.nbytes) == 0
        assert_within(out, want, f"strides {batch_stride}, {token_stride}")
        for p in (big, vbig, ws):
            cabi.ormi_hip_free(p)
    for p in small:
        cabi.ormi_hip_free(p)


# ---------------------------------------------------------------- refusals --
def tensors(dev, q=(2, 5, 4, 8), k=(2, 6, 2, 8), v=None, dtype="float32"):
    from ormi_amd import Tensor

    return [Tensor(np.zeros(s, np.float32), dev, dtype=dtype) for s in (q, k, v or k)]


@pytest.mark.parametrize("shapes,message", [
    (dict(q=(2, 5, 4)), "batch, length, heads, features"), (dict(v=(2, 6, 2, 9)), "one shape"), (dict(k=(3, 6, 2, 8)), "one batch"),
    (dict(q=(2, 5, 4, 9)), "as many features"), (dict(q=(2, 5, 5, 8)), "multiples of the key heads"),
    (dict(q=(2, 5, 2, 257), k=(2, 6, 2, 257)), "1 to 256"), (dict(dtype="int32"), "of one type")])
def test_refuses_shapes(cpu, shapes, message):
    from ormi_amd import attention

    with pytest.raises(RuntimeError, match=message):
        attention(*tensors(cpu, **shapes))


def test_refuses_rules(cpu):
    from ormi_amd import Tensor, attention

    t = tensors(cpu)
    ints = lambda *s: Tensor(np.zeros(s, np.int32), cpu, dtype="int32")  # noqa: E731
    with pytest.raises(RuntimeError, match="prefix with causal"):
        attention(*t, prefix=ints(2))
    with pytest.raises(RuntimeError, match="documents .* another shape"):
        attention(*t, documents=ints(2, 5))
    with pytest.raises(RuntimeError, match="lengths .*as int32"):
        attention(*t, lengths=Tensor(np.zeros(2, np.float32), cpu))
    with pytest.raises(RuntimeError, match="no gradient for slopes"):
        attention(*t, slopes=Tensor(np.zeros(4, np.float32), cpu, requires_grad=True))
    with pytest.raises(RuntimeError, match="cap"):
        attention(*t, cap=-1.0)
    with pytest.raises(RuntimeError, match="finite scale"):
        attention(*t, scale=math.inf)
    with pytest.raises(TypeError):
        attention(*t, lengths=np.zeros(2, np.int32))
    with pytest.raises(RuntimeError, match="one type"):
        attention(t[0], *tensors(cpu, dtype="bfloat16")[1:])


def test_c_entry_refuses_without_a_gpu(cabi):
    """Descriptors are checked before the device is touched."""
    assert cabi.ormi_hip_attention(None) == 3 and b"null descriptor" in cabi.ormi_hip_last_error()
    assert cabi.ormi_hip_attention_grad(None) == 3
    buf = (ctypes.c_char * 1024)()  # all zero: no heads
    assert cabi.ormi_hip_attention(ctypes.byref(buf)) == 3 and b"heads" in cabi.ormi_hip_last_error()

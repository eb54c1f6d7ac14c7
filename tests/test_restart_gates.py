"""A token that starts from nothing takes no part of what its value gate holds."""
import numpy as np
import pytest

import recurrent_ref as ref
from test_recurrence import documents_of, tensor, values


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
@pytest.mark.parametrize("dtype,gate_dtype", [("float32", "float32"), ("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float16", "float16")])
@pytest.mark.parametrize("shape", [(2, 40, 9), (3, 900, 24), (520, 300, 5)])  # one tile; tiles that wait for one another; tiles in turn
def test_value_gates_at_a_documents_first_token(hip, shape, dtype, gate_dtype, bad):
    from ormi_amd import linear_recurrence, realize_all

    batch, length, channels = shape
    rng = np.random.default_rng(6)
    docs = documents_of(batch, length, 5, rng, padding=0)
    docs[:, 9:11] = 77  # restarts inside a segment of 8 tokens
    first = np.zeros((batch, length), bool)
    first[:, 1:] = docs[:, 1:] != docs[:, :-1]
    g, x = values(shape, False, rng)
    w = rng.standard_normal(shape).astype(np.float32)
    h0, wl = rng.standard_normal((2, batch, channels)).astype(np.float32)
    g[first] = bad
    g, x, w = tensor(g, gate_dtype, True), tensor(x, dtype, True), tensor(w, dtype)
    h0, wl = tensor(h0, grad=True), tensor(wl)
    y, last = linear_recurrence(g, x, h0, documents=tensor(docs, "int32"))
    ((y * w).sum() + (last * wl).sum()).backward()
    realize_all(y, last, g.grad, x.grad, h0.grad)
    clean = np.where(first[..., None], np.float32(0.5), g.numpy())
    want, bound = ref.recurrence(clean, x.numpy(), False, h0.numpy(), docs, None, w.numpy(), wl.numpy())
    for name, t, kind in (("y", y, dtype), ("last", last, "float32"), ("dg", g.grad, gate_dtype), ("dx", x.grad, dtype), ("dinitial", h0.grad, "float32")):
        ref.close(t.numpy(), want[name], bound[name], kind, name)

"""Gradients that one call fills together, where that call is refused: each of them raises, none is memory that nothing wrote."""
import numpy as np
import pytest


@pytest.mark.gpu
def test_a_refused_gradient_leaves_none_behind(hip):
    """One token of 32768 heads: the attention takes it, but its gradient's copy of a transposed dout would pass the 2^31
    bytes of a tile's offsets, and is refused. With a contiguous one the same call gives the gradients."""
    from ormi_amd import Tensor, attention, ormi_backend, realize_all

    heads, dim = 32768, 256
    rng = np.random.default_rng(1)
    x = rng.standard_normal((1, 1, heads, dim)).astype(np.float32)
    w = rng.standard_normal((1, 1, heads, dim)).astype(np.float32)
    kv = rng.standard_normal((2, 1, 1, 1, dim)).astype(np.float32)
    q, k, v = (Tensor(t, "hip", requires_grad=True) for t in (x, *kv))
    y = attention(q, k, v, causal=False)
    turned = Tensor(np.ascontiguousarray(w.transpose(0, 1, 3, 2)), "hip").transpose([0, 1, 3, 2])
    turned.realize()
    y._node.grad = turned._node
    ormi_backend.compute_gradients(y._node)
    for t in (k, v, q, v, k, q):
        with pytest.raises(RuntimeError, match="heads \\* dim too large"):
            t.grad.numpy()
    for t in (q, k, v):
        t.zero_grad()
    y._node.grad = Tensor(w, "hip")._node
    ormi_backend.compute_gradients(y._node)
    realize_all(*(t.grad for t in (q, k, v)))
    # of one key: every weight is 1, so dv is the sum of dout and dq and dk are zero, up to the roundings of
    # dout . v, which cancels: 256 products, held to 300 u of their size at most 6^2 * 256 each, over 32768 rows
    u = 2.0 ** -24
    total = w.astype(np.float64).sum((0, 1, 2))
    assert np.abs(v.grad.numpy()[0, 0, 0] - total).max() <= heads * u * np.abs(w).sum((0, 1, 2)).max()
    slack = 300 * u * np.abs(w).max() * np.abs(kv[1]).max() * dim
    assert np.abs(q.grad.numpy()).max() <= slack * np.abs(kv[0]).max()
    assert np.abs(k.grad.numpy()).max() <= slack * np.abs(x).max() * heads

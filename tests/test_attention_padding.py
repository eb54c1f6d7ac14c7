"""Widths that are no tile's: what a tile holds past a row's features is zero, so
that an infinity among the features meets no product of its own with the padding.
A key that every query sees with a score of minus infinity has weight zero: the
results are those without it, at every width."""
import numpy as np
import pytest

from attention_ref import assert_within, attention as ref
from test_attention import DTYPES, make, rounded

WIDTHS = [24, 40, 64, 72, 80, 96, 100, 104, 128, 136, 168, 200, 256]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", WIDTHS)
@pytest.mark.parametrize("queries,keys,heads", [(70, 70, 2), (1, 300, 4)])
def test_a_score_of_minus_infinity_weighs_nothing(hip, dtype, dim, queries, keys, heads):
    from ormi_amd import Tensor, attention, realize_all

    c = make(1, queries, keys, heads, 1, dim, seed=dim)
    c["q"][..., 0] = -np.abs(c["q"][..., 0]) - np.float32(0.25)
    data = {n: rounded(c[n], dtype) for n in "qkv"}
    w = rounded(np.random.default_rng(2).standard_normal(c["q"].shape, dtype=np.float32), dtype)
    at = 5
    others = np.delete(np.arange(keys), at)
    want = ref(data["q"], data["k"][:, others], data["v"][:, others], w, dtype=dtype)
    data["k"][0, at, 0, 0] = np.inf
    t = {n: Tensor(data[n], "hip", requires_grad=True, dtype=dtype) for n in "qkv"}
    out = attention(t["q"], t["k"], t["v"])
    (out * Tensor(w, "hip", dtype=dtype)).sum().backward()
    grads = [t[n].grad for n in "qkv"]
    realize_all(out, *grads)
    dq, dk, dv = (g.numpy() for g in grads)
    assert_within(out.numpy(), want["out"], "out")
    assert_within(dv[:, others], want["dv"], "dv")
    assert_within(dk[:, others], want["dk"], "dk")
    assert not dv[:, at].any() and not dk[:, at].any()
    exact, bound = want["dq"]  # zero times the infinity itself is the first feature's own
    assert_within(dq[..., 1:], (exact[..., 1:], bound[..., 1:]), "dq")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", WIDTHS)
def test_an_infinite_value_stands_in_its_feature(hip, dtype, dim):
    from ormi_amd import Tensor, attention

    c = make(1, 150, 150, 2, 1, dim, seed=dim)
    c["v"][0, 0, 0, 5] = np.inf
    out = attention(*(Tensor(c[n], "hip", dtype=dtype) for n in "qkv"), causal=True).numpy()
    assert (out[..., 5] == np.inf).all() and np.isfinite(np.delete(out, 5, axis=-1)).all()

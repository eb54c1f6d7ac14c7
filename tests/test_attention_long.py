"""Paths that only longer calls reach: documents over more than one window of
64 ranges (4096 keys) and of 64 tiles of rows (2048 rows), documents with splits
and with key lengths, slopes steep enough for tiles without any weight."""
import numpy as np
import pytest

from attention_ref import assert_within, attention as ref
from test_attention import DTYPES, check, make, packed, rounded


def few_long(b, keys, cuts, tail=0):
    ids = np.zeros((b, keys), np.int32)
    for i in range(b):
        ids[i] = np.searchsorted(np.array(cuts[i]), np.arange(keys), side="right")
    if tail:
        ids[:, keys - tail:] = -1
    return ids


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("rows", [2200, 300])
def test_documents_past_a_window_of_ranges(hip, dtype, causal, rows):
    """4600 keys: the first document goes to key 4200, the second to 4300, the third has the rest and no padding;
    rows are the last of the sequence. Keys are split over work-groups forward and in dq, rows in dk and dv."""
    docs = few_long(1, 4600, [[4200, 4300]])
    check(make(1, rows, 4600, 1, 1, 32, seed=rows, causal=causal, documents=docs), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("dim", [64, 256])
def test_one_document_over_several_windows(hip, dtype, dim):
    """9000 keys, all but 70 of one document, shared key heads, few rows."""
    docs = few_long(2, 9000, [[30, 8960], [8990]])
    check(make(2, 70, 9000, 4, 2, dim, seed=dim, causal=True, documents=docs), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_document_runs_that_come_again(hip, dtype):
    """The same id far apart, with others between: the tiles between are passed over."""
    docs = np.repeat(np.int32([4, 1, 4, 2, -1, 4]), [900, 1000, 60, 1100, 40, 1500])[None]
    check(make(1, 2100, 4600, 1, 1, 32, seed=6, causal=True, documents=docs), dtype)
    check(make(1, 4, 4600, 8, 1, 64, seed=7, documents=docs), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,dim", [(150, 64), (40, 80), (1, 128)])
def test_documents_and_lengths(hip, dtype, causal, queries, dim):
    docs = packed(4, 150, 4, 9)
    lengths = np.array([150, 97, 1, 0], np.int32)
    got = check(make(4, queries, 150, 4, 2, dim, seed=dim, causal=causal, documents=docs, lengths=lengths), dtype)
    assert not any(got[n][3].any() for n in got)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("queries,keys,heads", [(1000, 1000, 2), (5, 1500, 8), (40, 1200, 2)])
@pytest.mark.parametrize("lengths", [False, True])
def test_steep_slopes(hip, dtype, causal, queries, keys, heads, lengths):
    """Slopes of 4 to 1/4: from 40 to 600 keys away the weights are below float32's least."""
    slopes = np.float32(2.0) ** np.linspace(2, -2, heads, dtype=np.float32)
    more = {"lengths": np.array([keys - 333, keys], np.int32)} if lengths else {}
    check(make(2, queries, keys, heads, 1, 64, seed=keys, causal=causal, slopes=slopes.astype(np.float32), **more), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_steep_slopes_and_documents(hip, dtype):
    docs = few_long(1, 1300, [[500, 505]], tail=20)
    check(make(1, 700, 1300, 2, 2, 96, seed=8, causal=True, documents=docs, slopes=np.float32([3.0, 0.5])), dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_slopes_past_two_to_the_24(hip, dtype):
    """Positions that float32 does not hold: distances are exact all the same. The weights reach back some 300
    keys; of the keys before the last 1024 the gradients are zero."""
    from ormi_amd import Tensor, attention, realize_all

    keys, near = (1 << 24) + 1041, 1024
    slopes = np.float32([0.5, 1.0])
    c = make(1, 5, near, 2, 1, 8, seed=3)
    data = {n: rounded(c[n], dtype) for n in "qkv"}
    w = rounded(np.random.default_rng(4).standard_normal(c["q"].shape, dtype=np.float32), dtype)
    want = ref(data["q"], data["k"], data["v"], w, dtype=dtype, causal=True, slopes=slopes)
    t = {}
    for n in "kv":
        whole = np.zeros((1, keys, 1, 8), np.float32)
        whole[:, keys - near:] = data[n]
        t[n] = Tensor(whole, "hip", requires_grad=True, dtype=dtype)
    q = Tensor(data["q"], "hip", requires_grad=True, dtype=dtype)
    out = attention(q, t["k"], t["v"], causal=True, slopes=Tensor(slopes, "hip"))
    (out * Tensor(w, "hip", dtype=dtype)).sum().backward()
    realize_all(out, q.grad, t["k"].grad, t["v"].grad)
    assert_within(out.numpy(), want["out"], "out")
    assert_within(q.grad.numpy(), want["dq"], "dq")
    for n in "kv":
        g = t[n].grad.numpy()
        assert_within(g[:, keys - near:], want["d" + n], "d" + n)
        assert not g[:, : keys - near].any(), n

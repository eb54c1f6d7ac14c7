"""float16 score gradients are held times a power of two taken from dout and v.
What stands at positions that reach no result does not move it, nor does another
sequence or key head: gradients of losses of 2^-20 against the formula in 64 bits.

q and k are 2^6 times unequal, so that the gradient of the one with the small
values is far above float16's least numbers while the score gradients are not."""
import numpy as np
import pytest

from attention_ref import assert_within, attention as ref
from test_attention import make, packed, rounded


def gradients(data, w, **rules):
    from ormi_amd import Tensor, attention, realize_all

    leaves = {n: Tensor(data[n], "hip", requires_grad=True, dtype="float16") for n in "qkv"}
    given = {n: Tensor(x, "hip", dtype=str(x.dtype)) if isinstance(x, np.ndarray) else x for n, x in rules.items()}
    out = attention(*(leaves[n] for n in "qkv"), **given)
    (out * Tensor(w, "hip", dtype="float16")).sum().backward()
    grads = [leaves[n].grad for n in "qkv"]
    realize_all(out, *grads)
    return {n: t.numpy() for n, t in zip(("out", "dq", "dk", "dv"), (out, *grads))}


def case(b, lq, lk, heads, kvh, d, large, seed, loss=2.0 ** -20):
    c = make(b, lq, lk, heads, kvh, d, seed=seed)
    for n in "qk":
        c[n] *= np.float32(64.0 if n == large else 1 / 64)
    data = {n: rounded(c[n], "float16") for n in "qkv"}
    return data, rounded(np.random.default_rng(seed + 1).standard_normal(c["q"].shape, dtype=np.float32) * np.float32(loss), "float16")


@pytest.mark.gpu
@pytest.mark.parametrize("large", ["q", "k"])
@pytest.mark.parametrize("bad", [np.inf, np.nan, 65504.0])
@pytest.mark.parametrize("dim", [64, 80, 128, 256])
def test_padding_does_not_move_the_hold(hip, large, bad, dim):
    docs = packed(2, 200, 2, 13)
    data, w = case(2, 200, 200, 4, 2, dim, large, dim)
    pad = docs < 0
    data["v"][pad] = 0
    w[pad] = 0
    want = ref(data["q"], data["k"], data["v"], w, dtype="float16", causal=True, documents=docs)
    data["v"][pad] = bad
    w[pad] = bad
    for n, g in gradients(data, w, causal=True, documents=docs).items():
        assert_within(g, want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("large", ["q", "k"])
@pytest.mark.parametrize("bad", [np.inf, np.nan, 65504.0])
def test_rows_that_see_nothing_do_not_move_the_hold(hip, large, bad):
    lengths = np.array([25, 50], np.int32)
    data, w = case(2, 40, 50, 2, 1, 64, large, 7)
    w[0, :15] = 0  # before the sequence's first token
    data["v"][0, 25:] = 0
    want = ref(data["q"], data["k"], data["v"], w, dtype="float16", causal=True, lengths=lengths)
    w[0, :15] = bad
    data["v"][0, 25:] = bad
    for n, g in gradients(data, w, causal=True, lengths=lengths).items():
        assert_within(g, want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("large", ["q", "k"])
@pytest.mark.parametrize("apart", ["batch", "head"])
def test_other_sequences_and_heads_do_not_move_the_hold(hip, large, apart):
    """One sequence's (or key head's) loss is 2^22 times the others'."""
    data, w = case(3, 150, 150, 4, 2, 64, large, 17)
    grown = w[1] if apart == "batch" else w[:, :, 2:]
    grown *= np.float32(2.0 ** 22)
    want = ref(data["q"], data["k"], data["v"], w, dtype="float16", causal=True)
    for n, g in gradients(data, w, causal=True).items():
        assert_within(g, want[n], n)

"""The convolution's gradient at a sequence's end, and where a work-group goes through
several tiles of tokens. Against the formula in 64 bits (recurrent_ref.py)."""
import numpy as np
import pytest

import recurrent_ref as ref
from test_causal_conv import run
from test_recurrence import documents_of, tensor


@pytest.mark.gpu
@pytest.mark.parametrize("bad", [np.inf, np.nan])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("width", [2, 3, 4, 6])
@pytest.mark.parametrize("length", [5, 64, 257, 283])
def test_infinite_inputs_reach_the_taps_that_read_them(hip, length, width, dtype, bad):
    """The last token is read by the last tap alone, the one before by the last two: the other taps' gradients, and every
    input's, stay finite."""
    from ormi_amd import causal_conv, realize_all

    rng = np.random.default_rng(length)
    x, w = rng.standard_normal((2, 2, length, 10)).astype(np.float32)
    weight = rng.standard_normal((10, width)).astype(np.float32)
    clean = x.copy()
    x[:, -1, :7] = bad
    x[0, -2, 3] = bad
    tokens, taps = tensor(x, dtype, True), tensor(weight, grad=True)
    bias, w = tensor(np.ones(10, np.float32), grad=True), tensor(w, dtype)
    y, _ = causal_conv(tokens, taps, bias)
    (y * w).sum().backward()
    realize_all(y, tokens.grad, taps.grad, bias.grad)
    want, bound = ref.conv(tensor(clean, dtype).numpy(), weight, np.ones(10, np.float32), False, dy=w.numpy())
    reads = np.zeros((10, width), bool)
    reads[:7, width - 1] = True
    if width > 1:
        reads[3, width - 2] = True
    got = taps.grad.numpy()
    assert not np.isfinite(got[reads]).any()
    ref.close(got[~reads], want["dw"][~reads], bound["dw"][~reads], "float32", "dw")
    ref.close(bias.grad.numpy(), want["db"], bound["db"], "float32", "db")
    ref.close(tokens.grad.numpy(), want["dx"], bound["dx"], dtype, "dx")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("width,masks", [(3, ""), (4, ""), (8, ""), (2, "documents"), (4, "documents and lengths"), (8, "lengths")])
def test_several_tiles_to_a_work_group(hip, width, masks, dtype):
    """2100 batches leave one work-group for each batch's tiles. A weight's gradient adds up 2 tiles' runs of 32 tokens in
    a thread, 8 runs in 3 steps, and the 2100 rows 16 side by side: 64 + 3 + 132 + 4 additions at most, fewer than the
    2140 that the bounds count for these sizes."""
    shape = (2100, 270, 3)
    rng = np.random.default_rng(width)
    held = {}
    if "documents" in masks:
        held["documents"] = documents_of(*shape[:2], 5, rng)
    if "lengths" in masks:
        held["lengths"] = rng.integers(0, shape[1] + 1, shape[0]).astype(np.int32)
        held["lengths"][:5] = 0, 1, shape[1], 256, 257
    run(shape, width, dtype, "silu", rng, initial=True, dlast=True, **held)
    if dtype != "float32":
        run(shape, width, dtype, None, rng, bias=False, wide=True, **held)

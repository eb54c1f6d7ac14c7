"""Clipping where no norm is too large: max_norm=inf leaves every element as it is but for a norm of NaN."""
import numpy as np
import pytest


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_infinite_bounds(hip, dtype):
    from ormi_amd import Tensor, clip_grads

    a = np.array([1.0, -2.0, np.inf, 0.5, -np.inf], np.float32)
    (c,), norm = clip_grads([Tensor(a, "hip", dtype=dtype)], np.inf)
    assert np.isinf(norm.numpy()) and np.array_equal(c.numpy(), a)
    (c,), norm = clip_grads([Tensor(a, "hip", dtype=dtype)], 1e30)
    assert np.isnan(c.numpy()[[2, 4]]).all() and not c.numpy()[[0, 1, 3]].any()
    a[1] = np.nan
    (c,), norm = clip_grads([Tensor(a, "hip", dtype=dtype)], np.inf)
    assert np.isnan(norm.numpy()) and np.isnan(c.numpy()).all()

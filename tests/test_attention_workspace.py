"""Packed operands of more than 8 GiB together: the workspace's size is past what
one 32-bit extent of words holds."""
import numpy as np
import pytest

KEYS = (1 << 28) + 4096  # rows of one float32 feature are packed to 16 bytes, twice


@pytest.mark.gpu
def test_a_workspace_past_8_gib(hip, ob):
    """Equal scores over equal values. Each lane's counts stay below 2^24 and its sums are multiples of 1/4 below
    2^22, exact; 64 splits are joined by at most 64 + 6 additions and two products and a quotient more."""
    from ormi_amd import Tensor, attention

    q = Tensor(np.ones((1, 1, 1, 1), np.float32), "hip")
    v = Tensor(np.full((1, 1, 1, 1), 0.75, np.float32), "hip")
    out = attention(q, q.expand((1, KEYS, 1, 1)), v.expand((1, KEYS, 1, 1))).numpy()
    ob.empty_cache()  # so much is not kept for the tests after this one
    assert out.shape == (1, 1, 1, 1) and abs(float(out[0, 0, 0, 0]) - 0.75) <= 74 * 2.0 ** -24 * 0.75

"""Wide caps: the capped score keeps the score's own accuracy, however far the
cap is above it. The bounds are those of uncapped scores (attention_ref.py) and a
tenth more: a tanh off by 3 units in the last place and two products more put
6 u |t| on top of a score's (D + 8) u S + 4 u |t| with S >= |t|, at most a twelfth
of it for D of 64 and more."""
import numpy as np
import pytest

from attention_ref import assert_within, attention as ref
from test_attention import DTYPES, make, run


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("cap", [1e3, 1e4, 1e6, 1e8, 1e30])
@pytest.mark.parametrize("dim,slopes", [(64, False), (96, True), (128, False), (256, True)])
def test_wide_caps_keep_the_scores(hip, dtype, cap, dim, slopes):
    more = {"slopes": np.float32([0.5, 0.1])} if slopes else {}
    got, data, host, options, w = run(make(1, 100, 140, 2, 1, dim, seed=dim, size=1.7, causal=True, cap=cap, **more), dtype)
    exact = ref(data["q"], data["k"], data["v"], w, dtype=dtype, **options, **host)
    plain = ref(data["q"], data["k"], data["v"], w, dtype=dtype, causal=True, **host)
    for n in exact:
        assert_within(got[n], (exact[n][0], 1.1 * plain[n][1]), n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_wide_caps_bend_large_scores(hip, dtype):
    """Scores of several caps of 300: the bent part counts, and its derivative."""
    case = make(1, 60, 60, 2, 1, 64, seed=3, size=1.0, causal=True, cap=300.0, scale=60.0)
    got, data, host, options, w = run(case, dtype)
    want = ref(data["q"], data["k"], data["v"], w, dtype=dtype, **options)
    for n in want:
        assert_within(got[n], want[n], n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", DTYPES)
def test_one_token_under_a_wide_cap(hip, dtype):
    got, data, host, options, _ = run(make(2, 1, 700, 8, 2, 64, seed=5, size=1.7, causal=True, cap=1e6), dtype, grad=False)
    exact = ref(data["q"], data["k"], data["v"], dtype=dtype, **options)["out"][0]
    bound = ref(data["q"], data["k"], data["v"], dtype=dtype, causal=True)["out"][1]
    assert_within(got["out"], (exact, 1.1 * bound), "out")

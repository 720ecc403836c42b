"""Host-side arguments of the paged operators and 4-bit weights at their edges, without a GPU."""
import warnings

import numpy as np
import pytest

from mira_b200 import kernels as K


@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_w4_quantize_shows_what_is_not_finite(bad):
    """absmax / 7 of a group with a NaN or infinity is one, and so what its codes stand for is NaN or infinite;
    other groups are as ever."""
    rng = np.random.default_rng(0)
    w = rng.standard_normal((3, 100)).astype(np.float32)
    want, want_s = K.w4_quantize(w, 32)
    w[1, 40] = bad
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        q, s = K.w4_quantize(w, 32)
    assert not np.isfinite(s[1, 1])
    group = np.zeros((3, 100), bool)
    group[1, 32:64] = True
    with np.errstate(invalid="ignore"):
        back = q * np.repeat(s, 32, 1)[:, :100]
    assert not np.isfinite(back[1, 40]) and np.abs(q).max() <= 7
    np.testing.assert_array_equal(q[~group], want[~group])
    np.testing.assert_array_equal(np.delete(s.ravel(), 5), np.delete(want_s.ravel(), 5))


def test_w4_quantize_of_the_smallest_weights():
    """Where absmax / 7 is 0 the codes stand for 0, without a warning."""
    w = np.zeros((1, 32), np.float32)
    w[0, 3] = 1e-45
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        q, s = K.w4_quantize(w, 32)
    assert (q * s == 0).all() and np.abs(q).max() <= 7

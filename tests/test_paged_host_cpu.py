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


@pytest.mark.parametrize("src,dst", [([2 ** 32], [1]), ([0], [2 ** 32 + 1]), ([-2 ** 32], [1]), ([0.7], [1]), ([0], [1.5]),
                                     ([float("nan")], [1]), ([True], [False]), (["0"], ["1"])])
@pytest.mark.parametrize("array", [True, False])
def test_page_copy_takes_page_ids_only(monkeypatch, src, dst, array):
    """Ids that 32 bits do not hold, and what is no whole number, are refused, not cut to some page's id."""
    calls = []
    monkeypatch.setattr(K._lib, "call", lambda *a: calls.append(a))
    region = [K.PageRegion(1 << 20, page_bytes=16, page_stride=16)]
    if array:
        src, dst = np.array(src), np.array(dst)
    with pytest.raises(ValueError):
        K.page_copy(region, 4, src, dst)
    assert not calls


@pytest.mark.parametrize("kind", [list, tuple, np.array, lambda x: np.array(x, np.int64), lambda x: np.array(x, np.uint8)])
def test_page_copy_passes_page_ids(monkeypatch, kind):
    calls = []

    def call(name, n_regions, regions, num_pages, n, src, dst):
        import ctypes
        read = lambda at: list((ctypes.c_int32 * n).from_address(at)) if n else []
        calls.append((name, num_pages, n, read(src), read(dst)))

    monkeypatch.setattr(K._lib, "call", call)
    region = [K.PageRegion(1 << 20, page_bytes=16, page_stride=16)]
    K.page_copy(region, 9, kind([3, 3]), kind([5, 8]))
    K.page_copy(region, 9, [], [])
    assert calls == [("mira_cuda_page_copy", 9, 2, [3, 3], [5, 8]), ("mira_cuda_page_copy", 9, 0, [], [])]


@pytest.mark.parametrize("bad", [8, -9, 127, -128])
@pytest.mark.parametrize("dtype", [np.int8, np.int32])
def test_w4_weight_takes_4_bit_codes_only(bad, dtype):
    """A code that four bits do not hold would change its neighbour's."""
    q = np.zeros((2, 5), dtype)
    q[1, 2] = bad
    with pytest.raises(ValueError):
        K.w4_weight(q)
    q[1, 2] = 7
    q[0, 3] = -8
    packed = K.w4_weight(q)
    assert packed[1, 1] == 0x8f and packed[0, 1] == 0x08
    assert K.w4_weight(np.zeros((0, 5), dtype)).shape == (0, 16)

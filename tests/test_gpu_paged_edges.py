"""Appends and attention over pages where the caller's lengths, rows or values are at their edges."""
import numpy as np
import pytest

import paged_ref as R
from test_gpu_paged import Case, _append, _pages_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kv", ["f32", "bf16", "i8"])
@pytest.mark.parametrize("over,new", [(1, 1), (1, 3), (2, 2), (5, 20), (1 << 20, 1)])
@pytest.mark.parametrize("starts", ["given", None])
def test_append_beyond_the_table_writes_nothing(cuda_device, kv, over, new, starts):
    """A full sequence whose length says that it has outgrown its table row keeps every row; the other
    sequence gets its own."""
    from mira_b200 import _lib
    if starts is None:
        new = 1
    c = Case(31, kv, 2, 2, 64, 16, [48, 17], fill="zero")
    c.max_pages = 3                                   # the table row ends with the sequence's last page
    c.table = np.ascontiguousarray(c.table[:, :3])
    c.lengths[0] = 48 + over
    c.upload()
    want = [c.k_bits.copy(), c.v_bits.copy()]
    want_s = [s.copy() for s in c.scales]
    x = np.random.default_rng(over + new).standard_normal((2, new + 1, 2, 64)).astype(np.float32)
    with pytest.raises(_lib.CudaError) as e:
        _append(c, [new, 1], "f32", x[0], x[1], **({} if starts else {"row_start": None}))
    assert e.value.code == _lib.EKERNEL
    page, slot = c.table[1, 1], 0
    for j in range(2):
        row = x[j, new]
        if kv == "i8":
            want[j][page, :, slot], want_s[j][page, :, slot] = R.quantize_row(row)
        else:
            want[j][page, :, slot] = R.to_bits(row, kv)
    got, got_s = _pages_of(c)
    for g, w in zip(got + got_s, want + want_s):
        np.testing.assert_array_equal(g, w)


def test_append_negative_length_writes_nothing(cuda_device):
    from mira_b200 import _lib
    c = Case(32, "f16", 2, 2, 64, 16, [40], fill="zero")
    c.lengths[0] = -3
    c.upload()
    x = np.ones((2, 2, 64), np.float32)
    with pytest.raises(_lib.CudaError):
        _append(c, [2], "f32", x, x)
    got, _ = _pages_of(c)
    np.testing.assert_array_equal(got[0], c.k_bits)
    np.testing.assert_array_equal(got[1], c.v_bits)


@pytest.mark.parametrize("dh", [64, 7])
@pytest.mark.parametrize("src", ["f32", "bf16"])
def test_append_nan_shows_in_8_bit_pages(cuda_device, src, dh):
    """absmax / 127 of a row with a NaN is NaN, and so is every value that its codes stand for; other rows
    and heads are as ever, and attention over the row is NaN for the sequence that sees it alone."""
    c = Case(33, "i8", 2, 2, dh, 16, [20, 20], fill="zero")
    x = R.from_bits(R.to_bits(np.random.default_rng(dh).standard_normal((2, 40, 2, dh)).astype(np.float32), src), src).copy()
    x[0, 3, 1, 5] = np.nan                      # a key of sequence 0, head 1
    x[1, 9, 0, 2] = np.nan                      # a value of sequence 0, head 0
    _append(c, [20, 20], src, x[0], x[1])
    codes, scales = _pages_of(c)
    t = np.arange(20)
    for b in range(2):
        for j in range(2):
            rows = x[j, 20 * b: 20 * b + 20]
            with np.errstate(invalid="ignore"):
                want, want_s = R.quantize_row(rows)
            got = codes[j][c.table[b, t // 16], :, t % 16]
            got_s = scales[j][c.table[b, t // 16], :, t % 16]
            bad = np.isnan(rows).any(-1)
            assert np.isnan(got_s[bad]).all()
            np.testing.assert_array_equal(got_s[~bad], want_s[~bad])
            np.testing.assert_array_equal(got[~bad], want[~bad])
    o, lse = c.attend()
    assert np.isnan(o[0]).all() and np.isnan(lse[0, 1]) and np.isfinite(lse[0, 0])
    assert np.isfinite(o[1]).all() and np.isfinite(lse[1]).all()


@pytest.mark.parametrize("src", ["f32", "f16"])
def test_append_smallest_and_largest_rows_to_8_bit_pages(cuda_device, src):
    """Zeros of either sign, subnormal and the largest finite values keep the formula's codes and scales."""
    c = Case(34, "i8", 1, 1, 64, 16, [6], fill="zero")
    x = np.random.default_rng(3).uniform(-1, 1, (2, 6, 1, 64)).astype(np.float32)
    x[:, 0] = 0.0
    x[:, 1] = -0.0
    x[:, 2] *= np.float32(1e-38 if src == "f32" else 6e-8)
    x[:, 3] *= np.float32(3.3e38 if src == "f32" else 65000)
    x[:, 4, :, 1:] = 0
    x = R.from_bits(R.to_bits(x, src), src)
    _append(c, [6], src, x[0], x[1])
    codes, scales = _pages_of(c)
    for j in range(2):
        want, want_s = R.quantize_row(x[j])
        np.testing.assert_array_equal(codes[j][c.table[0, 0], :, :6].transpose(1, 0, 2), want)
        np.testing.assert_array_equal(scales[j][c.table[0, 0], :, :6].T, want_s)

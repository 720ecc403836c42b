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

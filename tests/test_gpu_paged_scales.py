"""8-bit pages whose rows have scales of very different size: a weight's accuracy is relative to what its head
adds up, not to the largest scale there is."""
import numpy as np
import pytest

import paged_ref as R
import paged_tight as T
from test_gpu_paged import Case, _append, _pages_of

pytestmark = pytest.mark.gpu


def _check(c, window=0, sinks=0):
    got, lse = c.attend(window, sinks)[:2]
    o, bound, _, want_lse, lse_bound = T.of(c, window=window, sinks=sinks)
    assert np.isfinite(got).all()
    off = np.abs(got - o)
    worst = np.unravel_index(np.argmax(off / np.maximum(bound, 1e-300)), off.shape)
    assert (off <= bound).all(), (worst, float(off[worst]), float(bound[worst]), float(o[worst]))
    live = np.isfinite(want_lse)
    assert (np.abs(lse[live] - want_lse[live]) <= lse_bound[live]).all()
    return o, bound


def _rescale(c, j, by):
    """Multiplies the scales (and values) of keys (0) or values (1) by `by` [pages, kv heads, slots]."""
    c.scales[j] = (c.scales[j] * by).astype(np.float32)
    codes = (c.k_bits, c.v_bits)[j]
    val = codes.astype(np.float64) * np.nan_to_num(c.scales[j], nan=0.0)[..., None].astype(np.float64)
    if j == 0:
        c.k_val = val
    else:
        c.v_val = val


CASES = [(4, 2, 64, [700, 40, 0, 1]), (5, 1, 80, [3000]), (20, 2, 96, [500, 33]), (6, 6, 128, [300]), (3, 1, 256, [900, 7]),
         (12, 1, 48, [400])]


@pytest.mark.parametrize("q", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("heads,kv_heads,dh,lengths", CASES)
@pytest.mark.parametrize("bits", [12, 20, 40])
def test_zero_rows_beside_small_values(cuda_device, q, heads, kv_heads, dh, lengths, bits):
    """Values of a row size around 2^-bits and, among them, rows of zeros, which an append gives the scale 1."""
    c = Case(dh + bits, "i8", heads, kv_heads, dh, 16, lengths, q=q)
    _rescale(c, 1, np.float32(2.0 ** -bits))
    zero = np.random.default_rng(1).random(c.scales[1].shape) < 0.05
    zero[c.table[0, 0], :, 0] = True
    c.v_bits[zero] = 0
    c.v_val[zero] = 0
    c.scales[1][zero & ~np.isnan(c.scales[1])] = 1.0
    c.upload()
    _check(c)


@pytest.mark.parametrize("heads,kv_heads,dh,lengths", CASES)
@pytest.mark.parametrize("which", ["values", "keys and values"])
def test_scales_spread_over_2_40(cuda_device, heads, kv_heads, dh, lengths, which):
    """Whichever rows are large, the outputs of each head are as accurate as the terms that make them up."""
    c = Case(dh + 7, "i8", heads, kv_heads, dh, 16, lengths)
    rng = np.random.default_rng(2)
    _rescale(c, 1, 2.0 ** rng.integers(-40, 1, c.scales[1].shape))
    if which != "values":
        _rescale(c, 0, 2.0 ** rng.integers(-6, 2, c.scales[0].shape))
    c.upload()
    _check(c)


@pytest.mark.parametrize("large", [0, 5, 250, 399])
@pytest.mark.parametrize("size", [2.0 ** 20, 2.0 ** 60])
def test_a_large_value_that_weighs_nothing(cuda_device, large, size):
    """One token with large values and a weight below 2^-100 of the others' in every second head: there the
    other tokens decide, to the bits that they have alone; in the other heads the large one does."""
    c = Case(61, "i8", 8, 1, 64, 16, [400])
    page, slot = c.table[0, large // 16], large % 16
    by = np.ones(c.scales[1].shape)
    by[page, 0, slot] = size
    _rescale(c, 1, by)
    x = R.from_bits(c.q_bits, "f32")[0].astype(np.float64)
    # a key along head 0's query, which the odd heads turn away from
    c.q_bits[0, 1::2] = -c.q_bits[0, 0]
    c.q_bits[0, 0::2] = c.q_bits[0, 0]
    key = (x[0] / np.linalg.norm(x[0]) ** 2 * 140 * 8).astype(np.float32)
    codes, s = R.quantize_row(key)
    c.k_bits[page, 0, slot], c.scales[0][page, 0, slot] = codes, s
    c.k_val[page, 0, slot] = codes.astype(np.float64) * s
    c.upload()
    o, _ = _check(c)
    assert np.abs(o[0, 1::2]).max() < 1 or size > 2.0 ** 40
    assert np.abs(o[0, 0::2]).max() > size / 100


@pytest.mark.parametrize("order", ["rising", "falling"])
@pytest.mark.parametrize("heads", [1, 8, 16])
def test_scores_and_scales_that_go_opposite_ways(cuda_device, order, heads):
    """Every later step has a larger score and smaller values (or the reverse), so that what the sums are taken
    relative to changes all the time."""
    n = 1024
    c = Case(62, "i8", heads, 1, 64, 16, [n])
    t = np.arange(n)
    page, slot = c.table[0, t // 16], t % 16
    up = t if order == "rising" else n - 1 - t
    by = np.ones(c.scales[1].shape)
    by[page, 0, slot] = 2.0 ** -(up / 16.0).round()
    _rescale(c, 1, by)
    x = R.from_bits(c.q_bits, "f32")[0, 0].astype(np.float64)
    c.q_bits[0, :] = c.q_bits[0, 0]
    along = x / np.linalg.norm(x) ** 2 * 8
    rows = (along[None] * (up / 16.0 * np.log(2) * 0.9)[:, None]).astype(np.float32)
    codes, s = R.quantize_row(rows)
    c.k_bits[page, 0, slot], c.scales[0][page, 0, slot] = codes, s
    c.k_val[page, 0, slot] = codes.astype(np.float64) * s[:, None]
    c.upload()
    _check(c)


def test_appended_zero_rows(cuda_device):
    """The same through kv_append, which chooses the scales itself."""
    c = Case(63, "i8", 6, 2, 64, 16, [600, 50], fill="zero")
    rng = np.random.default_rng(5)
    x = rng.standard_normal((2, 650, 2, 64)).astype(np.float32)
    x[1] *= np.float32(1e-6)
    x[1, rng.random(650) < 0.1] = 0
    _append(c, [600, 50], "f32", x[0], x[1])
    codes, scales = _pages_of(c)
    c.k_val, c.v_val = (q.astype(np.float64) * s[..., None] for q, s in zip(codes, scales))
    _check(c)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("heads", [2, 5, 16])
def test_a_scale_that_is_not_finite_shows(cuda_device, bad, heads):
    """A visible row with such a scale makes the results infinite or NaN where its codes are not 0, of its
    sequence only."""
    for j in range(2):
        c = Case(64, "i8", heads, 1, 64, 16, [70, 70])
        c.scales[j][c.table[0, 2], 0, 3] = bad
        c.upload()
        o, lse = c.attend()
        codes = (c.k_bits, c.v_bits)[j][c.table[0, 2], 0, 3]
        if j == 1:
            assert (~np.isfinite(o[0][:, codes != 0])).all() and np.isfinite(lse).all()
        elif np.isnan(bad):
            assert np.isnan(o[0]).all() and np.isnan(lse[0]).all()
        else:        # the row's score is infinite: -inf leaves it out, else nothing is finite
            out = np.isfinite(lse[0])
            assert np.isfinite(o[0][out]).all() and not np.isfinite(o[0][~out]).any()
        assert np.isfinite(o[1]).all() and np.isfinite(lse[1]).all()

"""Long sequences, whose parts are worked out by many blocks and joined: every result against a bound that a
missing or misweighted part exceeds (paged_tight), which the tests show of the oracle as well."""
import numpy as np
import pytest

import paged_ref as R
import paged_tight as T
from test_gpu_paged import Case

pytestmark = pytest.mark.gpu

LONG = [("f32", "bf16", 8, 2, 128, [20000]), ("f32", "f32", 3, 3, 64, [9999, 5]), ("f32", "i8", 16, 2, 64, [7000] * 3 + [1]),
        ("f32", "f16", 32, 1, 64, [4097]), ("f32", "f32", 1, 1, 16, [70001]), ("bf16", "bf16", 8, 1, 64, [1500, 700, 3000]),
        ("f16", "f16", 4, 4, 64, [12000]), ("f32", "f32", 8, 2, 64, [6000, 100]), ("bf16", "i8", 5, 1, 80, [9000])]


def _holds(c, got, lse, window=0, sinks=0):
    o, bound, _, want_lse, lse_bound = T.of(c, window=window, sinks=sinks)
    off = np.abs(got - o)
    assert (off <= bound).all(), float((off / np.maximum(bound, 1e-300)).max())
    live = np.isfinite(want_lse)
    assert (lse[~live] == -np.inf).all() and (np.abs(lse[live] - want_lse[live]) <= lse_bound[live]).all()
    return o, bound


@pytest.mark.parametrize("q,kv,heads,kv_heads,dh,lengths", LONG)
def test_long_sequences(cuda_device, q, kv, heads, kv_heads, dh, lengths):
    c = Case(len(lengths) + dh, kv, heads, kv_heads, dh, 16, lengths, q=q)
    got, lse = c.attend()
    o, bound = _holds(c, got, lse)
    # the bound is small beside the results of the longest sequence: zeros fail, and so does a result without
    # one part in 64 of its tokens
    b = int(np.argmax(lengths))
    rms = np.sqrt((o[b] ** 2).mean())
    assert np.median(bound[b]) < (0.05 if q == "f32" else 0.2) * rms
    assert (np.abs(o[b]) > bound[b]).mean() > 0.8
    for first in (0, lengths[b] // 2, lengths[b] - lengths[b] // 64):
        without = T.of(c, leave=lambda s, t: np.arange(first, first + lengths[b] // 64))[0]
        assert (np.abs(without[b] - o[b]) > bound[b]).mean() > 0.3


@pytest.mark.parametrize("q,kv,heads", [("f32", "f32", 2), ("f32", "bf16", 8), ("bf16", "bf16", 8), ("f16", "f16", 4), ("f32", "i8", 6)])
@pytest.mark.parametrize("at", [0, 1, 4999, 9000, 9999])
def test_one_part_decides(cuda_device, q, kv, heads, at):
    """Nearly all of the weight lies in 16 tokens of 10000: the part that holds them has to reach the result
    with its own weight, the others with theirs."""
    c = Case(at + 40, kv, heads, 1, 64, 16, [10000, 40], q=q)
    t = np.arange(at, at + 16) % 10000
    page, slot = c.table[0, t // 16], t % 16
    for h in range(heads):
        c.q_bits[0, h] = c.q_bits[0, 0]
    x = R.from_bits(c.q_bits, q)[0, 0].astype(np.float64)
    along = (x / np.linalg.norm(x) * 60 / np.linalg.norm(x) * np.sqrt(64) / 4).astype(np.float32)      # a score of about 15 above the rest
    if kv == "i8":
        codes, s = R.quantize_row(np.broadcast_to(along, (16, 64)))
        c.k_bits[page, 0, slot], c.scales[0][page, 0, slot] = codes, s
        c.k_val[page, 0, slot] = codes.astype(np.float64) * s[:, None]
    else:
        c.k_bits[page, 0, slot] = R.to_bits(along, kv)
        c.k_val[page, 0, slot] = R.from_bits(c.k_bits[page, 0, slot], kv)
    c.upload()
    got, lse = c.attend()
    o, bound = _holds(c, got, lse)
    without = T.of(c, leave=lambda b, s: t if b == 0 else [])[0]
    assert (np.abs(without[0] - o[0]) > bound[0]).mean() > 0.9


@pytest.mark.parametrize("q,kv,heads,window,sinks", [("f32", "bf16", 8, 4000, 5), ("f32", "f32", 2, 3000, 100), ("f32", "i8", 6, 4095, 4)])
def test_long_windows(cuda_device, q, kv, heads, window, sinks):
    c = Case(51, kv, heads, 2, 64, 16, [9000, 2500, 4100], q=q)
    got, lse = c.attend(window, sinks)
    _holds(c, got, lse, window, sinks)

"""A bound of paged attention's error by the terms of its sums.

For one (sequence, head) and element d let A_d = sum_t p_t |v_td| with p the softmax weights.  A weight is off by
the error of its score, relatively, and by the rounding of the exponential; the sums over t round each term
independently, so that their errors add like sqrt(n), to A_d and to the sum of the weights alike:

  |o_d - exact| <= 2 A_d (score + piece + (sqrt(n) + 8) eps) + |o_d| unit + n 2^-126 (max_t |v_td| + 128)
  score = (dh + 8) eps max_t sum_d |scale q_d k_td|  (+ what splitting q leaves, 2^-22 of its largest element)
  piece = what the values that a weight enters the products as leave of it, relatively
the last term is for weights below 2^-126 of the largest, which are 0, and 8-bit codes times what f32 holds of a
weight times a scale.

It shrinks with the outputs, which are averages over n tokens, so that a missing or misweighted part shows."""
import numpy as np

import paged_ref as R


def piece(q, kv):
    """What the weights' 16-bit values leave, twice over for the rounding of the largest: nothing on the f32 path;
    two bf16 values 2^-16, three 2^-24; two f16 values 2^-22."""
    if kv == "f32":
        return 0.0
    if kv == "bf16":
        return 2.0 ** -15 if q == "bf16" else 2.0 ** -23
    return 2.0 ** -21


def attention(q, k, v, table, lengths, page_size, scale, q_dtype, kv, window=0, sinks=0, leave=None):
    """q [B, H, dh]; k, v [pages, kv heads, page_size, dh] as values.  Returns o, its bound, A and lse with its
    bound.  leave(b, tokens): positions to leave out, for a result that has to be found wrong."""
    B, H, dh = q.shape
    g = H // k.shape[1]
    o, bound, size = (np.zeros((B, H, dh)) for _ in range(3))
    lse, lse_bound = np.full((B, H), -np.inf), np.zeros((B, H))
    split = 2.0 ** -22 if kv in ("f16", "i8") and q_dtype != "f16" else 0.0
    for b in range(B):
        t = R.visible(int(lengths[b]), window, sinks)
        if leave is not None:
            t = np.setdiff1d(t, leave(b, t))
        if not len(t):
            continue
        page, slot = table[b, t // page_size], t % page_size
        for h in range(H):
            kk, vv = k[page, h // g, slot].astype(np.float64), v[page, h // g, slot].astype(np.float64)
            x = q[b, h].astype(np.float64)
            s = kk @ x * scale
            score = (dh + 8) * R.EPS * (np.abs(kk) @ np.abs(x)).max() * abs(scale)
            score += split * np.abs(x).max() * np.abs(kk).sum(1).max() * abs(scale)
            m = s.max()
            p = np.exp(s - m)
            total = p.sum()
            o[b, h], size[b, h] = p @ vv / total, p @ np.abs(vv) / total
            lse[b, h] = m + np.log(total)
            off = score + (np.sqrt(len(t)) + 8) * R.EPS
            bound[b, h] = 2 * size[b, h] * (off + piece(q_dtype, kv)) + len(t) * 2.0 ** -126 * (np.abs(vv).max(0) + 128)
            lse_bound[b, h] = off + 8 * R.EPS * abs(lse[b, h])
    bound += np.abs(o) * R.UNIT[q_dtype] * 1.01 + (2.0 ** -25 if q_dtype == "f16" else 0)
    return o, bound, size, lse, lse_bound


def of(case, leave=None, window=0, sinks=0):
    """The same of a test's Case."""
    return attention(R.from_bits(case.q_bits, case.q_dtype), case.k_val, case.v_val, case.table, case.lengths, case.page,
                     np.float64(np.float32(case.dh ** -0.5)), case.q_dtype, case.kv, window, sinks, leave)

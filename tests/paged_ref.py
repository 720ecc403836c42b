"""Plain 64-bit forms of the paged operators and 4-bit products, and the element types NumPy lacks."""
import numpy as np

EPS = 2.0 ** -23        # a product or sum on the tensor cores may round toward zero
UNIT = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}


def to_bits(x, dtype):
    """f32 values -> the stored elements of `dtype` (round to nearest even), bf16 as uint16."""
    x = np.asarray(x, np.float32)
    if dtype == "f32":
        return x
    if dtype == "f16":
        with np.errstate(over="ignore"):
            return x.astype(np.float16)
    if dtype == "bf16":
        u = x.view(np.uint32).astype(np.uint64)
        r = (u + 0x7FFF + ((u >> 16) & 1)) >> 16
        return np.where(np.isnan(x), 0x7FFF, r).astype(np.uint16)
    raise ValueError(dtype)


def from_bits(b, dtype):
    if dtype == "bf16":
        return (np.asarray(b, np.uint16).astype(np.uint32) << 16).view(np.float32)
    return np.asarray(b).astype(np.float32)


NP = {"f32": np.float32, "f16": np.float16, "bf16": np.uint16, "i8": np.int8}


def quantize_row(x):
    """int8 codes and scale of rows over the last axis."""
    x = np.asarray(x, np.float32)
    top = np.abs(x).max(axis=-1)
    s = np.where(top > 0, top / np.float32(127), np.float32(1)).astype(np.float32)
    return np.clip(np.rint(x / s[..., None]), -127, 127).astype(np.int8), s


def visible(n, window, sinks):
    start = max(0, n - window) if window else 0
    return np.concatenate([np.arange(min(sinks, start)), np.arange(start, n)]).astype(np.int64)


def attention(q, k, v, table, lengths, page_size, scale, window=0, sinks=0):
    """q [B, H, dh]; k, v [pages, kv heads, page_size, dh] as values.  Returns o, lse and an error bound
    of each for f32 arithmetic: scores are off by at most (dh + 8) eps S, S = scale sum |q k|, each
    weight by that and the rounding of exp2, and a sum of n terms by n eps."""
    B, H, dh = q.shape
    g = H // k.shape[1]
    o, lse = np.zeros((B, H, dh)), np.full((B, H), -np.inf)
    bo, bl = np.zeros((B, H, 1)), np.zeros((B, H))
    for b in range(B):
        t = visible(int(lengths[b]), window, sinks)
        if not len(t):
            continue
        page, slot = table[b, t // page_size], t % page_size
        for h in range(H):
            kk, vv = k[page, h // g, slot].astype(np.float64), v[page, h // g, slot].astype(np.float64)
            s = kk @ q[b, h].astype(np.float64) * scale
            size = np.abs(kk) @ np.abs(q[b, h].astype(np.float64)) * abs(scale)
            m = s.max()
            p = np.exp(s - m)
            o[b, h] = p @ vv / p.sum()
            lse[b, h] = m + np.log(p.sum())
            off = (dh + 8) * EPS * size.max() + 8 * EPS
            bo[b, h] = 2 * np.abs(vv).max() * (off + len(t) * EPS)
            bl[b, h] = off + len(t) * EPS + 8 * EPS * abs(lse[b, h])
    return o, lse, bo, bl

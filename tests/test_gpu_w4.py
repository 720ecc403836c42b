"""Products with 4-bit weights on the GPU against the 64-bit formula: sizes and groups that end inside a
word, a tile or a group, types, strides, epilogue steps, and what is refused.

The bound of a result is k eps sum |x w s| (f32 sums of exact products) and the output's rounding."""
import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu


def _k():
    from mira_b200 import kernels as K
    from mira_b200.device import DeviceBuffer
    return K, DeviceBuffer


class Product:
    def __init__(self, m, n, k, group, x="f32", scales="f32", out=None, seed=0, pad_x=0, pad_s=0, pad_out=0, garbage=True):
        self.K, self.DB = _k()
        rng = np.random.default_rng(seed + m * 3 + n * 5 + k * 7)
        self.m, self.n, self.k, self.group, self.xt, self.st, self.ot = m, n, k, group, x, scales, out or x
        self.groups = -(-k // group)
        self.x = R.to_bits(rng.standard_normal((m, k + pad_x)).astype(np.float32), x)
        if pad_x:
            self.x[:, k:] = R.to_bits(np.float32(np.nan), x)
        self.q = rng.integers(-8, 8, (n, k)).astype(np.int8)
        self.s = R.to_bits(rng.uniform(0.2, 1.5, (n, self.groups + pad_s)).astype(np.float32) / 8, scales)
        self.w = self.K.w4_weight(self.q)
        if garbage:      # what a row holds past element k is not used
            full = np.stack([self.w & 15, self.w >> 4], -1).reshape(n, -1)
            full[:, k:] = rng.integers(0, 16, full[:, k:].shape)
            self.w = (full[:, 0::2] | (full[:, 1::2] << 4)).astype(np.uint8)
        self.ld_x, self.ld_s, self.ld_out = k + pad_x, self.groups + pad_s, n + pad_out
        self.xb, self.wb, self.sb = (self.DB.from_array(a) for a in (self.x, self.w, self.s))
        self.out = self.DB(m * self.ld_out * np.dtype(R.NP[self.ot]).itemsize, zero=True)

    def exact(self):
        x = R.from_bits(self.x, self.xt)[:, : self.k].astype(np.float64)
        w = self.q * np.repeat(R.from_bits(self.s, self.st)[:, : self.groups].astype(np.float64), self.group, 1)[:, : self.k]
        return x @ w.T, (np.abs(x) @ np.abs(w).T) * (self.k + 8) * R.EPS

    def desc(self, **kw):
        size = self.K.w4_matvec_workspace(self.m, self.n, self.k)
        self.ws = self.DB(size, zero=True) if size else None
        args = dict(m=self.m, n=self.n, k=self.k, group=self.group, x=self.xb, ld_x=self.ld_x, w=self.wb, ld_w=self.w.shape[1],
                    scales=self.sb, ld_scales=self.ld_s, out=self.out, ld_out=self.ld_out, x_dtype=self.xt, scale_dtype=self.st,
                    out_dtype=self.ot, workspace=self.ws, workspace_bytes=size)
        args.update(kw)
        return self.K.W4Matvec(**args)

    def run(self, **kw):
        from mira_b200 import _lib
        d = self.desc(**kw).struct()
        for _ in range(2):          # the second call finds the workspace as the first left it
            self.K.w4_matvec(d)
        _lib.call("mira_cuda_sync")
        return R.from_bits(self.out.download((self.m, self.ld_out), R.NP[self.ot]), self.ot)[:, : self.n]

    def check(self):
        want, bound = self.exact()
        got = self.run()
        bound = bound + np.abs(want) * R.UNIT[self.ot] * 1.01 + (2.0 ** -25 if self.ot == "f16" else 0)
        off = np.abs(got - want)
        assert (off <= bound).all(), (float((off / bound).max()), np.argwhere(~(off <= bound))[:4].tolist())


@pytest.mark.parametrize("x", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("scales", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
def test_types_and_groups(cuda_device, x, scales, group):
    Product(3, 200, 768, group, x, scales).check()


@pytest.mark.parametrize("m,n,k,group", [
    (1, 1, 1, 32), (1, 1, 33, 32), (2, 3, 7, 32), (1, 16, 64, 64), (1, 17, 65, 32), (5, 15, 31, 32), (4, 100, 1000, 128),
    (7, 129, 255, 64), (8, 64, 513, 32), (9, 33, 129, 128), (16, 48, 2049, 256), (17, 50, 96, 32), (33, 31, 160, 32), (1, 4096, 4096, 128),
    (2, 777, 5003, 64), (1, 5, 40000, 32), (12, 1000, 31, 64), (100, 20, 500, 128), (3, 70, 2048, 1 << 33), (1, 640, 300, 160)])
@pytest.mark.parametrize("x", ["f32", "bf16"])
def test_sizes(cuda_device, m, n, k, group, x):
    p = Product(m, n, k, min(group, 1 << 20), x, "f16" if x == "f32" else "bf16")
    p.check()
    if group > 1 << 20:
        np.testing.assert_array_equal(p.run(group=group), p.run())


@pytest.mark.parametrize("m", range(1, 17))
def test_rows_of_a_decode_batch(cuda_device, m):
    for x in ("f32", "f16", "bf16"):
        Product(m, 130, 1024, 64, x, "f32").check()


@pytest.mark.parametrize("x,pad_x", [("f32", 1), ("f32", 4), ("bf16", 3), ("f16", 8)])
def test_strides(cuda_device, x, pad_x):
    p = Product(5, 70, 333, 64, x, "f16", pad_x=pad_x, pad_s=3, pad_out=5)
    p.check()
    rest = p.out.download((5, 75), R.NP[x])[:, 70:]
    assert (R.from_bits(rest, x) == 0).all()


@pytest.mark.parametrize("x,out", [("f32", "f16"), ("bf16", "f32"), ("f16", "bf16")])
def test_result_type_is_its_own(cuda_device, x, out):
    Product(2, 100, 512, 128, x, "f32", out).check()


def test_wide_range_of_rows(cuda_device):
    """Rows of very different size keep their relative accuracy, and equal calls give equal bits."""
    p = Product(4, 64, 512, 64, "f32", "f32")
    p.x *= np.array([[1e-30], [1e30], [1.0], [1e-3]], np.float32)
    p.xb = p.DB.from_array(p.x)
    p.check()
    np.testing.assert_array_equal(p.run(), p.run())


def test_zero_and_infinite_values(cuda_device):
    p = Product(2, 40, 100, 32, "f32", "f32")
    p.x[0] = 0
    p.x[1, 50] = np.inf
    p.xb = p.DB.from_array(p.x)
    got = p.run()
    assert (got[0] == 0).all()
    # an infinity times the code 0 is NaN, as in the formula
    with np.errstate(invalid="ignore"):
        want = np.float32(np.inf) * p.q[:, 50].astype(np.float32)
    np.testing.assert_array_equal(got[1], want)


def test_epilogue_steps(cuda_device):
    K, DB = _k()
    p = Product(6, 90, 256, 64, "f32", "f32")
    base = p.run()
    rng = np.random.default_rng(1)
    bias, res, row = (rng.standard_normal(s).astype(np.float32) for s in (90, (6, 95), 6))
    bb, rb, wb = DB.from_array(bias), DB.from_array(res), DB.from_array(row)
    got = p.run(steps=[K.Step("add", "channel", ptr=bb), K.Step("relu"), K.Step("add", "full", ptr=rb, ld=95),
                       K.Step("mul", "row", ptr=wb), K.Step("sub", "scalar", swapped=True, scalar=2.0)])
    want = np.float32(2.0) - (np.maximum(base + bias, np.float32(0)) + res[:, :90]) * row[:, None]
    np.testing.assert_array_equal(got, want)
    got = p.run(steps=[K.Step("gelu")])
    from oracle import w8a8 as ref
    np.testing.assert_allclose(got, ref._gelu(base.astype(np.float64)), rtol=1e-5, atol=1e-6)


def test_quantized_weights(cuda_device):
    """w4_quantize and w4_weight give what the kernel multiplies by."""
    K, DB = _k()
    rng = np.random.default_rng(2)
    w = rng.standard_normal((50, 200)).astype(np.float32)
    w[3, 64:128] = 0
    q, s = K.w4_quantize(w, 64)
    assert q.min() >= -7 and q.max() <= 7 and (s[3, 1] == 1)
    back = q * np.repeat(s, 64, 1)[:, :200]
    assert (np.abs(back - w) <= np.repeat(s, 64, 1)[:, :200] * 0.5001).all()
    p = Product(2, 50, 200, 64)
    p.q, p.s, p.w = q, s, K.w4_weight(q)
    p.wb, p.sb = DB.from_array(p.w), DB.from_array(p.s)
    p.check()


def test_refusals(cuda_device):
    from mira_b200 import _lib
    p = Product(2, 40, 100, 32, "f32", "f32", garbage=False)
    K = p.K
    before = p.out.download((2, 40), np.float32)
    bad = [dict(group=0), dict(group=48), dict(group=-32), dict(k=0), dict(m=-1), dict(n=-1), dict(ld_x=99), dict(ld_w=40), dict(ld_w=56),
           dict(ld_scales=3), dict(ld_out=39), dict(x=None), dict(w=None), dict(scales=None), dict(out=None), dict(w=p.wb.ptr + 8),
           dict(x=p.xb.ptr + 2), dict(x_dtype="i8"), dict(scale_dtype="i8"), dict(out_dtype="i8"),
           dict(steps=[K.Step("add", "channel")]), dict(steps=[K.Step("add", "none")]), dict(steps=[K.Step("relu", "scalar")])]
    if K.w4_matvec_workspace(2, 40, 100):
        bad += [dict(workspace=None), dict(workspace_bytes=0)]
    for kw in bad:
        with pytest.raises(_lib.CudaError) as e:
            K.w4_matvec(p.desc(**kw))
        assert e.value.code == _lib.EINVAL, kw
    with pytest.raises(ValueError):
        p.desc(steps=[K.Step("relu")] * 9).struct()
    np.testing.assert_array_equal(p.out.download((2, 40), np.float32), before)
    launches = _lib.launch_count()
    K.w4_matvec(p.desc(m=0))
    K.w4_matvec(p.desc(n=0))
    assert _lib.launch_count() == launches
    p.check()

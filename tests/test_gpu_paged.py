"""Paged attention, appended rows and page copies on the GPU against plain 64-bit forms (paged_ref):
element types, head layouts, page sizes, lengths from none to thousands, windows with sinks, strides,
offsets beyond 32 bits, and what is refused."""
import ctypes as C

import numpy as np
import pytest

import paged_ref as R

pytestmark = pytest.mark.gpu


def _k():
    from mira_b200 import kernels as K
    from mira_b200.device import DeviceBuffer
    return K, DeviceBuffer


class Case:
    """A paged cache with random contents on the device, and its values on the host."""

    def __init__(self, seed, kv, heads, kv_heads, dh, page, lengths, q="f32", order="head", fill="nan", shared=False, scale_q=1.5):
        self.K, self.DB = _k()
        rng = np.random.default_rng(seed)
        self.kv, self.q_dtype, self.heads, self.kv_heads, self.dh, self.page = kv, q, heads, kv_heads, dh, page
        self.lengths = np.array(lengths, np.int32)
        B = len(lengths)
        need = [-(-int(n) // page) for n in lengths]
        self.max_pages = max(1, max(need)) + 1
        self.num_pages = sum(need) + 2
        order_ids = rng.permutation(self.num_pages)[: sum(need)]
        self.table = np.full((B, self.max_pages), -7, np.int32)      # entries past the last page: no page
        at = 0
        for b, n in enumerate(need):
            self.table[b, :n] = order_ids[at: at + n]
            at += n
        if shared and B > 1:      # the second sequence starts with the first one's pages
            both = min(need[0], need[1])
            self.table[1, :both] = self.table[0, :both]
        shape = (self.num_pages, kv_heads, page, dh)
        seen = np.zeros((self.num_pages, page), bool)
        for b, n in enumerate(lengths):
            t = np.arange(n)
            seen[self.table[b, t // page], t % page] = True
        vals = []
        self.scales = []
        for _ in range(2):
            x = rng.standard_normal(shape).astype(np.float32)
            if kv == "i8":
                codes, s = R.quantize_row(x)
                vals.append(codes.astype(np.float64) * s[..., None].astype(np.float64))
                s[~np.broadcast_to(seen[:, None, :], s.shape)] = np.nan if fill == "nan" else 1
                self.scales.append(s)
                bits = codes
            else:
                bits = R.to_bits(x, kv)
                vals.append(R.from_bits(bits, kv))
                if fill == "nan":
                    bad = np.broadcast_to(~seen[:, None, :, None], shape)
                    bits = np.where(bad, R.to_bits(np.float32(np.nan), kv), bits).astype(bits.dtype)
            setattr(self, "kv"[len(vals) - 1] + "_bits", bits)
        self.k_val, self.v_val = vals
        self.q_bits = R.to_bits(rng.standard_normal((B, heads, dh)).astype(np.float32) * scale_q, q)
        self.order = order
        self.upload()

    def _dev(self, a):
        return self.DB.from_array(np.ascontiguousarray(a if self.order == "head" else np.swapaxes(a, 1, 2)))

    def strides(self):
        h, p, d = self.kv_heads, self.page, self.dh
        return (h * p * d, p * d, d, 1) if self.order == "head" else (h * p * d, d, h * d, 1)

    def upload(self):
        self.kb, self.vb = self._dev(self.k_bits), self._dev(self.v_bits)
        self.sb = [self._dev(s) for s in self.scales]
        self.tb, self.lb, self.qb = (self.DB.from_array(x) for x in (self.table, self.lengths, self.q_bits))

    def pages(self, **kw):
        K = self.K
        st = self.strides()
        ss = (self.kv_heads * self.page, self.page, 1, 1) if self.order == "head" else (self.kv_heads * self.page, 1, self.kv_heads, 1)
        more = dict(k_scale=K.View(self.sb[0], ss), v_scale=K.View(self.sb[1], ss)) if self.kv == "i8" else {}
        args = dict(num_pages=self.num_pages, page_size=self.page, kv_heads=self.kv_heads, dh=self.dh, dtype=self.kv,
                    k=K.View(self.kb, st), v=K.View(self.vb, st), batch=len(self.lengths), table=self.tb,
                    table_ld=self.max_pages, max_pages=self.max_pages, lengths=self.lb, **more)
        args.update(kw)
        return K.PagedKV(**args)

    def attend(self, window=0, sinks=0, scale=None, i8=None, calls=1, **kw):
        K, DB = self.K, self.DB
        B, H, dh = len(self.lengths), self.heads, self.dh
        size = K.paged_attention_workspace(B, H, self.kv_heads, dh)
        ws = DB(size, zero=True)
        itemsize = np.dtype(R.NP[self.q_dtype]).itemsize
        out, lse = DB(B * H * dh * itemsize), DB(B * H * 4)
        o8 = DB(B * H * dh) if i8 else None
        st = (H * dh, dh, 0, 1)
        args = dict(kv=self.pages(), heads=H, q=K.View(self.qb, st), q_dtype=self.q_dtype,
                    scale=dh ** -0.5 if scale is None else scale, window=window, sinks=sinks, out=K.View(out, st), lse=lse,
                    out_i8=K.View(o8, st, itemsize=1) if i8 else None, out_scale=i8 or 1.0, workspace=ws, workspace_bytes=size)
        args.update(kw)
        plan = K.PagedAttn(**args).struct()
        for _ in range(calls):
            K.paged_attention(plan)
        from mira_b200 import _lib
        _lib.call("mira_cuda_sync")
        o = R.from_bits(out.download((B, H, dh), R.NP[self.q_dtype]), self.q_dtype)
        got = (o, lse.download((B, H), np.float32))
        return got + (o8.download((B, H, dh), np.int8),) if i8 else got

    def check(self, window=0, sinks=0, **kw):
        got, lse = self.attend(window, sinks, **kw)[:2]
        q = R.from_bits(self.q_bits, self.q_dtype)
        o, want_lse, bo, bl = R.attention(q, self.k_val, self.v_val, self.table, self.lengths, self.page,
                                          np.float64(np.float32(kw.get("scale") or self.dh ** -0.5)), window, sinks)
        assert np.isfinite(got).all()
        bound = bo + np.abs(o) * R.UNIT[self.q_dtype] + (2.0 ** -25 if self.q_dtype == "f16" else 0)
        off = np.abs(got - o)
        assert (off <= bound).all(), (float((off / np.maximum(bound, 1e-300)).max()), np.argwhere(off > bound)[:3].tolist())
        empty = ~np.isfinite(want_lse)
        assert (lse[empty] == -np.inf).all()
        assert (np.abs(lse[~empty] - want_lse[~empty]) <= bl[~empty]).all()


RAGGED = [0, 1, 2, 15, 16, 17, 31, 33, 64, 100, 129, 300]
KINDS = [("f32", "f32"), ("f16", "f16"), ("bf16", "bf16"), ("f32", "f16"), ("f32", "bf16"), ("bf16", "f16"), ("f16", "f32"),
         ("f32", "i8"), ("f16", "i8"), ("bf16", "i8")]


@pytest.mark.parametrize("q,kv", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dh", [(12, 12, 64), (8, 2, 128), (6, 2, 80)])
def test_attention_types(cuda_device, q, kv, heads, kv_heads, dh):
    Case(heads * dh, kv, heads, kv_heads, dh, 16, RAGGED, q=q).check()


@pytest.mark.parametrize("kv,heads,kv_heads,dh", [
    (kv, *h) for kv in ("f32", "bf16", "i8") for h in
    [(1, 1, 32), (2, 1, 64), (5, 5, 40), (9, 3, 96), (4, 1, 112), (5, 1, 64), (12, 2, 72), (7, 1, 128), (8, 1, 160),
     (16, 1, 256), (24, 1, 64), (34, 2, 32), (3, 3, 36), (2, 2, 1), (6, 3, 7), (4, 1, 250), (33, 1, 17)]])
def test_attention_heads_and_sizes(cuda_device, kv, heads, kv_heads, dh):
    Case(heads * 7 + dh, kv, heads, kv_heads, dh, 5, [40, 0, 129, 1, 16], q="f32").check()


@pytest.mark.parametrize("kv,group", [("f32", 1), ("bf16", 4), ("i8", 5), ("f16", 2)])
@pytest.mark.parametrize("page", [1, 3, 16, 100, 512])
def test_attention_page_sizes_and_orders(cuda_device, kv, group, page):
    for order in ("head", "token"):
        Case(page, kv, 2 * group, 2, 64, page, [257, 31, 1, 0, 600], order=order, shared=True).check()


@pytest.mark.parametrize("kv,group", [("f32", 1), ("bf16", 4), ("i8", 3), ("f16", 8)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (1, 4), (7, 3), (64, 1), (100, 17), (299, 2), (300, 5), (5000, 9), (33, 5000),
                                          (1 << 40, 1 << 40)])
def test_attention_window_and_sinks(cuda_device, kv, group, window, sinks):
    c = Case(window % 97 + sinks % 89, kv, 2 * group, 2, 64, 16, RAGGED)
    c.check(window, sinks)
    # what the window hides is not read into the result, whatever it holds
    t = c.table[11, (np.arange(300) // 16)]
    hidden = np.setdiff1d(np.arange(300), R.visible(300, window, sinks))
    if len(hidden):
        for a in (c.scales if kv == "i8" else (c.k_bits, c.v_bits)):
            a[t[hidden], :, hidden % 16] = np.inf if kv == "i8" else R.to_bits(np.float32(np.inf), kv)
        c.upload()
        c.check(window, sinks)


@pytest.mark.parametrize("kv,heads,kv_heads,dh,lengths", [
    ("bf16", 8, 2, 128, [20000]), ("f32", 3, 3, 64, [9999, 5]), ("i8", 16, 2, 64, [7000] * 3 + [1]),
    ("f16", 32, 1, 64, [4097]), ("f32", 1, 1, 16, [70001]), ("bf16", 40, 40, 64, [1] * 200 + [3000] + [0] * 100)])
def test_attention_split_and_joined(cuda_device, kv, heads, kv_heads, dh, lengths):
    """Long sequences are cut into parts on many blocks; short ones share a block."""
    c = Case(len(lengths) + dh, kv, heads, kv_heads, dh, 16, lengths)
    c.check(calls=3)                            # the workspace is ready again after every call
    a, b = c.attend(), c.attend()
    assert np.array_equal(a[0], b[0]) and np.array_equal(a[1], b[1])


def test_attention_many_sequences(cuda_device):
    """More sequences than a block has threads."""
    rng = np.random.default_rng(2)
    Case(1, "bf16", 4, 1, 64, 16, rng.integers(0, 40, 1500).tolist()).check()


@pytest.mark.parametrize("kv", ["f32", "bf16", "f16", "i8"])
def test_attention_one_key_decides(cuda_device, kv):
    """Scores hundreds apart: all but one weight underflow, in whatever order the tiles come."""
    c = Case(3, kv, 4, 2, 64, 16, [500, 40], scale_q=60.0)
    c.check()
    c.check(scale=-0.5)
    c.check(scale=1e-30)


def test_attention_scores_of_minus_infinity(cuda_device):
    """Keys whose score is -inf weigh nothing; a sequence of only such keys gives 0 and -inf."""
    c = Case(4, "f32", 2, 2, 32, 16, [50, 20], fill="zero")
    c.q_bits[:] = np.abs(c.q_bits)
    half = c.table[0, np.arange(25) // 16], np.arange(25) % 16
    c.k_bits[half[0], :, half[1], 3] = -np.inf
    all_of = c.table[1, np.arange(20) // 16], np.arange(20) % 16
    c.k_bits[all_of[0], :, all_of[1], 0] = -np.inf
    c.upload()
    o, lse = c.attend()
    assert (o[1] == 0).all() and (lse[1] == -np.inf).all()
    # sequence 0 equals the same sequence without the first 25 keys
    keep = np.arange(25, 50)
    for h in range(2):
        kk = c.k_val[c.table[0, keep // 16], h, keep % 16].astype(np.float64)
        vv = c.v_val[c.table[0, keep // 16], h, keep % 16].astype(np.float64)
        s = kk @ c.q_bits[0, h].astype(np.float64) * 32 ** -0.5
        p = np.exp(s - s.max())
        np.testing.assert_allclose(o[0, h], p @ vv / p.sum(), rtol=0, atol=2e-5)


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("kv,heads", [("f32", 2), ("bf16", 8)])
def test_attention_visible_nan_shows(cuda_device, kv, heads, bad):
    c = Case(5, kv, heads, 1, 64, 16, [70, 70])
    c.v_bits[c.table[0, 2], 0, 3, 5] = R.to_bits(np.float32(bad), kv)
    c.upload()
    o, lse = c.attend()
    if np.isnan(bad):
        assert np.isnan(o[0, :, 5]).all()
    else:
        assert (~np.isfinite(o[0, :, 5])).all()
    rest = np.arange(64) != 5
    assert np.isfinite(o[0][:, rest]).all() and np.isfinite(o[1]).all() and np.isfinite(lse).all()


@pytest.mark.parametrize("kv,group", [("f32", 1), ("bf16", 4)])
def test_attention_strides(cuda_device, kv, group):
    """Queries as columns of a wider buffer, transposed outputs, padded pages."""
    c = Case(6, kv, 2 * group, 2, 64, 16, [33, 90, 5])
    K, DB = c.K, c.DB
    B, H, dh = 3, 2 * group, 64
    wide = np.zeros((B, 3, H, dh), np.float32)
    wide[:, 1] = c.q_bits
    qb = DB.from_array(wide)
    padded_k = np.full((c.num_pages, 2, 20, 72), 1e30, np.float32)
    padded_k[:, :, :16, :64] = R.from_bits(c.k_bits, kv)
    kb = DB.from_array(R.to_bits(padded_k, kv))
    out = DB(B * H * dh * 4)
    got, lse = c.attend(kv=c.pages(k=K.View(kb, (2 * 20 * 72, 20 * 72, 72, 1))), q=K.View(qb, (3 * H * dh, dh, 0, 1), offset=H * dh),
                        out=K.View(out, (dh, B * dh, 0, 1)))
    want, want_lse = c.attend()
    np.testing.assert_array_equal(out.download((H, B, dh), np.float32).transpose(1, 0, 2), want)
    np.testing.assert_array_equal(lse, want_lse)


@pytest.mark.parametrize("kv,group,offset", [("bf16", 4, 1), ("bf16", 4, 4), ("f32", 1, 1), ("f32", 2, 2), ("i8", 4, 3), ("i8", 4, 8),
                                             ("f16", 1, 3)])
def test_attention_unaligned_pages(cuda_device, kv, group, offset):
    """Pages that start off a 16-byte boundary take another access width, with the same result."""
    c = Case(7, kv, 2 * group, 2, 64, 16, [33, 90, 0, 5])
    item = np.dtype(R.NP[kv]).itemsize
    for name in ("kb", "vb"):
        bits = (c.k_bits if name == "kb" else c.v_bits).ravel()
        buf = np.zeros(bits.size + offset, bits.dtype)
        buf[offset:] = bits
        setattr(c, name, c.DB.from_array(buf))
    K = c.K
    st = c.strides()
    pages = c.pages(k=K.View(c.kb, st, offset=offset, itemsize=item), v=K.View(c.vb, st, offset=offset, itemsize=item))
    c.check(kv=pages)


def test_attention_int8_output(cuda_device):
    c = Case(8, "f32", 4, 4, 64, 16, [33, 90, 0, 5])
    o, _, o8 = c.attend(i8=0.013)
    want = np.clip(np.rint(o / np.float32(0.013)), -127, 127).astype(np.int8)
    np.testing.assert_array_equal(o8, want)


@pytest.mark.parametrize("kv,heads", [("f16", 1), ("bf16", 8)])
def test_attention_offsets_beyond_32_bits(cuda_device, kv, heads):
    """Pages more than 2^31 elements into the pool."""
    K, DB = _k()
    c = Case(9, kv, heads, 1, 64, 16, [40, 17])
    per = 16 * 64
    far = (1 << 31) // per + 11
    pool = DB((far + c.num_pages) * per * 2)
    k_off = far * per
    for name, bits in (("k", c.k_bits), ("v", c.v_bits)):
        pool.upload(bits, offset=k_off * 2)
        big = K.View(pool, (per, per, 64, 1))
        c.table_far = np.where(c.table >= 0, c.table + far, c.table).astype(np.int32)
        tb = DB.from_array(c.table_far)
        other = c.pages()
        pages = c.pages(num_pages=far + c.num_pages, table=tb, **{name: big})
        # the other of the two stays in its small pool, addressed from a base that far below it
        small = K.View((c.vb if name == "k" else c.kb).ptr - far * per * 2, (per, per, 64, 1))
        setattr(pages, "v" if name == "k" else "k", small)
        got = c.attend(kv=pages)
        want = c.attend(kv=other)
        np.testing.assert_array_equal(got[0], want[0])


def test_attention_bad_tables_are_reported_not_read(cuda_device):
    from mira_b200 import _lib
    for kv, heads in (("f32", 2), ("bf16", 8), ("i8", 8)):
        for what in ("page", "negative page", "length", "negative length"):
            c = Case(10, kv, heads, 2, 64, 16, [40, 17])
            if what.endswith("page"):
                c.table[0, 1] = -1 if what.startswith("neg") else c.num_pages
            else:
                c.lengths[0] = -5 if what.startswith("neg") else c.max_pages * 16 + 1
            c.upload()
            with pytest.raises(_lib.CudaError) as e:
                c.attend()
            assert e.value.code == _lib.EKERNEL and "page" in str(e.value)
            c = Case(10, kv, heads, 2, 64, 16, [40, 17])
            c.check()                                # the device goes on


def test_attention_refusals(cuda_device):
    from mira_b200 import _lib
    c = Case(11, "bf16", 8, 2, 64, 16, [40, 17])
    K = c.K
    size = K.paged_attention_workspace(2, 8, 2, 64)
    assert size > 0
    assert K.paged_attention_workspace(2, 7, 2, 64) == 0 and K.paged_attention_workspace(0, 8, 2, 64) == 0
    assert K.paged_attention_workspace(2, 8, 2, 257) == 0
    small = c.DB(size, zero=True)
    cases = [dict(heads=7), dict(heads=0), dict(scale=np.inf), dict(window=-1), dict(sinks=-1), dict(out=None),
             dict(workspace=None), dict(workspace_bytes=size - 1), dict(q=K.View(None, (1, 1, 1, 1))),
             dict(q_dtype="i8"), dict(workspace=small.ptr + 4), dict(q=K.View(c.qb.ptr + 1, (512, 64, 0, 1)))]
    cases += [dict(kv=c.pages(**kw)) for kw in (dict(dh=257), dict(dh=0), dict(num_pages=0), dict(page_size=0), dict(kv_heads=0),
                                               dict(max_pages=0), dict(table_ld=1, max_pages=2), dict(table=None),
                                               dict(lengths=None), dict(batch=-1), dict(k=K.View(None, (1, 1, 1, 1))),
                                               dict(k=K.View(c.kb, (2048, 1024, 64, 2))), dict(dtype="i8"),
                                               dict(page_size=1 << 20, max_pages=1 << 20, table_ld=1 << 20))]
    for kw in cases:
        with pytest.raises(_lib.CudaError) as e:
            c.attend(**kw)
        assert e.value.code == _lib.EINVAL, kw
    with pytest.raises(ValueError):
        c.pages(dtype="f64").struct()
    c.check()


def test_attention_empty_batch_launches_nothing(cuda_device):
    from mira_b200 import _lib
    c = Case(12, "f32", 2, 2, 64, 16, [3])
    before = _lib.launch_count()
    c.K.paged_attention(c.K.PagedAttn(kv=c.pages(batch=0), heads=2, q=c.K.View(c.qb, (128, 64, 0, 1)), scale=1.0,
                                      out=c.K.View(c.qb, (128, 64, 0, 1))))
    assert _lib.launch_count() == before


# ------------------------------------------------------------------------------------------- append

def _append(c, news, src, keys, values, row_start="given", rows=None, **kw):
    K, DB = c.K, c.DB
    h, d = c.kv_heads, c.dh
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    kb, vb = DB.from_array(R.to_bits(keys, src)), DB.from_array(R.to_bits(values, src))
    sb = DB.from_array(starts) if isinstance(row_start, str) else row_start
    row = (0, d, h * d, 1)
    args = dict(kv=c.pages(), rows=int(starts[-1]) if rows is None else rows, src_dtype=src, k_new=K.View(kb, row),
                v_new=K.View(vb, row), row_start=sb)
    args.update(kw)
    K.kv_append(K.KvAppend(**args))
    from mira_b200 import _lib
    _lib.call("mira_cuda_sync")


def _pages_of(c):
    shape = (c.num_pages, c.kv_heads, c.page, c.dh) if c.order == "head" else (c.num_pages, c.page, c.kv_heads, c.dh)
    got = [b.download(shape, R.NP[c.kv]) for b in (c.kb, c.vb)]
    sc = [b.download(shape[:3], np.float32) for b in c.sb]
    if c.order != "head":
        got, sc = [np.swapaxes(g, 1, 2) for g in got], [np.swapaxes(s, 1, 2) for s in sc]
    return got, sc


@pytest.mark.parametrize("src", ["f32", "f16", "bf16"])
@pytest.mark.parametrize("kv", ["f32", "f16", "bf16", "i8"])
@pytest.mark.parametrize("kv_heads,dh,page,order", [(12, 64, 16, "head"), (2, 128, 5, "token"), (3, 80, 16, "token"), (1, 7, 3, "head"),
                                                     (2, 256, 1, "head"), (5, 36, 16, "head")])
def test_append_bit_exact(cuda_device, src, kv, kv_heads, dh, page, order):
    """Every stored element is the one rounding of its value; nothing else in the pages changes."""
    lengths = [0, 1, 7, 40, 16, 33]
    news = [0, 1, 3, 40, 0, 17]
    c = Case(dh, kv, kv_heads, kv_heads, dh, page, lengths, order=order, fill="zero")
    rng = np.random.default_rng(dh + page)
    k_new, v_new = (rng.standard_normal((sum(news), kv_heads, dh)).astype(np.float32) * rng.choice([1e-6, 1, 300], (sum(news), 1, 1))
                    .astype(np.float32) for _ in range(2))
    k_new[0] = 0.0
    k_new, v_new = (R.from_bits(R.to_bits(x, src), src) for x in (k_new, v_new))
    want, want_s = [c.k_bits.copy(), c.v_bits.copy()], [s.copy() for s in c.scales]
    at = 0
    for b, (n, r) in enumerate(zip(lengths, news)):
        pos = np.arange(n - r, n)
        pg, sl = c.table[b, pos // page], pos % page
        for j, x in enumerate((k_new, v_new)):
            rows = x[at: at + r]
            if kv == "i8":
                codes, s = R.quantize_row(rows)
                want[j][pg, :, sl], want_s[j][pg, :, sl] = codes, s
            else:
                want[j][pg, :, sl] = R.to_bits(rows, kv)
        at += r
    _append(c, news, src, k_new, v_new)
    got, got_s = _pages_of(c)
    for g, w in zip(got, want):
        np.testing.assert_array_equal(g, w)
    for g, w in zip(got_s, want_s):
        np.testing.assert_array_equal(g, w)


def test_append_one_row_per_sequence(cuda_device):
    """The decode step's form without row_start; sequences of length 0 take no row."""
    c = Case(20, "bf16", 2, 2, 64, 16, [5, 0, 16, 17], fill="zero")
    x = np.random.default_rng(1).standard_normal((2, 4, 2, 64)).astype(np.float32)
    want = c.k_bits.copy()
    _append(c, [1, 1, 1, 1], "f32", x[0], x[1], row_start=None)
    for b, n in enumerate([5, 0, 16, 17]):
        if n:
            want[c.table[b, (n - 1) // 16], :, (n - 1) % 16] = R.to_bits(x[0, b], "bf16")
    np.testing.assert_array_equal(_pages_of(c)[0][0], want)


def test_append_strided_rows(cuda_device):
    """Keys and values as column ranges of a fused projection's output."""
    c = Case(21, "f32", 3, 3, 40, 16, [9, 30], fill="zero")
    K, DB = c.K, c.DB
    rng = np.random.default_rng(3)
    wide = rng.standard_normal((7, 3 * 3 * 40)).astype(np.float32)      # [row][q | k | v][head][dh]
    wb = DB.from_array(wide)
    starts = DB.from_array(np.array([0, 2, 7], np.int32))
    row = (0, 40, 360, 1)
    K.kv_append(K.KvAppend(kv=c.pages(), rows=7, k_new=K.View(wb, row, offset=120), v_new=K.View(wb, row, offset=240), row_start=starts))
    (k, v), _ = _pages_of(c)
    for r, (b, pos) in enumerate([(0, 7), (0, 8), (1, 25), (1, 26), (1, 27), (1, 28), (1, 29)]):
        np.testing.assert_array_equal(k[c.table[b, pos // 16], :, pos % 16], wide[r, 120:240].reshape(3, 40))
        np.testing.assert_array_equal(v[c.table[b, pos // 16], :, pos % 16], wide[r, 240:].reshape(3, 40))


def test_append_then_attend_is_the_attention_of_the_new_rows(cuda_device):
    """Rows go in as a prompt, then one by one; attention over the pages sees them."""
    rng = np.random.default_rng(4)
    c = Case(22, "i8", 6, 2, 64, 16, [50, 3, 0], fill="zero")
    x = rng.standard_normal((2, 53, 2, 64)).astype(np.float32)
    _append(c, [50, 3, 0], "f32", x[0], x[1])
    codes, scales = _pages_of(c)
    c.k_val, c.v_val = (q.astype(np.float64) * s[..., None] for q, s in zip(codes, scales))
    c.check()
    t = np.arange(50)
    assert np.abs(c.k_val[c.table[0, t // 16], :, t % 16] - x[0, :50]).max() <= np.abs(x[0]).max() / 254 * 1.0001


def test_append_bad_rows_are_reported_not_written(cuda_device):
    from mira_b200 import _lib
    for what in ("page", "length", "rows"):
        c = Case(23, "f32", 2, 2, 64, 16, [20, 17], fill="zero")
        news = [2, 2]
        if what == "page":
            c.table[0, 1] = c.num_pages
        elif what == "length":
            c.lengths[0] = c.max_pages * 16 + 1
        else:
            news = [21, 2]
        c.upload()
        x = np.ones((sum(news), 2, 64), np.float32)
        with pytest.raises(_lib.CudaError) as e:
            _append(c, news, "f32", x, x)
        assert e.value.code == _lib.EKERNEL


def test_append_refusals(cuda_device):
    from mira_b200 import _lib
    c = Case(24, "f32", 2, 2, 64, 16, [20, 17], fill="zero")
    K = c.K
    x = np.ones((2, 2, 64), np.float32)
    row = (0, 64, 128, 1)
    for kw in (dict(rows=-1), dict(row_start=None, rows=3), dict(k_new=K.View(None, row)), dict(src_dtype="i8"),
               dict(v_new=K.View(c.kb, (0, 64, 128, 2))), dict(k_new=K.View(c.kb.ptr + 2, row)), dict(kv=c.pages(batch=0))):
        with pytest.raises(_lib.CudaError) as e:
            _append(c, [1, 1], "f32", x, x, **kw)
        assert e.value.code == _lib.EINVAL, kw
    _append(c, [1, 1], "f32", x, x)
    before = _lib.launch_count()
    _append(c, [0, 0], "f32", x, x)
    assert _lib.launch_count() == before


# --------------------------------------------------------------------------------------------- copy

@pytest.mark.parametrize("planes,pages,page_bytes,stride,n", [(1, 4, 16, 16, 1), (2, 9, 3072, 3072, 4), (24, 40, 49152, 49152, 11),
                                                              (3, 1200, 272, 272, 600), (2, 50, 1000, 1024, 20), (1, 30, 7, 9, 15),
                                                              (5, 20, 40000, 40000, 10)])
def test_page_copy(cuda_device, planes, pages, page_bytes, stride, n):
    K, DB = _k()
    rng = np.random.default_rng(pages)
    plane = pages * stride + 32 * (planes > 1)
    pool = rng.integers(0, 256, planes * plane).astype(np.uint8)
    ids = rng.permutation(pages)
    src, dst = rng.choice(ids[n:], n), ids[:n]         # a page may be a source several times
    want = pool.copy()
    for p in range(planes):
        for a, b in zip(src, dst):
            want[p * plane + b * stride: p * plane + b * stride + page_bytes] = \
                pool[p * plane + a * stride: p * plane + a * stride + page_bytes]
    buf = DB.from_array(pool)
    K.page_copy([K.PageRegion(buf, page_bytes=page_bytes, page_stride=stride, planes=planes, plane_stride=plane)], pages, src, dst)
    np.testing.assert_array_equal(buf.download(pool.shape, np.uint8), want)


@pytest.mark.parametrize("n", [31, 32, 33, 255, 256, 257, 999, 1000, 1001, 2001])
def test_page_copy_around_launch_sizes(cuda_device, n):
    """As many pages as one launch takes, one fewer and one more, and several launches."""
    test_page_copy(cuda_device, 2, 2 * n + 3, 48, 64, n)


def test_page_copy_several_regions(cuda_device):
    """Keys, values and their scales in one call, regions of different sizes and alignments."""
    K, DB = _k()
    rng = np.random.default_rng(5)
    sizes = [(4, 4096), (4, 4096), (4, 132), (1, 50000)]
    bufs, pools = [], []
    for planes, nbytes in sizes:
        pools.append(rng.integers(0, 256, (planes, 30, nbytes)).astype(np.uint8))
        bufs.append(DB.from_array(pools[-1]))
    src, dst = np.array([3, 3, 17, 29], np.int32), np.array([0, 8, 20, 1], np.int32)
    K.page_copy([K.PageRegion(b, page_bytes=n, page_stride=n, planes=p, plane_stride=30 * n) for b, (p, n) in zip(bufs, sizes)], 30, src, dst)
    for b, pool in zip(bufs, pools):
        want = pool.copy()
        want[:, dst] = pool[:, src]
        np.testing.assert_array_equal(b.download(pool.shape, np.uint8), want)


def test_page_copy_refusals(cuda_device):
    from mira_b200 import _lib
    K, DB = _k()
    pool = np.arange(80, dtype=np.uint8)
    buf = DB.from_array(pool)
    r = [K.PageRegion(buf, page_bytes=8, page_stride=8)]
    for src, dst in (([0], [10]), ([10], [0]), ([-1], [0]), ([0], [-1]), ([0, 1], [2, 2]), ([0, 1], [1, 2]), ([3], [3]),
                     (list(range(11)), list(range(11)))):
        with pytest.raises(_lib.CudaError) as e:
            K.page_copy(r, 10, src, dst)
        assert e.value.code == _lib.EINVAL
    for bad in (dict(page_bytes=0), dict(page_stride=7), dict(planes=0), dict(base=None), dict(plane_stride=-8)):
        with pytest.raises(_lib.CudaError):
            K.page_copy([K.PageRegion(**{**dict(base=buf, page_bytes=8, page_stride=8), **bad})], 10, [0], [1])
    with pytest.raises(ValueError):
        K.page_copy(r, 10, [0, 1], [2])
    with pytest.raises(ValueError):
        K.page_copy([], 10, [0], [2])
    np.testing.assert_array_equal(buf.download((80,), np.uint8), pool)
    before = _lib.launch_count()
    K.page_copy(r, 10, [], [])
    assert _lib.launch_count() == before
    assert C.sizeof(_lib.PageRegion) == 40

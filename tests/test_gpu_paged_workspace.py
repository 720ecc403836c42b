"""One workspace, zeroed once, under calls of different sizes in turn: every call has to find it as the
calls before left it, whatever their sizes and whichever of the two operators they were."""
import numpy as np
import pytest

import paged_ref as R
from test_gpu_paged import Case
from test_gpu_paged_decode import _host_logits
from test_gpu_w4 import Product

pytestmark = pytest.mark.gpu


def _k():
    from mira_b200 import kernels as K
    from mira_b200.device import DeviceBuffer
    return K, DeviceBuffer


def _nan(buf):
    """Fills a buffer with NaN, so that a result that is not written shows."""
    buf.upload(np.full(buf.nbytes // 4, np.nan, np.float32))


def _sync():
    from mira_b200 import _lib
    _lib.call("mira_cuda_sync")


class _W4:
    """A product whose scratch is given, and its check against the formula."""

    def __init__(self, m, n, k, group=32, x="f32"):
        self.p = Product(m, n, k, group, x, "f32", "f32")
        self.size = self.p.K.w4_matvec_workspace(m, n, k)

    def run(self, ws, size):
        p = self.p
        _nan(p.out)
        p.K.w4_matvec(p.desc(workspace=ws, workspace_bytes=size).struct())
        _sync()
        got = p.out.download((p.m, p.n), np.float32)
        want, bound = p.exact()
        off = np.abs(got - want)
        assert (off <= bound + np.abs(want) * R.UNIT["f32"] * 1.01).all(), (p.m, p.n, p.k, int((~(off <= bound)).sum()))


class _Attention:
    """One attention call whose scratch is given; the same call with scratch of its own says what is right."""

    def __init__(self, seed, kv, heads, kv_heads, dh, lengths):
        self.c = Case(seed, kv, heads, kv_heads, dh, 16, lengths)
        self.size = self.c.K.paged_attention_workspace(len(lengths), heads, kv_heads, dh)
        self.want = self.c.attend()

    def run(self, ws, size):
        K, DB = _k()
        c = self.c
        B, H, dh = len(c.lengths), c.heads, c.dh
        out, lse = DB(B * H * dh * 4), DB(B * H * 4)
        _nan(out)
        _nan(lse)
        c.attend(workspace=ws, workspace_bytes=size, out=K.View(out, (H * dh, dh, 0, 1)), lse=lse)
        np.testing.assert_array_equal(out.download((B, H, dh), np.float32), self.want[0])
        np.testing.assert_array_equal(lse.download((B, H), np.float32), self.want[1])


def _in_turn(calls):
    K, DB = _k()
    size = max(c.size for c in calls)
    ws = DB(size, zero=True)
    for _ in range(2):
        for c in calls:
            c.run(ws, size)
    for c in reversed(calls):
        c.run(ws, size)


@pytest.mark.parametrize("shapes", [
    # projections of a transformer of width 1024 and its head, 16 sequences: cut in two or four along k
    [(16, 512, 1024), (16, 3072, 1024), (16, 4096, 1024), (16, 1024, 4096)],
    # few and many row groups
    [(1, 64, 40000), (1, 3000, 9000), (12, 1000, 6000), (33, 2000, 8000)]])
def test_products_of_different_sizes(cuda_device, shapes):
    calls = [_W4(*s) for s in shapes]
    assert sum(c.size > 0 for c in calls) >= 3          # cut along k, so that the scratch is used
    _in_turn(calls)


def test_attention_of_different_batches(cuda_device):
    rng = np.random.default_rng(0)
    _in_turn([_Attention(1, "bf16", 8, 2, 128, [9000]),
              _Attention(2, "f32", 12, 12, 64, rng.integers(0, 400, 64).tolist()),
              _Attention(3, "i8", 16, 2, 64, [3000] * 5),
              _Attention(4, "bf16", 4, 4, 64, rng.integers(1, 90, 700).tolist()),
              _Attention(5, "f16", 3, 1, 33, [1200, 0, 800])])


def test_attention_and_products_share(cuda_device):
    _in_turn([_Attention(6, "bf16", 8, 2, 128, [5000, 40]), _W4(16, 4096, 1024), _W4(2, 300, 8000, 64, "bf16"),
              _Attention(7, "f32", 4, 4, 64, [700] * 90), _W4(16, 512, 1024)])


def test_transformer_whose_projections_are_cut(cuda_device):
    """Width 1024: the projections have one scratch buffer and different cuts; three steps of 16 sequences."""
    from mira_b200.paged_decode import PagedTransformer, random_weights
    import test_gpu_paged_decode as T
    w = random_weights(layers=1, d_model=1024, d_mlp=4096, vocab=512, max_seq=16, seed=3)
    model = PagedTransformer(w, T.HEADS, num_pages=16, page_size=8, batch=16, kv_dtype="f32", group=32)
    slots = [model.cache.open() for _ in range(16)]
    rng = np.random.default_rng(1)
    tokens = rng.integers(0, 512, (3, 16))
    got = []
    for t in range(3):
        out = model.step({s: int(tokens[t, s]) for s in slots})
        got.append(np.stack([out[s] for s in slots]))
    got = np.stack(got)
    for s in slots:
        want = _host_logits(w, model, tokens[:, s])
        assert np.abs(got[:, s] - want).max() <= 2e-5 * np.abs(want).max(), s
    model.close()

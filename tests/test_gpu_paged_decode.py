"""The paged operators together: a small transformer with 4-bit weights decoding sequences of different
lengths over paged caches, against the same model in 64 bits on the host."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

HEADS = 4


def _model(kv_dtype="f32", **kw):
    from mira_b200.paged_decode import PagedTransformer, random_weights
    w = random_weights(layers=2, d_model=128, d_mlp=256, vocab=50, max_seq=200, seed=1)
    for b in w["blocks"]:      # attention that looks at something
        b["qkv"] = (b["qkv"][0] * 6, b["qkv"][1])
    return w, PagedTransformer(w, HEADS, num_pages=60, page_size=8, batch=5, kv_dtype=kv_dtype, group=64, **kw)


def _host_logits(w, model, tokens, window=0, sinks=0):
    """Logits after each token, from the dequantized 4-bit weights, in 64 bits."""
    lin = lambda l, x: x @ l.dequantized.T.astype(np.float64) + l.b.download((l.n,), np.float32)
    norm = lambda x, ln: (x - x.mean(-1, keepdims=True)) / np.sqrt(x.var(-1, keepdims=True) + 1e-5) * ln[0] + ln[1]
    d = w["embed"].shape[1]
    n, dh = len(tokens), d // HEADS
    h = w["embed"][tokens].astype(np.float64) + w["position"][:n]
    at = np.arange(n)
    see = at[None, :] <= at[:, None]
    if window:
        see &= (at[None, :] > at[:, None] - window) | (at[None, :] < sinks)
    for raw, b in zip(w["blocks"], model.blocks):
        q, k, v = np.split(lin(b["qkv"], norm(h, raw["ln1"])), 3, axis=1)
        o = np.zeros_like(q)
        for i in range(HEADS):
            c = slice(i * dh, (i + 1) * dh)
            s = np.where(see, q[:, c] @ k[:, c].T * dh ** -0.5, -np.inf)
            p = np.exp(s - s.max(1, keepdims=True))
            o[:, c] = p / p.sum(1, keepdims=True) @ v[:, c]
        h = h + lin(b["out"], o)
        m = lin(b["up"], norm(h, raw["ln2"]))
        m = 0.5 * m * (1 + np.tanh(np.sqrt(2 / np.pi) * (m + 0.044715 * m ** 3)))
        h = h + lin(b["down"], m)
    return lin(model.head, norm(h, w["ln"]))


# relative to the largest logit: f32 pages carry the f32 arithmetic of a few dozen operations; 16-bit and
# 8-bit pages round keys and values once, by 2^-11, 2^-9 and 2^-8 of a row's values
@pytest.mark.parametrize("kv_dtype,tol", [("f32", 2e-5), ("f16", 2e-3), ("bf16", 1.5e-2), ("i8", 2e-2)])
@pytest.mark.parametrize("graph", [True, False])
def test_ragged_batch_with_forks(cuda_device, kv_dtype, tol, graph):
    w, model = _model(kv_dtype, graph=graph)
    rng = np.random.default_rng(0)
    cache = model.cache
    a, b = cache.open(), cache.open()
    fed = {a: [], b: []}
    got = {a: [], b: []}

    def feed(slots):
        tokens = {s: int(rng.integers(50)) for s in slots}
        out = model.step(tokens)
        for s in slots:
            fed[s].append(tokens[s])
            got[s].append(out[s])

    for i in range(21):
        feed([a] if i % 3 else [a, b])                  # different lengths, one idle at times
    c = cache.fork(a)                                   # shares two pages, copies the third
    fed[c], got[c] = list(fed[a]), list(got[a])
    for i in range(12):
        feed([a, b, c])
    cache.close(a)                                      # its own pages go back, the shared ones stay
    moved = cache.compact()
    d = cache.open()
    fed[d], got[d] = [], []
    for i in range(9):
        feed([b, c, d])
    assert moved > 0
    for s in (a, b, c, d):
        want = _host_logits(w, model, np.array(fed[s]))
        scale = np.abs(want).max()
        assert np.abs(np.array(got[s]) - want).max() <= tol * scale, (s, np.abs(np.array(got[s]) - want).max() / scale)
    model.close()


def test_window_and_trimmed_pages(cuda_device):
    """With a window, pages that nothing sees any more go back to the pool without changing a result."""
    w, model = _model("f32", window=11, sinks=3)
    slot = model.cache.open()
    rng = np.random.default_rng(3)
    tokens = rng.integers(0, 50, 70)
    got, freed = [], 0
    for t in tokens:
        got.append(model.step({slot: int(t)})[slot])
        freed += model.cache.trim(slot, 11, 3)
    want = _host_logits(w, model, tokens, 11, 3)
    assert np.abs(np.array(got) - want).max() <= 2e-5 * np.abs(want).max()
    assert freed >= 6 and model.cache.pages.used_pages() <= 4
    model.close()


def test_generate_is_greedy(cuda_device):
    w, model = _model("f32")
    slot, out = model.generate([3, 7, 1], 6)
    tokens = [3, 7, 1]
    for t in out:
        want = _host_logits(w, model, np.array(tokens))[-1]
        assert want[t] >= want.max() - 1e-4
        tokens.append(t)
    model.close()


def test_step_refusals_change_nothing(cuda_device):
    from mira_b200.paged import OutOfPages
    w, model = _model("f32", max_pages=3)
    a = model.cache.open()
    for bad in ({a: 50}, {a: -1}, {a + 1: 0}, {-1: 0}):
        with pytest.raises(ValueError):
            model.step(bad)
    for t in range(24):
        model.step({a: t})
    with pytest.raises(OutOfPages):
        model.step({a: 0})
    assert model.cache.pages.lengths[a] == 24
    model.close()

"""Decoding a batch of sequences of different lengths with 4-bit weights and paged keys and values:
the decoder-only transformer of configs.transformer (pre-LayerNorm GPT block, reference
examples/gpt.mira) as a loop over the paged operators of kernels.py.

    model = PagedTransformer(weights, heads=12, num_pages=4096, batch=64)
    a = model.cache.open()
    logits = model.step({a: token})              # f32 [vocab] per sequence that was fed
    b = model.cache.fork(a)                      # continues with a's tokens from here on

Every step is the same sequence of launches over the whole batch (slots without a token this step
are computed and ignored; their lengths do not change), so it is captured once as a CUDA graph;
token ids, positions, lengths and the page table are device memory.
"""
from __future__ import annotations

import ctypes as C
from typing import Mapping, Optional

import numpy as np

from . import _lib
from . import kernels as K
from .device import DeviceBuffer, DeviceSlice
from .paged import OutOfPages, PagedCache


def random_weights(layers: int = 2, d_model: int = 64, d_mlp: int = 128, vocab: int = 64, max_seq: int = 256, seed: int = 0) -> dict:
    """Weights N(0, 0.02) in the layout PagedTransformer takes: matrices [out, in], f32."""
    rng = np.random.default_rng(seed)

    def normal(*shape):
        return (rng.standard_normal(shape) * 0.02).astype(np.float32)

    def block():
        return {"ln1": (1 + normal(d_model), normal(d_model)), "ln2": (1 + normal(d_model), normal(d_model)),
                "qkv": (normal(3 * d_model, d_model), normal(3 * d_model)), "out": (normal(d_model, d_model), normal(d_model)),
                "up": (normal(d_mlp, d_model), normal(d_mlp)), "down": (normal(d_model, d_mlp), normal(d_model))}

    return {"embed": normal(vocab, d_model), "position": normal(max_seq, d_model), "blocks": [block() for _ in range(layers)],
            "ln": (1 + normal(d_model), normal(d_model)), "head": (normal(vocab, d_model), np.zeros(vocab, np.float32))}


class _Linear:
    """A 4-bit weight matrix with its bias on the device."""

    def __init__(self, w: np.ndarray, b: np.ndarray, group: int):
        self.n, self.k = w.shape
        self.group = group
        q, s = K.w4_quantize(w, group)
        self.dequantized = q * np.repeat(s, group, axis=1)[:, : self.k]
        packed = K.w4_weight(q)
        self.w, self.s, self.b = DeviceBuffer.from_array(packed), DeviceBuffer.from_array(s), DeviceBuffer.from_array(b)
        self.ld_w, self.ld_s = packed.shape[1], s.shape[1]

    def call(self, m: int, x, out, steps, workspace, workspace_bytes):
        return K.W4Matvec(m=m, n=self.n, k=self.k, group=self.group, x=x, ld_x=self.k, w=self.w, ld_w=self.ld_w, scales=self.s,
                          ld_scales=self.ld_s, out=out, ld_out=self.n,
                          steps=[K.Step("add", "channel", ptr=self.b), *steps], workspace=workspace,
                          workspace_bytes=workspace_bytes).struct()


class PagedTransformer:
    """One decode step at a time over a PagedCache (`cache`): see the module's text."""

    def __init__(self, weights: dict, heads: int, num_pages: int, page_size: int = 16, batch: int = 8, kv_dtype: str = "bf16",
                 window: int = 0, sinks: int = 0, group: int = 32, max_pages: Optional[int] = None, graph: bool = True):
        self.d = d = weights["embed"].shape[1]
        if d % heads:
            raise ValueError("d_model must be a multiple of heads")
        self.heads, self.dh, self.batch = heads, d // heads, batch
        self.vocab, self.max_seq = weights["embed"].shape[0], weights["position"].shape[0]
        self.window, self.sinks = window, sinks
        self.cache = PagedCache(len(weights["blocks"]), heads, self.dh, num_pages, page_size, batch, max_pages, kv_dtype)
        up = DeviceBuffer.from_array
        self.embed, self.position = up(weights["embed"]), up(weights["position"])
        self.blocks = [{k: (_Linear(*v, group) if v[0].ndim == 2 else (up(v[0]), up(v[1]))) for k, v in b.items()} for b in weights["blocks"]]
        self.ln = (up(weights["ln"][0]), up(weights["ln"][1]))
        self.head = _Linear(*weights["head"], group)
        mlp = self.blocks[0]["up"].n
        f = lambda n: DeviceBuffer(batch * n * 4, zero=True)
        self.tok, self.pos = f(1), f(1)
        self.pe, self.h, self.x, self.qkv, self.o, self.m, self.logits = f(d), f(d), f(d), f(3 * d), f(d), f(mlp), f(self.vocab)
        size = max(16, max(K.w4_matvec_workspace(batch, n, k) for n, k in
                           [(3 * d, d), (d, d), (mlp, d), (d, mlp), (self.vocab, d)]))
        self.ws = DeviceBuffer(size, zero=True)
        self.att_ws_bytes = K.paged_attention_workspace(batch, heads, heads, self.dh)
        self.att_ws = DeviceBuffer(max(16, self.att_ws_bytes), zero=True)
        self._plan = self._build(size)
        self._graph = None
        self._use_graph = graph
        self._ran = False

    def _build(self, size: int) -> list:
        """The launches of a step, as (function, descriptor) with everything that stays the same built."""
        B, d, dh = self.batch, self.d, self.dh
        plan = []
        row = (3 * d, dh, 0, 1)
        add = lambda fn, *a: plan.append((fn, a))
        lin = lambda l, x, out, steps=(): add(K.w4_matvec, l.call(B, x, out, list(steps), self.ws, size))
        norm = lambda ln: add(K.layernorm_rows, self.h, B, d, d, ln[0], ln[1], 1e-5, self.x, d)
        add(K.embed_rows, self.position, self.max_seq, d, self.pos, B, self.pe, d)
        add(K.embed_rows, self.embed, self.vocab, d, self.tok, B, self.h, d, self.pe, B)
        for i, b in enumerate(self.blocks):
            kv = self.cache.layer(i)
            norm(b["ln1"])
            lin(b["qkv"], self.x, self.qkv)
            new = lambda part: K.View(DeviceSlice(self.qkv, part * d * 4), (0, dh, 3 * d, 1))
            add(K.kv_append, K.KvAppend(kv=kv, rows=B, k_new=new(1), v_new=new(2)).struct())
            add(K.paged_attention, K.PagedAttn(
                kv=kv, heads=self.heads, q=K.View(self.qkv, row), scale=dh ** -0.5, window=self.window, sinks=self.sinks,
                out=K.View(self.o, (d, dh, 0, 1)), workspace=self.att_ws, workspace_bytes=self.att_ws_bytes).struct())
            lin(b["out"], self.o, self.h, [K.Step("add", "full", ptr=self.h, ld=d)])
            norm(b["ln2"])
            lin(b["up"], self.x, self.m, [K.Step("gelu")])
            lin(b["down"], self.m, self.h, [K.Step("add", "full", ptr=self.h, ld=d)])
        norm(self.ln)
        lin(self.head, self.x, self.logits)
        return plan

    def _launch(self) -> None:
        if self._graph is not None:
            _lib.call("mira_cuda_graph_launch", self._graph)
            return
        if self._use_graph and self._ran:      # the first step set every kernel up
            _lib.call("mira_cuda_graph_begin")
            for fn, args in self._plan:
                fn(*args)
            g = C.c_void_p()
            _lib.call("mira_cuda_graph_end", C.byref(g))
            self._graph = g
            _lib.call("mira_cuda_graph_launch", g)
            return
        for fn, args in self._plan:
            fn(*args)
        self._ran = True

    def step(self, tokens: Mapping[int, int]) -> dict:
        """Feeds one token to each of the given slots; returns {slot: logits f32 [vocab]}."""
        pages = self.cache.pages
        for slot, t in tokens.items():
            if not 0 <= int(t) < self.vocab:
                raise ValueError(f"token {t} outside the vocabulary")
            if not 0 <= slot < self.batch or not pages.live[slot]:
                raise ValueError(f"no sequence in slot {slot}")
            if pages.lengths[slot] >= self.max_seq:
                raise ValueError(f"a sequence has at most {self.max_seq} positions")
        fresh = [s for s in tokens if pages.lengths[s] % pages.page_size == 0]
        if len(fresh) > pages.free_pages():
            raise OutOfPages(f"{len(fresh)} pages wanted, {pages.free_pages()} free")
        if any(pages.lengths[s] // pages.page_size >= pages.max_pages for s in fresh):
            raise OutOfPages(f"a sequence has at most {pages.max_pages} pages")
        tok, pos = np.zeros(self.batch, np.int32), np.zeros(self.batch, np.int32)
        for slot, t in tokens.items():
            tok[slot], pos[slot] = int(t), pages.lengths[slot]
            self.cache.extend(slot)
        # a slot that is not fed keeps its pages out of this step: its length reads 0
        kept = pages.lengths.copy()
        idle = np.ones(self.batch, bool)
        idle[list(tokens)] = False
        pages.lengths[idle] = 0
        try:
            self.cache.sync_tables()
        finally:
            pages.lengths[...] = kept
        self.tok.upload(tok)
        self.pos.upload(pos)
        self._launch()
        _lib.call("mira_cuda_sync")
        logits = self.logits.download((self.batch, self.vocab), np.float32)
        return {s: logits[s] for s in tokens}

    def generate(self, prompt, new_tokens: int, slot: Optional[int] = None) -> tuple[int, list]:
        """Feeds a prompt to a new sequence (or to `slot`) and appends `new_tokens` greedy ones; returns
        (slot, the new tokens).  If it raises, a sequence that it opened is closed again; one that was
        there keeps the tokens that it was fed."""
        if not len(prompt):
            raise ValueError("an empty prompt")
        opened = slot is None
        slot = self.cache.open() if opened else slot
        out, logits = [], None
        try:
            for t in prompt:
                logits = self.step({slot: int(t)})[slot]
            for i in range(new_tokens):
                out.append(int(np.argmax(logits)))
                if i + 1 < new_tokens:
                    logits = self.step({slot: out[-1]})[slot]
        except Exception:
            if opened:      # the caller does not know the slot
                self.cache.close(slot)
            raise
        return slot, out

    def close(self) -> None:
        if self._graph is not None:
            _lib.call("mira_cuda_sync")
            _lib.call("mira_cuda_graph_destroy", self._graph)
            self._graph = None
        self.cache.free()

"""The serving operators of a decoder that keeps its keys and values in pages: measured cases.

One pass of a case is one call of one operator:

  attention   one new token per sequence attends to the sequence's pages
              o[b, h] = sum_t p_t v_t,  p = softmax(scale * q[b, h] . k_t) over the visible t < length[b]
              (with a window: the last `window` positions and the first `sinks` ones), and
              lse[b, h] = log sum_t exp(scale * q[b, h] . k_t)
  append      new keys and values go to their sequences' last positions, converted to the pages' type
  copy        pages are duplicated inside a pool, all layers at once (fork, compaction)
  matvec      y = act(x @ (s * (w - 8))^T + bias) with 4-bit w and one scale s per group of k

`own` chooses between the plain form (elementary torch operations in 32 bits) and mira_b200's kernels.
"""
import math
import random

import torch

own = False

TORCH = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "i8": torch.int8}
SIZE = {"f32": 4, "f16": 2, "bf16": 2, "i8": 1}


# ------------------------------------------------------------------------------------------ the cases

def attention(name, q, kv, batch, heads, kv_heads, dh, page, longest, spread="ragged", window=0, sinks=0, order="head"):
    return dict(name=name, op="attention", q=q, kv=kv, batch=batch, heads=heads, kv_heads=kv_heads, dh=dh, page=page,
                longest=longest, spread=spread, window=window, sinks=sinks, order=order)


def append(name, src, kv, batch, kv_heads, dh, page, longest, new):
    return dict(name=name, op="append", src=src, kv=kv, batch=batch, kv_heads=kv_heads, dh=dh, page=page,
                longest=longest, new=new)


def copy(name, kv, layers, pages, kv_heads, dh, page, moved):
    return dict(name=name, op="copy", kv=kv, layers=layers, pages=pages, kv_heads=kv_heads, dh=dh, page=page,
                moved=moved)


def matvec(name, x, scales, m, n, k, group, act):
    return dict(name=name, op="matvec", x=x, scales=scales, m=m, n=n, k=k, group=group, act=act)


def listed():
    return [
        # the first tokens of one conversation: latency is all there is
        attention("attention 1x12 first tokens", "f32", "f32", 1, 12, 12, 64, 16, 23),
        # this repository's decode workload (64 sequences, 12 heads of 64, up to 1024 positions) on pages
        attention("attention 64x12x1024 f32", "f32", "f32", 64, 12, 12, 64, 16, 1024),
        # a serving batch of ragged requests, grouped heads, 16-bit pages
        attention("attention 32x32/8 bf16", "bf16", "bf16", 32, 32, 8, 128, 32, 8192),
        # one long document: a single sequence has to fill the whole card
        attention("attention 1x32/4 131071 f16", "f16", "f16", 1, 32, 4, 128, 64, 131071),
        # 8-bit pages under a sliding window with four sinks, head size and page size not powers of two
        attention("attention 48x20/4 i8 window", "f32", "i8", 48, 20, 4, 80, 24, 20000, window=4095, sinks=4),
        # one decode step's new rows: a row per sequence
        append("append 64 rows f32", "f32", "f32", 64, 12, 64, 16, 1024, 1),
        # prompts of very different lengths enter 16-bit pages together
        append("append ragged prompts bf16", "f32", "bf16", 24, 8, 128, 32, 8192, 4096),
        # forks of a few sequences: their partly filled last pages, in every layer
        copy("copy 5 pages x 12 layers", "f32", 12, 64, 12, 64, 16, 5),
        # compaction of a pool: hundreds of pages change places
        copy("copy 700 pages x 16 layers", "bf16", 16, 2048, 8, 64, 16, 700),
        # a projection of this repository's transformer for one token
        matvec("matvec 1x768x768", "f32", "f32", 1, 768, 768, 32, "none"),
        # a small batch through a middle-sized projection with an activation
        matvec("matvec 16x4096x4096 bf16", "bf16", "bf16", 16, 4096, 4096, 128, "gelu"),
        # one token through a matrix that is larger than the second-level cache
        matvec("matvec 1x32768x8192 f16", "f16", "f16", 1, 32768, 8192, 64, "none"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "append", "copy", "matvec", "matvec"])
    dh = rng.choice([32, 40, 64, 64, 72, 80, 96, 112, 128, 128, 160, 192, 256])
    page = rng.choice([5, 8, 16, 16, 24, 32, 64, 100, 128])
    if op == "attention":
        kv = rng.choice(["f32", "f16", "bf16", "i8"])
        q = rng.choice({"f32": ["f32"], "f16": ["f16", "f32"], "bf16": ["bf16", "f32"], "i8": ["f32", "f16", "bf16"]}[kv])
        kv_heads, group = rng.choice([1, 2, 3, 4, 8, 12, 16]), rng.choice([1, 1, 2, 3, 4, 5, 6, 7, 8, 12, 16])
        batch, longest = _log(rng, 1, 128), _log(rng, 1, 131072)
        most = (1 << 28) // 2 // (kv_heads * dh * batch)     # half the largest listed case's padded elements
        longest = max(1, min(longest, most))
        window = 0 if rng.random() < 0.6 else _log(rng, 1, longest)
        return {k: v for k, v in attention("", q, kv, batch, kv_heads * group, kv_heads, dh, page, longest,
                                           rng.choice(["ragged", "same"]), window, rng.choice([0, 1, 4, 17]) if window else 0,
                                           rng.choice(["head", "token"])).items() if k != "name"}
    if op == "append":
        src, kv = rng.choice([("f32", "f32"), ("f32", "bf16"), ("f32", "f16"), ("bf16", "bf16"), ("f16", "f16")])
        kv_heads, batch, new = rng.choice([1, 2, 4, 8, 12]), _log(rng, 1, 64), _log(rng, 1, 2048)
        longest = max(new, _log(rng, 1, 4096))
        return {k: v for k, v in append("", src, kv, batch, kv_heads, dh, page, longest, new).items() if k != "name"}
    if op == "copy":
        kv, layers, kv_heads = rng.choice(["f32", "f16", "bf16"]), _log(rng, 1, 24), rng.choice([1, 2, 4, 8, 12])
        each = 2 * layers * kv_heads * dh * page
        pages = max(2, min(_log(rng, 2, 2048), (1 << 27) // each))
        return {k: v for k, v in copy("", kv, layers, pages, kv_heads, dh, page, _log(rng, 1, pages // 2)).items() if k != "name"}
    x = rng.choice(["f32", "f16", "bf16"])
    return {k: v for k, v in matvec("", x, rng.choice(["f32", x]), _log(rng, 1, 16), _log(rng, 64, 14000), _log(rng, 64, 14000),
                                    rng.choice([32, 64, 128, 256]), rng.choice(["none", "gelu", "relu"])).items() if k != "name"}


# --------------------------------------------------------------------------------------- lengths, work

def lengths_of(case):
    """Tokens in each sequence: spread over the whole range, the longest and an empty slot among them."""
    b, longest = case["batch"], case["longest"]
    if b == 1 or case.get("spread") == "same":
        return [longest] * b
    got = [max(1, round(longest * (i + 1) / b)) for i in range(b)]
    if b >= 8:
        got[0] = 0          # a slot of the batch that no request holds
    random.Random(b * 1000003 + longest).shuffle(got)
    return got


def news_of(case):
    """New rows of each sequence: one each in a decode step, else spread up to `new` within its length."""
    b, new = case["batch"], case["new"]
    lens = [max(1, n) for n in lengths_of(case)]
    return lens, [1 if new == 1 else min(n, max(1, round(new * (i + 1) / b))) for i, n in enumerate(lens)]


def visible(case, n):
    """(first windowed position, sinks before it) of a sequence of n tokens."""
    start = max(0, n - case["window"]) if case["window"] else 0
    return start, min(case["sinks"], start)


def work(case):
    if case["op"] == "attention":
        lens = lengths_of(case)
        seen = sum(n - visible(case, n)[0] + visible(case, n)[1] for n in lens)
        row = case["dh"] * SIZE[case["kv"]] + (4 if case["kv"] == "i8" else 0)
        rows = case["batch"] * case["heads"]
        return {"bytes": 2 * seen * case["kv_heads"] * row + rows * (2 * case["dh"] * SIZE[case["q"]] + 4)
                + 4 * (case["batch"] + seen // case["page"]),
                "flops": 4 * seen * case["heads"] * case["dh"]}
    if case["op"] == "append":
        rows = sum(news_of(case)[1])
        return {"bytes": 2 * rows * case["kv_heads"] * case["dh"] * (SIZE[case["src"]] + SIZE[case["kv"]]), "flops": 0}
    if case["op"] == "copy":
        return {"bytes": 2 * case["moved"] * 2 * case["layers"] * case["page"] * case["kv_heads"] * case["dh"] * SIZE[case["kv"]],
                "flops": 0}
    m, n, k = case["m"], case["n"], case["k"]
    return {"bytes": n * (-(-k // 2) + -(-k // case["group"]) * SIZE[case["scales"]]) + m * (n + k) * SIZE[case["x"]] + 4 * n,
            "flops": 2 * m * n * k}


# ------------------------------------------------------------------------------------------ the inputs

class State(dict):
    __getattr__ = dict.__getitem__


def _pages(case, gen, lens):
    """A pool with every sequence's pages scattered over it, and the page table (int32)."""
    need = [-(-n // case["page"]) for n in lens]
    width = max(1, max(need))
    num = sum(need) + 3
    order = torch.randperm(num, generator=gen, device="cuda")[: sum(need)].to(torch.int32)
    table = torch.full((case["batch"], width), -1, dtype=torch.int32, device="cuda")
    held = torch.arange(width, device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
    table[held] = order
    return num, table


def _pool(case, num):
    """Shape of the pages, and the place of (page, kv head, slot, element) in it."""
    head = case.get("order", "head") == "head"
    shape = (num, case["kv_heads"], case["page"], case["dh"]) if head else (num, case["page"], case["kv_heads"], case["dh"])
    return shape, head


def _random(shape, gen, dtype, by=1.0):
    if dtype is torch.int8:
        return torch.randint(-127, 128, shape, generator=gen, device="cuda", dtype=torch.int8)
    return (torch.randn(shape, generator=gen, device="cuda") * by).to(dtype)


def _strides(t, head):
    """(page, kv head, slot, element) strides of pages in either order."""
    s = t.stride()
    return (s[0], s[1], s[2], s[3]) if head else (s[0], s[2], s[1], s[3])


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)
    s = State(case=case)
    if case["op"] == "attention":
        lens = lengths_of(case)
        num, s["table"] = _pages(case, gen, lens)
        shape, s["head"] = _pool(case, num)
        kv = TORCH[case["kv"]]
        s["k"], s["v"] = _random(shape, gen, kv), _random(shape, gen, kv)
        if case["kv"] == "i8":       # a row of N(0, 1) values spans about 2.7 either way
            s["ks"] = (torch.rand(shape[:3], generator=gen, device="cuda") + 2.2) / 127
            s["vs"] = (torch.rand(shape[:3], generator=gen, device="cuda") + 2.2) / 127
        # scores of a few units: some tokens matter more than others
        s["q"] = _random((case["batch"], case["heads"], case["dh"]), gen, TORCH[case["q"]], 1.7)
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["scale"] = case["dh"] ** -0.5
    elif case["op"] == "append":
        lens, news = news_of(case)
        num, s["table"] = _pages(case, gen, lens)
        shape, s["head"] = _pool(case, num)
        s["k"], s["v"] = (torch.zeros(shape, dtype=TORCH[case["kv"]], device="cuda") for _ in "kv")
        rows = sum(news)
        s["k_new"], s["v_new"] = (_random((rows, case["kv_heads"], case["dh"]), gen, TORCH[case["src"]]) for _ in "kv")
        s["lengths"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
        s["starts"] = torch.tensor([sum(news[:i]) for i in range(len(news) + 1)], dtype=torch.int32, device="cuda")
    elif case["op"] == "copy":
        shape = (2 * case["layers"], case["pages"], case["kv_heads"], case["page"], case["dh"])
        s["pool"] = _random(shape, gen, TORCH[case["kv"]])
        order = torch.randperm(case["pages"], generator=gen, device="cuda")[: 2 * case["moved"]].to(torch.int32).cpu().numpy()
        s["src"], s["dst"] = order[: case["moved"]].copy(), order[case["moved"]:].copy()
    else:
        m, n, k, group = case["m"], case["n"], case["k"], case["group"]
        ld, groups = -(-(-(-k // 2)) // 16) * 16, -(-k // group)
        s["x"] = _random((m, k), gen, TORCH[case["x"]])
        # normal weights rounded to 15 levels: the nibbles hold q + 8
        q = (torch.randn((n, 2 * ld), generator=gen, device="cuda", dtype=torch.float16) * 2.6).round_().clamp_(-7, 7).to(torch.int8).add_(8).view(torch.uint8)
        s["w"] = q[:, 0::2] | (q[:, 1::2] << 4)
        s["scales"] = ((torch.rand((n, groups), generator=gen, device="cuda") + 0.5) * (0.4 / math.sqrt(k))).to(TORCH[case["scales"]])
        s["bias"] = torch.randn(n, generator=gen, device="cuda") * 0.1
    if own:
        _handles(s)
    return s


def _handles(s):
    """What a program that serves with mira_b200 keeps between calls: outputs, scratch and descriptors."""
    from mira_b200 import kernels as K
    from mira_b200.device import set_device
    set_device(torch.cuda.current_device())
    c = s.case

    def pages():
        st = _strides(s.k, s.head)
        more = {}
        if c["kv"] == "i8":
            ss = s.ks.stride()
            ss = (ss[0], ss[1], ss[2], 1) if s.head else (ss[0], ss[2], ss[1], 1)
            more = dict(k_scale=K.View(s.ks.data_ptr(), ss), v_scale=K.View(s.vs.data_ptr(), ss))
        return K.PagedKV(num_pages=s.k.shape[0], page_size=c["page"], kv_heads=c["kv_heads"], dh=c["dh"], dtype=c["kv"],
                         k=K.View(s.k.data_ptr(), st), v=K.View(s.v.data_ptr(), st), batch=c["batch"], table=s.table.data_ptr(),
                         table_ld=s.table.shape[1], max_pages=s.table.shape[1], lengths=s.lengths.data_ptr(), **more)

    if c["op"] == "attention":
        s["out"] = torch.empty_like(s.q)
        s["lse"] = torch.empty((c["batch"], c["heads"]), device="cuda")
        size = K.paged_attention_workspace(c["batch"], c["heads"], c["kv_heads"], c["dh"])
        s["workspace"] = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
        row = (c["heads"] * c["dh"], c["dh"], 0, 1)
        s["plan"] = K.PagedAttn(kv=pages(), heads=c["heads"], q=K.View(s.q.data_ptr(), row), q_dtype=c["q"], scale=s.scale,
                                window=c["window"], sinks=c["sinks"], out=K.View(s.out.data_ptr(), row), lse=s.lse.data_ptr(),
                                workspace=s.workspace.data_ptr(), workspace_bytes=size).struct()
    elif c["op"] == "append":
        row = (0, c["dh"], c["kv_heads"] * c["dh"], 1)
        s["plan"] = K.KvAppend(kv=pages(), rows=s.k_new.shape[0], src_dtype=c["src"], k_new=K.View(s.k_new.data_ptr(), row),
                               v_new=K.View(s.v_new.data_ptr(), row), row_start=s.starts.data_ptr()).struct()
    elif c["op"] == "copy":
        size = s.pool.element_size()
        s["plan"] = K.page_regions([K.PageRegion(s.pool.data_ptr(), planes=s.pool.shape[0], plane_stride=s.pool.stride(0) * size,
                                                 page_stride=s.pool.stride(1) * size, page_bytes=s.pool.stride(1) * size)])
    else:
        s["out"] = torch.empty((c["m"], c["n"]), dtype=s.x.dtype, device="cuda")
        size = K.w4_matvec_workspace(c["m"], c["n"], c["k"])
        s["workspace"] = torch.zeros(max(size, 16), dtype=torch.uint8, device="cuda")
        steps = [K.Step("add", "channel", ptr=s.bias.data_ptr())] + ([K.Step(c["act"])] if c["act"] != "none" else [])
        s["plan"] = K.W4Matvec(m=c["m"], n=c["n"], k=c["k"], group=c["group"], x=s.x.data_ptr(), ld_x=c["k"], x_dtype=c["x"],
                               w=s.w.data_ptr(), ld_w=s.w.shape[1], scales=s.scales.data_ptr(), ld_scales=s.scales.shape[1],
                               scale_dtype=c["scales"], steps=steps, out=s.out.data_ptr(), ld_out=c["n"], out_dtype=c["x"],
                               workspace=s.workspace.data_ptr(), workspace_bytes=size).struct()
    torch.cuda.synchronize()     # the library launches on a stream of its own: the inputs have to be there


# -------------------------------------------------------------------------------------------- a pass

def run(s):
    return (_run_own if own else _run_plain)(s)


def _run_own(s):
    from mira_b200 import kernels as K
    op = s.case["op"]
    if op == "attention":
        K.paged_attention(s.plan)
        return {"out": s.out, "lse": s.lse}
    if op == "append":
        K.kv_append(s.plan)
        return {"k": s.k, "v": s.v}
    if op == "copy":
        K.page_copy(s.plan, s.case["pages"], s.src, s.dst)
        return s.pool
    K.w4_matvec(s.plan)
    return s.out


def _run_plain(s):
    return {"attention": _plain_attention, "append": _plain_append, "copy": _plain_copy, "matvec": _plain_matvec}[s.case["op"]](s)


def _plain_attention(s):
    c = s.case
    b, hkv, g, dh = c["batch"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dh"]

    def gather(pages, scales):
        x = pages[s.table.clamp(min=0).long()].float()                 # [batch, pages, head, slot, dh] or [.., slot, head, dh]
        if scales is not None:
            x = x * scales[s.table.clamp(min=0).long()][..., None]
        x = x if s.head else x.transpose(2, 3)
        return x.transpose(1, 2).reshape(b, hkv, -1, dh)               # [batch, head, position, dh]

    k, v = gather(s.k, s.get("ks")), gather(s.v, s.get("vs"))
    at = torch.arange(k.shape[2], device="cuda")[None, :]
    n = s.lengths[:, None]
    see = at < n
    if c["window"]:
        see = see & ((at >= n - c["window"]) | (at < c["sinks"]))
    scores = torch.matmul(s.q.float().view(b, hkv, g, dh), k.transpose(2, 3)) * s.scale
    scores = scores.masked_fill(~see[:, None, None, :], float("-inf"))
    top = scores.amax(-1, keepdim=True)
    top = top.masked_fill(top == float("-inf"), 0.0)                    # a sequence without tokens
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = torch.matmul(p, v) / torch.where(total == 0, 1.0, total)
    return {"out": out.view(b, hkv * g, dh).to(s.q.dtype), "lse": (top + torch.log(total)).view(b, hkv * g)}


def _plain_append(s):
    c = s.case
    row = torch.arange(s.k_new.shape[0], device="cuda")
    seq = torch.searchsorted(s.starts[1:].long(), row, right=True)
    pos = s.lengths.long()[seq] - (s.starts.long()[seq + 1] - row)
    page, slot = s.table[seq, pos // c["page"]].long(), pos % c["page"]
    for pages, new in ((s.k, s.k_new), (s.v, s.v_new)):
        pages.transpose(1, 2)[page, slot] = new.float().to(pages.dtype)   # [page, slot, head, dh]
    return {"k": s.k, "v": s.v}


def _plain_copy(s):
    src, dst = torch.from_numpy(s.src).cuda().long(), torch.from_numpy(s.dst).cuda().long()
    s.pool[:, dst] = s.pool[:, src]
    return s.pool


def _plain_matvec(s):
    c = s.case
    w = torch.stack((s.w & 15, s.w >> 4), -1).view(c["n"], -1)[:, : c["k"]].float() - 8.0
    w = w * s.scales.float().repeat_interleave(c["group"], 1)[:, : c["k"]]
    y = torch.matmul(s.x.float(), w.t()) + s.bias
    if c["act"] == "gelu":
        y = 0.5 * y * (1.0 + torch.tanh(0.7978845608028654 * (y + 0.044715 * y * y * y)))
    elif c["act"] == "relu":
        y = torch.where(y > 0, y, 0.0)
    return y.to(s.x.dtype)


# ------------------------------------------------------------------------------------ the definition

def exact(case, seed):
    """The same from the definitions in 64 bits, one sequence, one row or one page at a time."""
    global own
    kept, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = kept
    d = torch.float64
    if case["op"] == "attention":
        out = torch.zeros((case["batch"], case["heads"], case["dh"]), dtype=d, device="cuda")
        lse = torch.full((case["batch"], case["heads"]), float("-inf"), dtype=d, device="cuda")
        for b, n in enumerate(lengths_of(case)):
            start, sinks = visible(case, n)
            pos = torch.tensor(list(range(sinks)) + list(range(start, n)), dtype=torch.long, device="cuda")
            if not len(pos):
                continue
            page, slot = s.table[b].long()[pos // case["page"]], pos % case["page"]
            rows = []
            for x, sc in ((s.k, s.get("ks")), (s.v, s.get("vs"))):
                t = (x[page, :, slot] if s.head else x[page, slot]).to(d)      # [tokens, kv heads, dh]
                if sc is not None:
                    t = t * (sc[page, :, slot] if s.head else sc[page, slot]).to(d)[..., None]
                rows.append(t.repeat_interleave(case["heads"] // case["kv_heads"], 1))
            z = torch.einsum("hd,thd->ht", s.q[b].to(d), rows[0]) / math.sqrt(case["dh"])
            lse[b] = torch.logsumexp(z, 1)
            out[b] = torch.einsum("ht,thd->hd", torch.exp(z - lse[b][:, None]), rows[1])
        return {"out": out, "lse": lse}
    if case["op"] == "append":
        lens, news = news_of(case)
        k, v = torch.zeros_like(s.k, dtype=d), torch.zeros_like(s.v, dtype=d)
        at = 0
        for b, (n, r) in enumerate(zip(lens, news)):
            pos = torch.arange(n - r, n, device="cuda")
            page, slot = s.table[b].long()[pos // case["page"]], pos % case["page"]
            k[page, :, slot] = s.k_new[at: at + r].to(d)
            v[page, :, slot] = s.v_new[at: at + r].to(d)
            at += r
        return {"k": k, "v": v}
    if case["op"] == "copy":
        pool = s.pool.to(d)
        for a, b in zip(s.src.tolist(), s.dst.tolist()):
            pool[:, b] = pool[:, a]
        return pool
    low, high = (s.w % 16).to(d), torch.div(s.w, 16, rounding_mode="floor").to(d)
    y = s.bias.to(d).repeat(case["m"], 1)
    x = s.x.to(d)
    for g in range(s.scales.shape[1]):
        lo, hi = g * case["group"], min(case["k"], (g + 1) * case["group"])
        even, odd = x[:, lo:hi:2], x[:, lo + 1:hi:2]
        part = even @ (low[:, lo // 2: lo // 2 + even.shape[1]] - 8).t() + odd @ (high[:, lo // 2: lo // 2 + odd.shape[1]] - 8).t()
        y += part * s.scales[:, g].to(d)
    if case["act"] == "gelu":
        y = 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    elif case["act"] == "relu":
        y = y.clamp(min=0)
    return y

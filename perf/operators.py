"""The serving operators around the 8-bit paged cache, as cases that can be timed and compared.

Four operators of one decode step of the rollout engine: rows of keys and values quantised into the paged cache (``append``),
attention of single tokens over it (``decode``), pages copied when requests fork from a shared prompt (``copy``) and the next
token drawn under temperature, top-k, top-p and min-p from given random numbers (``sample``). Each has a plain form in
elementary torch operations and a statement in 64 bits; with ``own`` set, ``run`` makes the calls that the engine makes.
"""
import math
import random

import numpy as np
import torch

own = False

F8 = torch.float8_e4m3fn
F8_MAX = 448.0
E_MIN, E_MAX = -100, 120             # exponents a scale may have

# (query heads, key/value heads, head size) of the models that the framework configures
HEADS = [(32, 8, 128), (28, 4, 128), (12, 2, 128), (32, 4, 128), (4, 2, 64), (8, 8, 64), (16, 1, 128)]


def listed():
    return [
        # one decode step of 64 requests: a token each, some pages new, some rows of the batch without a request
        dict(name="append-decode-64", op="append", rows=64, tokens=1, kv_heads=8, dim=128, page=64),
        # the largest decode batch, pages of 16 tokens, heads of 64
        dict(name="append-decode-256", op="append", rows=256, tokens=1, kv_heads=2, dim=64, page=16),
        # a prefill of packed prompts of all lengths, the engine's budget of 16384 tokens
        dict(name="append-prefill-16k", op="append", rows=23, tokens=712, kv_heads=8, dim=128, page=64),
        # one request early in its answer: latency
        dict(name="decode-1x200", op="decode", rows=1, ctx=200, q_heads=32, kv_heads=8, dim=128, page=64),
        # the batch of the benchmark's rollout, contexts around a thousand tokens
        dict(name="decode-64x1k", op="decode", rows=64, ctx=1500, q_heads=32, kv_heads=8, dim=128, page=64),
        # the largest batch, ragged contexts up to 4k, seven query heads for each key head
        dict(name="decode-256x4k", op="decode", rows=256, ctx=4001, q_heads=28, kv_heads=4, dim=128, page=64),
        # few long requests: the split over the context
        dict(name="decode-3x32k", op="decode", rows=3, ctx=32767, q_heads=32, kv_heads=4, dim=128, page=64),
        # a group of 16 samples: fifteen requests take the partial last page of the prompt, all layers
        dict(name="copy-fork-15", op="copy", pairs=15, layers=36, kv_heads=8, dim=128, page=64, bits=8, fork=True),
        # pages moved in bulk, cache in 16 bits
        dict(name="copy-bulk-90", op="copy", pairs=90, layers=28, kv_heads=4, dim=128, page=64, bits=16, fork=False),
        # 64 requests with nucleus sampling
        dict(name="sample-64-nucleus", op="sample", rows=64, vocab=151936, mode="nucleus"),
        # the largest batch, every request with filters of its own
        dict(name="sample-256-mixed", op="sample", rows=256, vocab=151936, mode="mixed"),
        # a single request, top-k
        dict(name="sample-1-topk", op="sample", rows=1, vocab=151936, mode="topk"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "copy", "sample"])
    hq, hkv, dim = rng.choice(HEADS)
    page = rng.choice([16, 32, 64, 128])
    if op == "append":
        if rng.random() < 0.5:
            return dict(op=op, rows=_log(rng, 1, 256), tokens=1, kv_heads=hkv, dim=dim, page=page)
        rows = _log(rng, 1, 64)
        return dict(op=op, rows=rows, tokens=_log(rng, 2, max(3, 16384 // rows)), kv_heads=hkv, dim=dim, page=page)
    if op == "decode":
        rows = _log(rng, 1, 256)
        return dict(op=op, rows=rows, ctx=_log(rng, 1, min(32768, 500_000_000 // (rows * hkv * dim))), q_heads=hq, kv_heads=hkv, dim=dim, page=page)
    if op == "copy":
        return dict(op=op, pairs=_log(rng, 1, 60), layers=rng.choice([2, 4, 28]), kv_heads=min(hkv, 4), dim=dim, page=min(page, 64), bits=rng.choice([8, 16]),
                    fork=rng.random() < 0.5)
    return dict(op=op, rows=_log(rng, 1, 256), vocab=_log(rng, 1000, 151936), mode=rng.choice(["nucleus", "topk", "minp", "mixed"]))


def _lens(case):
    """Contexts (decode) or tokens of each row (append): they belong to the case, whatever the seed."""
    r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")))
    top = case["ctx"] if case["op"] == "decode" else case["tokens"]
    if case["op"] == "append" and top == 1:
        return [0 if r.random() < 0.1 and case["rows"] > 1 else 1 for _ in range(case["rows"])]
    lens = [r.randint(max(1, top // 2), top) for _ in range(case["rows"])]
    lens[r.randrange(len(lens))] = top
    if case["op"] == "decode" and len(lens) > 4:
        lens[r.randrange(len(lens))] = 0            # a row of the batch without a request
    return lens


def work(case):
    if case["op"] == "append":
        n = sum(_lens(case))
        return dict(bytes=n * case["kv_heads"] * case["dim"] * 2 * 3 + n * case["kv_heads"] * 4, flops=0)
    if case["op"] == "decode":
        n = sum(_lens(case))
        pages = sum(-(-x // case["page"]) for x in _lens(case))
        return dict(bytes=2 * n * case["kv_heads"] * case["dim"] + 8 * pages * case["kv_heads"] + 4 * case["rows"] * case["q_heads"] * case["dim"],
                    flops=4 * n * case["q_heads"] * case["dim"])
    if case["op"] == "copy":
        one = 2 * case["layers"] * case["kv_heads"] * (case["dim"] * _tail(case) * case["bits"] // 8 + (4 if case["bits"] == 8 else 0))
        return dict(bytes=one * (case["pairs"] + 1 if case["fork"] else 2 * case["pairs"]), flops=0)
    return dict(bytes=4 * case["rows"] * case["vocab"] + 8 * case["rows"], flops=case["rows"] * case["vocab"])


def _tail(case):
    return max(1, case["page"] * 5 // 8) if case["fork"] else case["page"]


# ------------------------------------------------------------------ inputs
def _keys(g, *shape):
    """Rows like keys and values: normal, with channels of their own size."""
    size = torch.exp(0.7 * torch.randn(shape[-1], device="cuda", generator=g))
    return (torch.randn(*shape, device="cuda", generator=g) * size).bfloat16()


def _cache(g, pages, kv_heads, page, dim):
    """Codes and scales of a cache in use."""
    out = []
    for _ in range(2):
        codes = torch.empty(pages, kv_heads, page, dim, device="cuda", dtype=F8)
        scale = torch.empty(pages, kv_heads, device="cuda")
        step = max(1, (1 << 27) // (kv_heads * page * dim))
        for i in range(0, pages, step):
            x = _keys(g, min(step, pages - i), kv_heads, page, dim).float()
            s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / F8_MAX)))
            codes[i:i + step] = (x / s[:, :, None, None]).clamp(-F8_MAX, F8_MAX).to(F8)
            scale[i:i + step] = s
        out += [codes, scale]
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    if case["op"] == "append":
        n, ps = _lens(case), case["page"]
        r = random.Random(repr(sorted((k, v) for k, v in case.items() if k != "name")) + "start")
        start = [r.randint(0, 3 * ps) for _ in n] if case["tokens"] == 1 else [r.choice([0, 0, r.randint(0, 2 * ps)]) for _ in n]
        lens = [s + t if t else 0 for s, t in zip(start, n)]
        width = max(1, max(-(-x // ps) for x in lens)) + 1
        pages = len(n) * width + 3
        # packed rows: a prefill gives cu_seqlens; in a decode step every row of the batch is there, requests or not
        total = sum(n) if case["tokens"] > 1 else len(n)
        kv = _keys(g, total, 2, case["kv_heads"], case["dim"]) * 3
        kc, ks, vc, vs = _cache(g, pages, case["kv_heads"], ps, case["dim"])
        st = dict(case=case, k=kv[:, 0], v=kv[:, 1], pages=[kc, vc, ks, vs], lens=torch.tensor(lens, dtype=torch.int32, device="cuda"),
                  table=torch.randperm(pages, device="cuda", generator=g)[:len(n) * width].int().view(len(n), width).contiguous(), cu=None)
        if case["tokens"] > 1:
            st["cu"] = torch.tensor([0] + list(np.cumsum(n)), dtype=torch.int32, device="cuda")
        return st
    if case["op"] == "decode":
        lens, ps = _lens(case), case["page"]
        width = case["ctx"] // ps + 1
        used = [-(-x // ps) for x in lens]
        pages = sum(used) + 3
        order = torch.randperm(pages, device="cuda", generator=g).int().cpu()
        table = torch.zeros(len(lens), width, dtype=torch.int32)
        at = 0
        for b, u in enumerate(used):
            table[b, :u] = order[at:at + u]
            at += u
        kc, ks, vc, vs = _cache(g, pages, case["kv_heads"], ps, case["dim"])
        return dict(case=case, q=torch.randn(len(lens), case["q_heads"], case["dim"], device="cuda", generator=g).bfloat16(), pages=[kc, vc, ks, vs],
                    table=table.cuda(), lens=torch.tensor(lens, dtype=torch.int32, device="cuda"), scale=case["dim"] ** -0.5)
    if case["op"] == "copy":
        n, ps, L = case["pairs"], case["page"], case["layers"]
        pages = 2 * n + 5
        shape = (L, 2, pages, case["kv_heads"], ps, case["dim"]) if case["bits"] == 8 else (L, 2, pages, ps, case["kv_heads"], case["dim"])
        data = torch.empty(*shape, device="cuda", dtype=F8 if case["bits"] == 8 else torch.bfloat16)
        for i in range(L):
            data[i] = torch.randn(*shape[1:], device="cuda", generator=g).to(data.dtype)
        order = np.random.RandomState(seed % (1 << 31)).permutation(pages).astype(np.int32)
        src = np.full(n, order[-1], np.int32) if case["fork"] else order[n:2 * n].copy()
        st = dict(case=case, data=data, src=src, dst=order[:n].copy(), tokens=np.full(n, _tail(case), np.int32) if case["fork"] else None)
        if case["bits"] == 8:
            st["scales"] = torch.exp2(torch.randint(-8, 3, (L, 2, pages, case["kv_heads"]), device="cuda", generator=g).float())
        return st
    B, V = case["rows"], case["vocab"]
    # logits of a language model: a wide bulk and, in most rows, a few tokens far above it
    x = torch.randn(B, V, device="cuda", generator=g) * 2.3
    near = torch.randint(0, V, (B, 40), device="cuda", generator=g)
    lift = torch.rand(B, 1, device="cuda", generator=g) * 20 * torch.rand(B, 40, device="cuda", generator=g)
    x.scatter_add_(1, near, lift)
    x = x.bfloat16().float()                         # the LM head's products are rounded to 16 bits: equal logits are common
    r = np.random.RandomState(seed % (1 << 31))
    t = r.choice([0.6, 0.7, 0.8, 1.0, 1.0, 1.2], B)
    k, p, m, greedy = np.zeros(B), np.ones(B), np.zeros(B), np.zeros(B)
    if case["mode"] in ("topk", "mixed"):
        k = r.choice([20, 40, 50, 1000] if case["mode"] == "topk" else [0, 0, 20, 50, 10 ** 8], B)
    if case["mode"] in ("nucleus", "mixed"):
        p = r.choice([0.9, 0.95, 0.95, 0.99, 0.8] if case["mode"] == "nucleus" else [1.0, 0.95, 0.9], B)
    if case["mode"] in ("minp", "mixed"):
        m = r.choice([0.02, 0.05, 0.1] if case["mode"] == "minp" else [0.0, 0.0, 0.05], B)
    if case["mode"] == "mixed":
        greedy = r.rand(B) < 0.1
    f32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.float32, device="cuda")     # noqa: E731
    i32 = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")       # noqa: E731
    return dict(case=case, logits=x, u=torch.rand(B, device="cuda", generator=g), inv_temp=f32(1.0 / t), top_k=i32(k), top_p=f32(p), min_p=f32(m), greedy=i32(greedy))


# ------------------------------------------------------------------ plain forms
def _pow2(e):
    return ((e + 127) << 23).int().view(torch.float32)


def _bytes(t):
    return t.view(torch.uint8) if t.dtype == F8 else t


def _plain_rows(x, codes, scale, page, off, live, touched):
    """Rows ``x`` [n, Hkv, D] to slot ``off`` of ``page`` where ``live``; ``touched``: the pages that get rows, some of them more than once."""
    a = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(-1)
    m, e = torch.frexp(a)
    e = torch.where(m <= F8_MAX / 512, e - 9, e - 8)                            # the smallest e with a <= 448 * 2^e
    want = torch.where(live[:, None], _pow2(torch.where(a > 0, e, E_MIN).clamp(E_MIN, E_MAX)), 0.0)
    new = torch.zeros(scale.shape[0], device=x.device, dtype=torch.int32).scatter_reduce_(0, page, ((off == 0) & live).int(), "amax")
    base = torch.where(new[:, None] > 0, 0.0, scale)                            # a page whose slot 0 is written holds nothing else
    scale.copy_(base.scatter_reduce(0, page[:, None].expand_as(want), want, "amax"))
    ratio = torch.where((base > 0) & (scale > base), base / scale, 1.0)
    raw = codes.view(torch.uint8)
    raw[touched] = (raw[touched].view(F8).float() * ratio[touched][:, :, None, None]).to(F8).view(torch.uint8)
    q = (x / scale[page][:, :, None]).clamp(-F8_MAX, F8_MAX).to(F8).view(torch.uint8)
    row = torch.where(live, torch.arange(live.numel(), device=x.device), torch.where(live, 0, 1).argmin())   # no token here: the first live one again
    raw[page[row], :, off[row]] = q[row]


def _plain_append(st):
    lens, cu, table, ps = st["lens"].long(), st["cu"], st["table"].long(), st["case"]["page"]
    t = torch.arange(st["k"].shape[0], device=lens.device)
    if cu is None:
        row, n, first = t, (lens > 0).long(), t
    else:
        row = torch.searchsorted(cu[1:].contiguous(), t.int(), right=True)
        n, first = (cu[1:] - cu[:-1]).long(), cu.long()[row]
    start = lens - n
    pos = (start[row] + t - first).clamp(min=0)
    live = n[row] > 0
    page, off = table[row, pos // ps], pos % ps
    one = page[torch.where(live, 0, 1).argmin()]
    page = torch.where(live, page, one)
    j = torch.arange(table.shape[1], device=lens.device)
    touched = torch.where((n[:, None] > 0) & (j >= start[:, None] // ps) & (j <= (lens[:, None] - 1) // ps), table, one).flatten()
    kc, vc, ks, vs = st["pages"]
    _plain_rows(st["k"].float(), kc, ks, page, off, live, touched)
    _plain_rows(st["v"].float(), vc, vs, page, off, live, touched)
    return [kc, vc, ks, vs]


def _plain_decode(st):
    (kc, vc, ks, vs), table, lens, q = st["pages"], st["table"].long(), st["lens"], st["q"]
    B, Hq, D = q.shape
    Hkv, ps = kc.shape[1:3]
    t = torch.arange(table.shape[1] * ps, device=q.device)

    def rows(codes, scale):                                                     # [B, Hkv, tokens, D]
        x = codes.view(torch.uint8)[table].view(F8).float() * scale[table][..., None, None]
        return x.transpose(1, 2).reshape(B, Hkv, -1, D)
    s = torch.matmul(q.float().view(B, Hkv, Hq // Hkv, D), rows(kc, ks).transpose(2, 3)) * st["scale"]
    s = torch.where(t < lens[:, None, None, None], s, -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top > -math.inf, top, 0.0))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, rows(vc, vs)) / torch.where(total > 0, total, 1.0)
    return o.view(B, Hq, D).to(q.dtype)


def _plain_copy(st):
    dev = st["data"].device
    src, dst = (torch.from_numpy(st[k]).to(dev).long() for k in ("src", "dst"))
    raw = _bytes(st["data"])
    if st["tokens"] is None:
        raw[:, :, dst] = raw[:, :, src]
    else:
        keep = torch.arange(st["case"]["page"], device=dev) < torch.from_numpy(st["tokens"]).to(dev)[:, None]
        keep = keep[:, None, :, None] if st["case"]["bits"] == 8 else keep[:, :, None, None]
        raw[:, :, dst] = torch.where(keep, raw[:, :, src], raw[:, :, dst])
    if "scales" in st:
        st["scales"][:, :, dst] = st["scales"][:, :, src]
    return [st["data"]] + ([st["scales"]] if "scales" in st else [])


def _plain_sample(st):
    x = st["logits"]
    x = torch.where(torch.isnan(x), -math.inf, x)
    order, idx = torch.sort(x, dim=-1, descending=True, stable=True)                # equal logits: the lowest index first
    order = order.double()
    it, u, top_p, min_p = (st[k].double()[:, None] for k in ("inv_temp", "u", "top_p", "min_p"))
    d = (order - order[:, :1]) * it
    w = torch.exp(d)
    V = x.shape[1]
    k = torch.where((st["top_k"] <= 0) | (st["top_k"] > V), V, st["top_k"])[:, None]
    wk = torch.where(torch.arange(V, device=x.device) < k, w, 0.0)
    cum = torch.cumsum(wk, -1)
    keep = (wk > 0) & ((top_p >= 1) | (cum - wk <= top_p * cum[:, -1:])) & (w >= min_p)
    kept = torch.zeros_like(w).scatter_(1, idx, torch.where(keep, w, 0.0))      # back in the order of the tokens
    run = torch.cumsum(kept, -1)
    total = run[:, -1:]
    hit = (run > u * total) & (kept > 0)
    tok = torch.where(hit, 1, 0).argmax(-1)
    lp = torch.log(kept.gather(1, tok[:, None]) / total)[:, 0]
    greedy = st["greedy"] != 0
    return [torch.where(greedy, idx[:, 0], tok).int(), torch.where(greedy, -torch.log(w.sum(-1)), lp).float()]


# ------------------------------------------------------------------ one pass
def run(st):
    op = st["case"]["op"]
    if not own:
        return {"append": _plain_append, "decode": _plain_decode, "copy": _plain_copy, "sample": _plain_sample}[op](st)
    from areal_b200.ops import cache_ops as CO
    from areal_b200.ops import sampling as SO
    if op == "append":
        CO.kv8_append(st["k"], st["v"], CO.QuantPages(*st["pages"]), st["table"], st["lens"], st["cu"])
        return st["pages"]
    if op == "decode":
        return CO.kv8_decode(st["q"], CO.QuantPages(*st["pages"]), st["table"], st["lens"], st["scale"])
    if op == "copy":
        wide = st["case"]["bits"] == 8
        planes = [(st["data"], 2, 4 if wide else 3)] + ([(st["scales"], 2, None)] if wide else [])
        CO.copy_pages(planes, st["src"], st["dst"], st["tokens"])
        return [p[0] for p in planes]
    return SO.sample_filtered(st["logits"], st["u"], st["inv_temp"], st["top_k"], st["top_p"], st["min_p"], st["greedy"])


# ------------------------------------------------------------------ in 64 bits
def _round_e4m3(x):
    a = np.minimum(np.abs(x), F8_MAX)
    e = np.maximum(np.frexp(a)[1] - 1, -6)                                      # below 2^-6 the steps stay 2^-9
    step = np.ldexp(1.0, e - 3)
    return np.copysign(np.minimum(np.round(a / step) * step, F8_MAX), x)        # np.round: halves to even


def _exact_append(case, st):
    host = lambda t: t.float().cpu().numpy().astype(np.float64)                 # noqa: E731
    kc, vc, ks, vs = (host(t) for t in st["pages"])
    table, lens, ps = st["table"].cpu().numpy(), st["lens"].tolist(), case["page"]
    cu = st["cu"].tolist() if st["cu"] is not None else None
    for x, codes, scale in ((host(st["k"]), kc, ks), (host(st["v"]), vc, vs)):
        for b, end in enumerate(lens):
            rows = x[cu[b]:cu[b + 1]] if cu else x[b:b + 1]
            begin = end - len(rows)
            if end == 0:
                continue
            for j in range(begin // ps, (end - 1) // ps + 1):
                lo, hi = max(begin, j * ps), min(end, (j + 1) * ps)
                part, pg = rows[lo - begin:hi - begin], table[b, j]
                for h in range(case["kv_heads"]):
                    old = 0.0 if lo == j * ps else scale[pg, h]
                    a, s = np.abs(part[:, h]).max(), 2.0 ** E_MIN
                    while a > F8_MAX * s:
                        s *= 2
                    s = max(s, old)
                    if old and s > old:
                        codes[pg, h] = _round_e4m3(codes[pg, h] * (old / s))
                    codes[pg, h, lo % ps:lo % ps + hi - lo] = _round_e4m3(part[:, h] / s)
                    scale[pg, h] = s
    return [kc, vc, ks, vs]


def _exact_decode(case, st):
    kc, vc, ks, vs = st["pages"]
    q, table, ps = st["q"].double(), st["table"].long(), case["page"]
    G = case["q_heads"] // case["kv_heads"]
    out = torch.zeros_like(q)
    for b, n in enumerate(st["lens"].tolist()):
        if n == 0:
            continue
        pg = table[b, :-(-n // ps)]
        K, V = ((c.view(torch.uint8)[pg].view(F8).double() * s[pg].double()[:, :, None, None]).transpose(0, 1).flatten(1, 2)[:, :n] for c, s in ((kc, ks), (vc, vs)))
        z = torch.einsum("hgd,htd->hgt", q[b].view(-1, G, q.shape[2]), K) * st["scale"]
        out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(z, -1), V).reshape(-1, q.shape[2])
    return out


def _exact_copy(case, st):
    data, ps = st["data"].clone(), case["page"]
    n = [ps] * case["pairs"] if st["tokens"] is None else st["tokens"].tolist()
    for s, d, m in zip(st["src"].tolist(), st["dst"].tolist(), n):
        if case["bits"] == 8:
            data[:, :, d, :, :m].copy_(st["data"][:, :, s, :, :m])
        else:
            data[:, :, d, :m].copy_(st["data"][:, :, s, :m])
    if case["bits"] == 16:
        return [data]
    scales = st["scales"].clone()
    for s, d in zip(st["src"].tolist(), st["dst"].tolist()):
        scales[:, :, d] = st["scales"][:, :, s]
    return [data, scales]


def _exact_sample(case, st):
    col = lambda k: st[k].cpu().numpy().astype(np.float64)                      # noqa: E731
    x, u, it, top_k, top_p, min_p, greedy = (col(k) for k in ("logits", "u", "inv_temp", "top_k", "top_p", "min_p", "greedy"))
    toks, lps = [], []
    for b in range(len(x)):
        order = np.argsort(-x[b], kind="stable")
        z = (x[b] - x[b][order[0]]) * it[b]
        w = np.exp(z).astype(np.longdouble)
        if greedy[b]:
            toks.append(int(order[0]))
            lps.append(float(-np.log(w.sum())))
            continue
        if 0 < top_k[b] < len(order):
            order = order[:int(top_k[b])]
        if top_p[b] < 1:
            before = np.concatenate([[0], np.cumsum(w[order])])
            order = order[before[:-1] <= top_p[b] * before[-1]]
        order = np.sort(order[w[order] >= min_p[b]])
        run = np.cumsum(w[order])
        i = min(int(np.searchsorted(run, u[b] * run[-1], side="right")), len(order) - 1)
        toks.append(int(order[i]))
        lps.append(float(np.log(w[order[i]] / run[-1])))
    return [np.asarray(toks, np.int32), np.asarray(lps)]


def exact(case, seed):
    return {"append": _exact_append, "decode": _exact_decode, "copy": _exact_copy, "sample": _exact_sample}[case["op"]](case, prepare(case, seed))

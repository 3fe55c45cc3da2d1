"""The 8-bit paged cache (append, attention of single tokens), page copies and filtered sampling, against plain statements in
64 bits. What runs without a GPU checks the statements themselves and every refusal."""
import math
from concurrent.futures import ThreadPoolExecutor

import numpy as np
import pytest
import torch

from areal_b200.ops import cache_ops as CO
from areal_b200.ops import lib as oplib
from areal_b200.ops import sampling as SO

F8 = torch.float8_e4m3fn


def _pages(P, Hkv, ps, D, seed=0, device="cpu"):
    """A cache in use: codes of normal rows, scales as an append leaves them."""
    g = torch.Generator().manual_seed(seed)
    p = CO.QuantPages.empty(P, Hkv, ps, D, "cpu")
    for codes, scale in ((p.k, p.k_scale), (p.v, p.v_scale)):
        x = torch.randn(P, Hkv, ps, D, generator=g).double() * torch.exp2(torch.randint(-3, 4, (P, Hkv, 1, 1), generator=g).double())
        s = torch.exp2(torch.ceil(torch.log2(x.abs().amax((2, 3)) / 448)))
        codes.copy_(CO.round_e4m3(x / s[:, :, None, None]).float().to(F8))
        scale.copy_(s)
    return CO.QuantPages(*(t.to(device) for t in (p.k, p.v, p.k_scale, p.v_scale)))


def _clone(p, device=None):
    return CO.QuantPages(*(t.view(torch.uint8).clone().view(F8).to(device or t.device) if t.dtype == F8 else t.clone().to(device or t.device)
                           for t in (p.k, p.v, p.k_scale, p.v_scale)))


def _same(a, b):
    """Equal bit for bit, NaN for NaN."""
    for x, y in zip((a.k, a.v, a.k_scale, a.v_scale), (b.k, b.v, b.k_scale, b.v_scale)):
        x, y = x.float().cpu(), y.float().cpu()
        torch.testing.assert_close(x, y, rtol=0, atol=0, equal_nan=True)


def _no_kernel_error():
    assert oplib.kernel_error() == 0


# ----------------------------------------------------------------------------- the statements themselves
def test_e4m3_rounding_takes_the_nearest_value():
    every = torch.arange(127, dtype=torch.uint8).view(F8).double()             # 0 .. 448
    assert torch.equal(CO.round_e4m3(every), every) and torch.equal(CO.round_e4m3(-every), -every)
    x = torch.linspace(0, 460, 20001, dtype=torch.float64)
    near = every[(x[:, None] - every[None]).abs().argmin(1)]
    assert torch.all((CO.round_e4m3(x) - x).abs() <= (near - x).abs())
    mid = (every[1:] + every[:-1]) / 2                                          # halves: the even code
    code = torch.arange(126) + torch.arange(126) % 2
    assert torch.equal(CO.round_e4m3(mid), every[code])
    assert CO.round_e4m3(torch.tensor(math.inf)) == 448 and torch.isnan(CO.round_e4m3(torch.tensor(math.nan)))


def test_a_scale_is_the_smallest_power_of_two_that_holds_its_page():
    p = CO.QuantPages.empty(2, 1, 16, 64, "cpu")
    table, k = torch.tensor([[1, 0]], dtype=torch.int32), torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    def put(pos, value):
        k[0, 0, 5] = value
        CO.kv8_append(k, k, p, table, torch.tensor([pos + 1], dtype=torch.int32))
        return float(p.k_scale[1, 0])
    assert put(0, 448.0) == 1 and float(p.k[1, 0, 0, 5].float()) == 448
    assert put(1, 450.0) == 2 and float(p.k[1, 0, 1, 5].float()) * 2 == 448        # 450 rounds down to 2 * 224
    assert float(p.k[1, 0, 0, 5].float()) * 2 == 448                            # the first row again, to the new scale
    assert put(2, 1.0) == 2 and put(3, math.inf) == 2 and float(p.k[1, 0, 3, 5].float()) == 448
    assert put(4, math.nan) == 2 and math.isnan(float(p.k[1, 0, 4, 5].float()))
    assert put(0, 2.0 ** -130) == 2.0 ** CO.KV8_E_MIN                           # slot 0: the page starts anew
    assert float(p.k_scale[0, 0]) == 0


def test_the_statement_of_sampling_draws_each_kept_token_with_its_share():
    g = torch.Generator().manual_seed(3)
    V, N = 50, 4000
    x = (torch.randn(1, V, generator=g) * 2).expand(N, V).contiguous()
    u = (torch.arange(N) + 0.5) / N
    one = lambda v, d=torch.float32: torch.full((N,), v, dtype=d)               # noqa: E731
    tok, lp = SO.sample_filtered(x, u, one(0.8), one(12, torch.int32), one(0.9), one(0.01))
    w = torch.exp((x[0].double() - x[0].max()) * float(torch.tensor(0.8)))
    order = torch.sort(w, descending=True).indices[:12]
    cum = torch.cumsum(w[order], 0)
    kept = order[(cum - w[order] <= float(torch.tensor(0.9)) * cum[-1]) & (w[order] >= float(torch.tensor(0.01)))]
    share = torch.zeros(V).double()
    share[kept] = w[kept] / w[kept].sum()
    count = torch.bincount(tok.long(), minlength=V)
    assert torch.all((count - share * N).abs() <= 1)                            # evenly spaced numbers: off by less than one
    assert torch.allclose(lp.double(), torch.log(share[tok.long()]), atol=1e-6)


# ----------------------------------------------------------------------------- refusals
def _append_args(dev="cpu"):
    p = CO.QuantPages.empty(4, 2, 16, 64, dev)
    k = torch.zeros(3, 2, 64, dtype=torch.bfloat16, device=dev)
    return [k, k.clone(), p, torch.zeros(3, 2, dtype=torch.int32, device=dev), torch.ones(3, dtype=torch.int32, device=dev)]


@pytest.mark.parametrize("what", ["dtype", "heads", "rows", "dim", "page", "scales", "table", "lens", "cu", "codes", "strided"])
def test_append_refuses(what):
    a = _append_args()
    if what == "dtype": a[0] = a[0].float()
    if what == "heads": a[0] = a[1] = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    if what == "rows": a[0] = a[1] = torch.zeros(2, 2, 64, dtype=torch.bfloat16)
    if what == "dim": a[0] = a[1] = torch.zeros(3, 2, 32, dtype=torch.bfloat16)
    if what == "page": a[2] = CO.QuantPages.empty(4, 2, 24, 64, "cpu")
    if what == "scales": a[2].k_scale = a[2].k_scale.double()
    if what == "table": a[3] = a[3].long()
    if what == "lens": a[4] = a[4][:2]
    if what == "cu": a.append(torch.zeros(3, dtype=torch.int32))
    if what == "codes": a[2].v = a[2].v.view(torch.uint8)
    if what == "strided": a[2].k = a[2].k.transpose(1, 2)
    with pytest.raises(ValueError):
        CO.kv8_append(*a)


@pytest.mark.parametrize("page,lens", [(4, 1), (-1, 1), (0, 40)])
def test_the_statement_refuses_pages_and_lengths_out_of_range(page, lens):
    a = _append_args()
    a[3][1, 0] = page
    a[4][1] = lens
    with pytest.raises(ValueError):
        CO.kv8_append(*a)


@pytest.mark.parametrize("page,lens", [(4, 1), (-1, 1), (0, 33)])
def test_decode_on_the_host_refuses_pages_and_lengths_out_of_range(page, lens):
    _, _, p, table, n = _append_args()
    q = torch.zeros(3, 4, 64, dtype=torch.bfloat16)
    table[1, 1], n[1] = -5, 16                                                  # an entry behind the sequence's length is not read
    CO.kv8_decode(q, p, table, n)
    table[1, 0], n[1] = page, lens
    with pytest.raises(ValueError):
        CO.kv8_decode(q, p, table, n)


@pytest.mark.parametrize("fits", [True, False])
def test_tables_of_2_to_31_tokens_are_refused(fits):
    """The end of a page has to be an int: 2^24 pages of 128 tokens are one too many."""
    p = CO.QuantPages.empty(4, 2, 128, 64, "cpu")
    k, q = torch.zeros(1, 2, 64, dtype=torch.bfloat16), torch.zeros(1, 4, 64, dtype=torch.bfloat16)
    table, n = torch.zeros(1, 2 ** 24 - fits, dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    for call in (lambda: CO.kv8_append(k, k, p, table, n), lambda: CO.kv8_decode(q, p, table, n)):
        if fits:
            call()
        else:
            with pytest.raises(ValueError, match="2\\^31"):
                call()


def test_decode_refuses_more_than_8192_sequences():
    p = CO.QuantPages.empty(1, 1, 16, 64, "cpu")
    for B in (8192, 8193):
        q, table, lens = torch.zeros(B, 1, 64, dtype=torch.bfloat16), torch.zeros(B, 1, dtype=torch.int32), torch.zeros(B, dtype=torch.int32)
        if B == 8192:
            assert not CO.kv8_decode(q, p, table, lens).any()
        else:
            with pytest.raises(ValueError):
                CO.kv8_decode(q, p, table, lens)


@pytest.mark.parametrize("what", ["dtype", "group", "batch", "dim", "out", "table", "pages"])
def test_decode_refuses(what):
    p = CO.QuantPages.empty(4, 2, 16, 64, "cpu")
    q, table, lens, kw = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.zeros(3, 2, dtype=torch.int32), torch.ones(3, dtype=torch.int32), {}
    if what == "dtype": q = q.half()
    if what == "group": q = torch.zeros(3, 5, 64, dtype=torch.bfloat16)
    if what == "batch": q = q[:2]
    if what == "dim": q = torch.zeros(3, 4, 128, dtype=torch.bfloat16)
    if what == "out": kw["out"] = torch.zeros(3, 4, 64)
    if what == "table": table = torch.zeros(3, 4, dtype=torch.int32)[:, ::2]
    if what == "pages": p = CO.QuantPages.empty(0, 2, 16, 64, "cpu")
    with pytest.raises(ValueError):
        CO.kv8_decode(q, p, table, lens, **kw)


def _off(shape, dtype, by):
    """Contiguous zeros that start ``by`` bytes behind an allocation's beginning."""
    n = int(np.prod(shape)) * torch.empty(0, dtype=dtype).element_size()
    return torch.zeros(n + 16, dtype=torch.uint8)[by:by + n].view(dtype).view(shape)


@pytest.mark.parametrize("what", ["k", "v", "out"])
def test_what_is_read_or_written_sixteen_bytes_at_a_time_has_to_start_there(what):
    a = _append_args()
    q, kw = torch.zeros(3, 4, 64, dtype=torch.bfloat16), {}
    if what == "out":
        kw["out"] = _off(q.shape, q.dtype, 2)
    else:
        setattr(a[2], what, _off(a[2].k.shape, F8, 8))
        with pytest.raises(ValueError, match="16 bytes"):
            CO.kv8_append(*a)
    with pytest.raises(ValueError, match="16 bytes"):
        CO.kv8_decode(q, *a[2:], **kw)


@pytest.mark.parametrize("shift,fits", [(0, False), (64, False), (9 * 64, False), (10 * 64, True)])
def test_decode_refuses_an_output_over_its_queries(shift, fits):
    """Queries are heads 0 to 3 of rows of 6, 2 rows: they end behind 10 heads."""
    a = _append_args()
    buf = torch.zeros(40 * 64, dtype=torch.bfloat16)
    q = buf[:12 * 64].view(2, 6, 64)[:, :4]
    out = buf[shift:][:8 * 64].view(2, 4, 64)
    args = (q, a[2], a[3][:2].contiguous(), a[4][:2].contiguous())
    if fits:
        assert CO.kv8_decode(*args, out=out) is out
    else:
        with pytest.raises(ValueError, match="overlaps"):
            CO.kv8_decode(*args, out=out)


@pytest.mark.parametrize("src,dst,tokens", [([1], [1], None), ([0, 1], [2, 2], None), ([0, 2], [2, 3], None), ([0], [6], None), ([-1], [2], None), ([0], [1, 2], None),
                                            ([0], [1], [17]), ([0], [1], [-1]), ([0, 1], [2, 3], [4])])
def test_copies_refuse(src, dst, tokens):
    t = torch.zeros(3, 6, 16, 8)
    with pytest.raises(ValueError):
        CO.copy_pages([(t, 1, 2)], src, dst, tokens)


def test_copies_refuse_buffers_of_different_caches():
    t = torch.zeros(3, 6, 16, 8)
    for other in ([(torch.zeros(3, 5, 16, 8), 1, 2)], [(torch.zeros(3, 6, 8, 8), 1, 2)], [(t.transpose(0, 1), 1, 2)], [(t, 1, 2)] * 4):
        with pytest.raises(ValueError):
            CO.copy_pages([(t, 1, 2)] + other, [0], [1], [2])


@pytest.mark.parametrize("what", ["logits", "u", "top_k", "rows", "greedy", "out"])
def test_sampling_refuses(what):
    B, V = 3, 10
    f, i = torch.ones(B), torch.ones(B, dtype=torch.int32)
    a = dict(logits=torch.zeros(B, V), u=f * 0.5, inv_temp=f, top_k=i, top_p=f, min_p=f, greedy=i, out=None)
    if what == "logits": a["logits"] = a["logits"].bfloat16()
    if what == "u": a["u"] = a["u"].double()
    if what == "top_k": a["top_k"] = f
    if what == "rows": a["top_p"] = torch.ones(B + 1)
    if what == "greedy": a["greedy"] = torch.ones(B, dtype=torch.bool)
    if what == "out": a["out"] = (i, i)
    with pytest.raises(ValueError):
        SO.sample_filtered(**a)


@pytest.mark.parametrize("which", ["k", "v", "q", "logits", "inv_temp"])
def test_what_requires_a_gradient_is_refused_and_taken_without(which):
    a = _append_args()
    q, f, i = torch.zeros(3, 4, 64, dtype=torch.bfloat16), torch.ones(3), torch.zeros(3, dtype=torch.int32)
    s = dict(logits=torch.zeros(3, 10), u=f * 0.5, inv_temp=f.clone(), top_k=i, top_p=f, min_p=f * 0)
    t, call = {"k": (a[0], lambda: CO.kv8_append(*a)), "v": (a[1], lambda: CO.kv8_append(*a)), "q": (q, lambda: CO.kv8_decode(q, *a[2:])),
               "logits": (s["logits"], lambda: SO.sample_filtered(**s)), "inv_temp": (s["inv_temp"], lambda: SO.sample_filtered(**s))}[which]
    call()
    t.requires_grad_(True)
    with pytest.raises(ValueError, match="no_grad"):
        call()
    with torch.no_grad():
        call()
    with torch.inference_mode():
        call()


def test_copies_on_the_host_leave_the_rest_of_a_page():
    t = torch.arange(2 * 5 * 4 * 3).view(2, 5, 4, 3).clone()
    s, was = torch.arange(10).view(2, 5).clone(), t.clone()
    CO.copy_pages([(t, 1, 2), (s, 1, None)], [0, 0], [3, 1], [2, 0])
    assert torch.equal(t[:, 3, :2], was[:, 0, :2]) and torch.equal(t[:, 3, 2:], was[:, 3, 2:]) and torch.equal(t[:, 1], was[:, 1])
    assert torch.equal(s, torch.tensor([[0, 0, 2, 0, 4], [5, 5, 7, 5, 9]]))


# ----------------------------------------------------------------------------- append on the GPU
def _rows(n, Hkv, D, seed, wide=True):
    """Rows of keys and values as parts of one wider projection, sizes from tiny to large."""
    g = torch.Generator().manual_seed(seed)
    z = torch.randn(n, (2 * Hkv + 3) * D, generator=g) * torch.exp2(torch.randint(-8, 9, (n, 1), generator=g).float())
    z = z.bfloat16()
    k, v = z[:, 3 * D:(3 + Hkv) * D].unflatten(1, (Hkv, D)), z[:, (3 + Hkv) * D:].unflatten(1, (Hkv, D))
    return k, v


def _to_gpu(k, v):
    """Both on the GPU, still as parts of one wider buffer."""
    n, Hkv, D = k.shape
    z = torch.zeros(n, (2 * Hkv + 3) * D, dtype=torch.bfloat16, device="cuda")
    z[:, 3 * D:(3 + Hkv) * D] = k.flatten(1).cuda()
    z[:, (3 + Hkv) * D:] = v.flatten(1).cuda()
    return z[:, 3 * D:(3 + Hkv) * D].unflatten(1, (Hkv, D)), z[:, (3 + Hkv) * D:].unflatten(1, (Hkv, D))


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,D,ps", [(8, 128, 64), (1, 128, 16), (2, 64, 16), (3, 64, 128), (2, 128, 128), (5, 64, 32)])
@pytest.mark.parametrize("B", [1, 3, 37])
def test_append_of_single_tokens(Hkv, D, ps, B):
    g = torch.Generator().manual_seed(B + ps)
    width = 3
    p = _pages(B * width + 2, Hkv, ps, D, B)
    table = torch.randperm(B * width + 2, generator=g)[:B * width].view(B, width).int()
    lens = torch.randint(0, width * ps + 1, (B,), generator=g).int()
    lens[0] = ps + 1                                                            # a new page
    mine = _clone(p, "cuda")
    for step in range(3):
        k, v = _rows(B, Hkv, D, 10 * step + B)
        if B > 2:
            k[1, 0, 3], v[1, Hkv - 1, 0], k[2, 0, 7] = math.inf, math.nan, -math.inf
        CO.kv8_append(k, v, p, table, lens)
        kc, vc = _to_gpu(k, v)
        CO.kv8_append(kc, vc, mine, table.cuda(), lens.cuda())
        _no_kernel_error()
        _same(mine, p)                                                          # every step rounds once, to nearest: the same bits
        lens = torch.where(lens > 0, (lens + 1).clamp(max=width * ps), lens).int()


@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,D,ps", [(8, 128, 64), (1, 128, 16), (2, 64, 16), (3, 64, 128), (2, 128, 128), (5, 64, 32), (2, 128, 32), (4, 64, 64)])
@pytest.mark.parametrize("counts", [[1], [0, 5, 0, 0, 300, 1, 16, 0], [64, 65, 63, 128, 127, 129], [1] * 150 + [0] * 5 + [40]])
def test_append_of_packed_rows(Hkv, D, ps, counts):
    g = torch.Generator().manual_seed(len(counts) + ps)
    B = len(counts)
    n = torch.tensor(counts)
    start = torch.randint(0, 2 * ps, (B,), generator=g)
    start[::3] = 0
    lens = torch.where(n > 0, start + n, 0).int()
    width = int(lens.max()) // ps + 1
    used = [-(-int(x) // ps) for x in lens]
    P = sum(used) + 4
    p = _pages(P, Hkv, ps, D, B)
    table = torch.full((B, width), P - 1, dtype=torch.int32)
    order, at = torch.randperm(P - 1, generator=g).int(), 0
    for b, m in enumerate(used):
        table[b, :m] = order[at:at + m]
        at += m
    cu = torch.tensor([0] + list(n.cumsum(0)), dtype=torch.int32)
    k, v = _rows(int(n.sum()) + 7, Hkv, D, ps)                                  # rows behind the last sequence
    mine = _clone(p, "cuda")
    CO.kv8_append(k, v, p, table, lens, cu)
    kc, vc = _to_gpu(k, v)
    CO.kv8_append(kc, vc, mine, table.cuda(), lens.cuda(), cu.cuda())
    _no_kernel_error()
    _same(mine, p)


@pytest.mark.gpu
def test_append_reports_a_page_out_of_the_cache_and_writes_the_others():
    p = _pages(4, 2, 16, 64, 1)
    mine, k = _clone(p, "cuda"), torch.randn(3, 2, 64).bfloat16()
    table = torch.tensor([[0], [9], [2]], dtype=torch.int32)
    CO.kv8_append(k.cuda(), k.cuda(), mine, table.cuda(), torch.tensor([3, 3, 3], dtype=torch.int32).cuda())
    assert oplib.kernel_error() == 6
    CO.kv8_append(k[::2], k[::2], p, table[::2].contiguous(), torch.tensor([3, 3], dtype=torch.int32))
    _same(mine, p)
    CO.kv8_append(k.cuda(), k.cuda(), mine, table.clamp(max=3).cuda(), torch.tensor([0, 0, 17], dtype=torch.int32).cuda())    # the table ends at 16
    assert oplib.kernel_error() == 6
    _same(mine, p)


# ----------------------------------------------------------------------------- attention of single tokens
def _decode_bound(q, p, table, lens, scale, ref):
    """How far the kernel may be from the statement, from its roundings: the result to bf16, half a step (2^-8); every probability to
    fp16, half a step (2^-11) of its share, and 2^-34 of the largest where it falls below fp16's normal range; a score, a sum of D
    products in fp32, D + 4 half steps (2^-24) of the sum of their sizes, which moves a probability by as much (twice: numerator and
    denominator); the exponential and the sums over tokens, 2^-18 together."""
    out = torch.zeros_like(ref)
    B, Hq, D = q.shape
    Hkv, ps = p.k.shape[1:3]
    for b, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        pg = table[b, :-(-n // ps)].long()
        K, V = ((c.view(torch.uint8)[pg].view(F8).double() * s[pg].double()[:, :, None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
                for c, s in ((p.k, p.k_scale), (p.v, p.v_scale)))
        qb = q[b].double().view(Hkv, -1, D)
        pr = torch.softmax(torch.einsum("hgd,htd->hgt", qb, K) * scale, -1)
        size = torch.einsum("hgd,htd->hgt", qb.abs(), K.abs()) * abs(scale)
        ds = 2 * (D + 4) * 2.0 ** -24 * size.amax(-1, keepdim=True)
        mean = torch.einsum("hgt,htd->hgd", pr, V.abs())
        out[b] = ((2.0 ** -11 + 2.0 ** -18 + ds) * mean + n * 2.0 ** -34 * V.abs().amax(1)[:, None] * pr.amax(-1, keepdim=True)).reshape(Hq, D)
    return out + 2.0 ** -8 * (ref.abs() + out)


def _decode_case(B, Hq, Hkv, D, ps, lens, seed, width=None):
    g = torch.Generator().manual_seed(seed)
    used = [-(-x // ps) for x in lens]
    P = sum(used) + 2
    p = _pages(P, Hkv, ps, D, seed)
    width = width or max(used + [1]) + 1
    table = torch.zeros(B, width, dtype=torch.int32)
    order, at = torch.randperm(P, generator=g).int(), 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    return torch.randn(B, Hq, D, generator=g).bfloat16(), p, table, torch.tensor(lens, dtype=torch.int32)


def _check_decode(q, p, table, lens, scale=None, **kw):
    scale = scale if scale is not None else q.shape[2] ** -0.5
    ref = CO.kv8_decode_ref(q, p, table, lens, scale)
    out = CO.kv8_decode(q.cuda(), _clone(p, "cuda"), table.cuda(), lens.cuda(), scale, **kw)
    _no_kernel_error()
    err = (out.cpu().double() - ref).abs()
    assert torch.all(err <= _decode_bound(q, p, table, lens, scale, ref)), float(err.max())
    return out


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D,ps", [(32, 8, 128, 64), (28, 4, 128, 16), (12, 2, 128, 32), (8, 8, 64, 16), (16, 1, 128, 128), (9, 1, 64, 64), (40, 1, 64, 32),
                                         (34, 2, 128, 16), (4, 4, 128, 64)])
@pytest.mark.parametrize("lens", [[1], [0, 1, 15, 16, 17, 63, 64, 65], [700, 0, 3, 129, 0], [1900], [5] * 60])
def test_decode_heads_and_lengths(Hq, Hkv, D, ps, lens):
    q, p, table, n = _decode_case(len(lens), Hq, Hkv, D, ps, lens, 7)
    out = _check_decode(q, p, table, n)
    assert torch.all(out[torch.tensor(lens).cuda() == 0] == 0)


@pytest.mark.gpu
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (14, 2, 64), (16, 1, 128)])
def test_decode_of_long_ragged_contexts(Hq, Hkv, D):
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(1, 5000, (11,), generator=g).tolist() + [20000, 1]
    q, p, table, n = _decode_case(len(lens), Hq, Hkv, D, 64, lens, 9, width=400)
    _check_decode(q, p, table, n)


@pytest.mark.gpu
def test_decode_values_out_of_the_ordinary():
    # scores far apart (one token takes all), scales that differ by 2^20 between pages, queries of 2^40, what stands behind the last token NaN
    q, p, table, n = _decode_case(4, 8, 2, 128, 16, [50, 33, 16, 100], 3)
    p.v_scale[table[0, 0].long()] *= 2.0 ** 10
    p.v_scale[table[0, 2].long()] *= 2.0 ** -10
    p.k_scale[table[1, 1].long()] *= 2.0 ** 6
    q[2] *= 2.0 ** 40
    p.k_scale[table[2, 0].long()] *= 2.0 ** -40
    for b, m in enumerate(n.tolist()):
        last, slot = int(table[b, (m - 1) // 16]), (m - 1) % 16 + 1
        for c in (p.k, p.v):
            c.view(torch.uint8)[last, :, slot:] = 0x7f
    q[3, 1] = 0
    _check_decode(q, p, table, n)
    _check_decode(q, p, table, n, scale=0.0)
    _check_decode(q, p, table, n, scale=-0.3)


@pytest.mark.gpu
@pytest.mark.parametrize("sign", [-1.0, 1.0])
@pytest.mark.parametrize("exponent", [-20, -8, 0, 60])
def test_decode_of_large_equal_scores(exponent, sign):
    """Equal keys, scores of 101 * 2^37 (101 of 128 dims; times log2 e it has to be rounded) times 2^exponent: the mean of the values. As the scores are equal to the last bit, they add nothing to
    the bound."""
    for lens in ([40], [700], [3, 0, 2000]):
        q, p, table, n = _decode_case(len(lens), 8, 2, 128, 16, lens, 12)
        q.fill_(sign * 2.0 ** 37)
        q[..., :27] = 0
        p.k.view(torch.uint8)[:] = torch.ones(1).to(F8).view(torch.uint8)
        p.k_scale.fill_(2.0 ** exponent)
        q0 = q * 0
        ref = CO.kv8_decode_ref(q, p, table, n, 1.0)
        out = CO.kv8_decode(q.cuda(), _clone(p, "cuda"), table.cuda(), n.cuda(), 1.0).cpu()
        _no_kernel_error()
        assert torch.all((out.double() - ref).abs() <= _decode_bound(q0, p, table, n, 1.0, ref))


def _shares_bound(q, p, table, lens, scale, ref):
    """As :func:`_decode_bound`, but what a probability loses below fp16's normal range is bounded by what the tokens add to the result, not by the largest value
    there is: probability times value scale is held to half of fp16's smallest step, 2^-25, in units in which the largest of them is 2^8 or
    more, and multiplies a code."""
    out = torch.zeros_like(ref)
    B, Hq, D = q.shape
    Hkv, ps = p.k.shape[1:3]
    for b, n in enumerate(lens.tolist()):
        if n <= 0:
            continue
        pg = table[b, :-(-n // ps)].long()
        codes = p.v.view(torch.uint8)[pg].view(F8).double().transpose(0, 1).reshape(Hkv, -1, D)[:, :n].abs()
        K = (p.k.view(torch.uint8)[pg].view(F8).double() * p.k_scale[pg].double()[:, :, None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
        vs = p.v_scale[pg].double().t().repeat_interleave(ps, 1)[:, None, :n]
        qb = q[b].double().view(Hkv, -1, D)
        pr = torch.softmax(torch.einsum("hgd,htd->hgt", qb, K) * scale, -1)
        size = torch.einsum("hgd,htd->hgt", qb.abs(), K.abs()) * abs(scale)
        ds = 2 * (D + 4) * 2.0 ** -24 * size.amax(-1, keepdim=True)
        mean = torch.einsum("hgt,htd->hgd", pr * vs, codes)
        low = 2.0 ** -33 * (pr * vs).amax(-1, keepdim=True) * codes.sum(1)[:, None]
        out[b] = ((2.0 ** -11 + 2.0 ** -18 + ds) * mean + low).reshape(Hq, D)
    return out + 2.0 ** -8 * (ref.abs() + out)


@pytest.mark.gpu
@pytest.mark.parametrize("order", ["large first", "small first", "in turn"])
@pytest.mark.parametrize("apart", [10, 24, 30, 60, 120, 220])
@pytest.mark.parametrize("Hq,Hkv,D,ps,n", [(8, 2, 128, 64, 256), (8, 2, 64, 16, 250), (16, 1, 128, 16, 130), (4, 2, 64, 128, 256), (8, 2, 128, 64, 9000), (24, 2, 64, 32, 5000)])
def test_decode_of_pages_whose_value_scales_are_far_apart(Hq, Hkv, D, ps, n, apart, order):
    """Pages of two value scales, 2^apart from one another. The tokens on the large ones have less weight, by the square root of 2^apart (their values
    decide the result and the others the sum of the weights), by 2^apart and by its square (they have no part in anything)."""
    P = -(-n // ps)
    large = torch.arange(P) < P // 2 if order == "large first" else torch.arange(P) >= -(-P // 2) if order == "small first" else torch.arange(P) // (64 // min(ps, 64)) % 2 == 0
    for much in (0.5, 1.0, 2.0):
        q, p, table, lens = _decode_case(1, Hq, Hkv, D, ps, [n], apart)
        pages = table[0, :P].long()
        p.k.copy_((torch.randn(p.k.shape, generator=torch.Generator().manual_seed(n)) * 0.05).to(F8))
        p.k_scale.fill_(1.0)
        q[..., 0] = 1.0
        raw = p.k.view(torch.uint8)
        raw[pages[large], :, :, 0] = torch.tensor([-much * apart * math.log(2)]).to(F8).view(torch.uint8)
        p.v_scale[pages] = torch.where(large, 2.0 ** (apart - 100), 2.0 ** -100)[:, None].expand(P, Hkv).float()
        ref = CO.kv8_decode_ref(q, p, table, lens, 1.0)
        out = CO.kv8_decode(q.cuda(), _clone(p, "cuda"), table.cuda(), lens.cuda(), 1.0).cpu()
        _no_kernel_error()
        assert torch.all((out.double() - ref).abs() <= _shares_bound(q, p, table, lens, 1.0, ref)), (much, float(((out.double() - ref).abs() / ref.abs()).max()))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [40, 250])
def test_decode_where_one_token_has_most_of_the_weight(n):
    """The largest probability is a power of two in fp16's unit and not rounded, so that the rounding of the others is all there is: less than a tenth of the weight on average, off by 2^-11 of itself at
    most. A result is on the other side of a border of bf16, whose steps are 2^-8 of it or more, with a probability of 0.1 * 2^-11 / 2^-9 = 2.5 % at most."""
    q, p, table, lens = _decode_case(64, 32, 8, 128, 64, [n] * 64, n)
    p.k.copy_((torch.randn(p.k.shape, generator=torch.Generator().manual_seed(n)) * 0.02).to(F8))              # scores of a few tenths, and one of ln(9 n) or a little more
    p.k_scale.fill_(1.0)
    p.v_scale.fill_(1.0)
    q[..., 0] = 1.0
    for b in range(64):
        at = (37 * b) % n
        p.k.view(torch.uint8)[table[b, at // 64].long(), :, at % 64, 0] = torch.tensor([math.log(9 * n) * 1.1]).to(F8).view(torch.uint8)
    ref = CO.kv8_decode_ref(q, p, table, lens, 1.0)
    out = CO.kv8_decode(q.cuda(), _clone(p, "cuda"), table.cuda(), lens.cuda(), 1.0).cpu()
    _no_kernel_error()
    assert float((out != ref.to(torch.bfloat16)).double().mean()) < 0.025


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 200, 6000])
def test_decode_of_the_largest_and_smallest_values(n):
    """Values next to bf16's largest number and to a scale's smallest: the result lies among them and is a number."""
    for e in (119, -100):
        q, p, table, lens = _decode_case(2, 8, 2, 128, 64, [n, n // 2], 31)
        p.v.copy_((torch.rand(p.v.shape, generator=torch.Generator().manual_seed(n)) * 100 + 150).to(F8))          # below 2^8: values below 2^127
        p.v_scale.fill_(2.0 ** e)
        ref = CO.kv8_decode_ref(q, p, table, lens)
        out = CO.kv8_decode(q.cuda(), _clone(p, "cuda"), table.cuda(), lens.cuda()).cpu()
        _no_kernel_error()
        assert torch.all((out.double() - ref).abs() <= _shares_bound(q, p, table, lens, 128 ** -0.5, ref))


@pytest.mark.gpu
def test_decode_takes_parts_of_a_projection_and_reports_bad_tables():
    q, p, table, n = _decode_case(5, 8, 2, 64, 32, [40, 1, 200, 0, 64], 4)
    z = torch.randn(5, 12 * 64).bfloat16().cuda()
    part = z[:, 2 * 64:10 * 64].unflatten(1, (8, 64))
    part.copy_(q.cuda())
    buf = torch.full((5, 8, 64), 7.0, dtype=torch.bfloat16, device="cuda")
    a = CO.kv8_decode(part, _clone(p, "cuda"), table.cuda(), n.cuda(), out=buf)
    assert a is buf and torch.equal(a, _check_decode(q, p, table, n))
    bad = table.clone()
    bad[2, 3] = 10 ** 6
    o = CO.kv8_decode(q.cuda(), _clone(p, "cuda"), bad.cuda(), n.cuda())
    assert oplib.kernel_error() == 6
    keep = torch.tensor([0, 1, 3, 4]).cuda()
    assert torch.equal(o[keep], a[keep])
    CO.kv8_decode(q.cuda(), _clone(p, "cuda"), table.cuda(), (n * 0 + table.shape[1] * 32 + 1).cuda())
    assert oplib.kernel_error() == 6


@pytest.mark.gpu
def test_decode_is_the_same_run_after_run_on_streams_and_in_graphs():
    q, p, table, n = (t.cuda() if torch.is_tensor(t) else _clone(t, "cuda") for t in _decode_case(9, 32, 8, 128, 64, [900, 1, 64, 0, 2000, 300, 77, 5, 1200], 6))
    first = CO.kv8_decode(q, p, table, n)
    torch.cuda.synchronize()
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    outs = []
    for i in range(6):
        with torch.cuda.stream((a, b)[i % 2]):
            outs.append(CO.kv8_decode(q, p, table, n))
    graphs = []
    for s in (a, b):
        g = torch.cuda.CUDAGraph()
        s.synchronize()
        with torch.cuda.graph(g, stream=s):
            o = CO.kv8_decode(q, p, table, n)
        graphs.append((g, o))
    torch.cuda.synchronize()
    for _ in range(3):
        for s, (g, _o) in zip((a, b), graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(o, first) for o in outs + [o for _, o in graphs])
    q2 = torch.randn_like(q)                                                    # new contents, other lengths: the graph reads them
    q.copy_(q2)
    n.copy_(torch.tensor([1, 900, 0, 64, 3, 301, 600, 5, 1100], dtype=torch.int32))
    table.copy_(table[[1, 0, 3, 2, 4, 5, 8, 7, 6]].contiguous())
    graphs[0][0].replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], CO.kv8_decode(q, p, table, n))
    _no_kernel_error()


@pytest.mark.gpu
@pytest.mark.parametrize("B", [129, 1000, 8192])
def test_decode_of_many_short_contexts(B):
    g = torch.Generator().manual_seed(B)
    lens = torch.randint(0, 30, (B,), generator=g).tolist()
    lens[B // 2] = 900
    _check_decode(*_decode_case(B, 2, 1, 64, 16, lens, B))


@pytest.mark.gpu
def test_pages_whose_offsets_pass_32_bits():
    """A cache of 4.3 GB of keys: append, attention and copies on its last pages do what they do on a small one with the same pages in front."""
    P, Hkv, ps, D, n = 66000, 8, 64, 128, 6
    big, small = CO.QuantPages.empty(P, Hkv, ps, D, "cuda"), CO.QuantPages.empty(n, Hkv, ps, D, "cuda")
    assert big.k.numel() > 2 ** 32
    table = torch.tensor([[0, 1, 2], [3, 4, 5]], dtype=torch.int32, device="cuda")
    lens = torch.tensor([150, 70], dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, 150, 220], dtype=torch.int32, device="cuda")
    k, v, q = (torch.randn(m, h, D, device="cuda").bfloat16() for m, h in ((220, Hkv), (220, Hkv), (2, 4 * Hkv)))
    outs = []
    for p, t in ((small, table), (big, table + (P - n))):
        CO.kv8_append(k, v, p, t, lens, cu)
        CO.kv8_append(k[:2], v[:2], p, t, lens + 1)
        outs.append(CO.kv8_decode(q, p, t, lens + 1))
    assert torch.equal(outs[0], outs[1])
    tail = lambda x: (x.view(torch.uint8) if x.dtype == F8 else x)[P - n:]                     # noqa: E731
    for x, y in zip((small.k, small.v, small.k_scale, small.v_scale), (big.k, big.v, big.k_scale, big.v_scale)):
        assert torch.equal(x.view(torch.uint8) if x.dtype == F8 else x, tail(y))
    codes = big.k.view(torch.uint8)
    assert not codes[:P - n].any()
    CO.copy_pages([(codes, 0, 2), (big.k_scale, 0, None)], [P - 6, P - 5, P - 3], [1, P - 1, 0], [64, 33, 1])
    for s, d, m in ((P - 6, 1, 64), (P - 5, P - 1, 33), (P - 3, 0, 1)):
        assert torch.equal(codes[s, :, :m], codes[d, :, :m]) and torch.equal(big.k_scale[s], big.k_scale[d]) and not codes[d, :, m:].any()
    _no_kernel_error()


@pytest.mark.gpu
def test_decode_called_by_threads_that_share_a_stream():
    args = []
    for i, lens in enumerate(([900, 1, 64, 3000], [0, 2000, 1200, 5], [1, 1, 1, 4000], [700, 700, 700, 700])):
        q, p, table, n = _decode_case(4, 16, 4, 64, 64, lens, 20 + i, width=70)
        args.append((q.cuda(), _clone(p, "cuda"), table.cuda(), n.cuda()))
    want = [CO.kv8_decode(*a) for a in args]
    torch.cuda.synchronize()

    def many(a):
        torch.cuda.set_device(0)
        return [CO.kv8_decode(*a) for _ in range(200)]
    with ThreadPoolExecutor(len(args)) as pool:
        got = list(pool.map(many, args))
    torch.cuda.synchronize()
    assert all(torch.equal(o, w) for outs, w in zip(got, want) for o in outs)
    _no_kernel_error()


# ----------------------------------------------------------------------------- launch accounting
def test_kernels_of_a_call_are_counted_from_its_arguments(monkeypatch):
    class Fake:
        def __getattr__(self, name):
            return lambda *a: 0
    fake = oplib._CountingLib(Fake())

    def counted(name, *a):
        before = oplib.launch_count()
        getattr(fake, name)(*a)
        return oplib.launch_count() - before
    monkeypatch.setitem(oplib.LAUNCHES, "count", 0)
    decode = lambda ps, width: counted("ab2_kv8_decode", *[0] * 9, 3, 8, 2, 64, ps, width, 10, 1.0, 0, 0)      # noqa: E731
    assert [decode(64, 4), decode(64, 5), decode(16, 16), decode(16, 17), decode(128, 2), decode(128, 3)] == [1, 2, 1, 2, 1, 2]
    assert [counted("ab2_copy_pages", b"", 1, b"", n, 0) for n in (1, 256, 257, 1000)] == [1, 1, 2, 4]
    assert counted("ab2_kv8_append") == 1 and counted("ab2_sample_filtered") == 1 and counted("ab2_gemm_splitk") == 2 and counted("ab2_num_sms") == 0


@pytest.mark.gpu
def test_kernels_counted_are_those_of_a_captured_call():
    from cuda.bindings import runtime as rt

    t, s = torch.zeros(700, 16, 8, device="cuda"), torch.cuda.Stream()
    small, long = (tuple(x.cuda() if torch.is_tensor(x) else _clone(x, "cuda") for x in _decode_case(2, 8, 2, 64, 16, lens, 8, width=w)) for lens, w in (([200, 5], 16), ([250, 5], 17)))
    c = {k: v.cuda() for k, v in _sampling_case(3, 1000, 1, "normal").items()}
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call, n in ((lambda: CO.kv8_decode(*small), 1), (lambda: CO.kv8_decode(*long), 2), (lambda: CO.copy_pages([(t, 0, 1)], range(300), range(300, 600)), 2),
                    (lambda: CO.copy_pages([(t, 0, 1)], [0], [1]), 1), (lambda: CO.kv8_append(k, k, small[1], small[2], small[3]), 1), (lambda: SO.sample_filtered(**c), 1)):
        call()
        torch.cuda.synchronize()
        g, before = torch.cuda.CUDAGraph(keep_graph=True), oplib.launch_count()
        with torch.cuda.graph(g, stream=s):
            call()
        assert oplib.launch_count() - before == n
        err, _, nodes = rt.cudaGraphGetNodes(rt.cudaGraph_t(g.raw_cuda_graph()), 0)
        assert int(err) == 0 and nodes == n


# ----------------------------------------------------------------------------- page copies
@pytest.mark.gpu
@pytest.mark.parametrize("Hkv,D,ps,layers", [(8, 128, 64, 3), (2, 64, 16, 4), (1, 128, 128, 1), (3, 24, 20, 2)])
@pytest.mark.parametrize("n", [1, 7, 300])
@pytest.mark.parametrize("part", [False, True])
def test_copies_of_both_caches(Hkv, D, ps, layers, n, part):
    rng = np.random.RandomState(n)
    P = 2 * n + 3
    order = rng.permutation(P)
    src, dst = order[:n].copy(), order[n:2 * n]
    src[n // 2:] = src[0]
    tokens = rng.randint(0, ps + 1, n) if part else None
    wide = torch.randn(layers, 2, P, ps, Hkv, D).bfloat16()
    codes = torch.randint(0, 256, (layers, 2, P, Hkv, ps, D), dtype=torch.uint8)
    scales = torch.randn(layers, 2, P, Hkv)
    odd = torch.randint(0, 256, (P, 3), dtype=torch.uint8)
    host = [wide, codes, scales, odd]
    dims = [(2, 3), (2, 4), (2, None), (0, None)]
    mine = [t.cuda() for t in host]
    CO.copy_pages([(t, *d) for t, d in zip(mine, dims)], src, dst, tokens)
    CO.copy_pages_ref([(t, *d) for t, d in zip(host, dims)], src, dst, tokens)
    assert all(torch.equal(a.cpu().view(torch.uint8), b.view(torch.uint8)) for a, b in zip(mine, host))


# ----------------------------------------------------------------------------- sampling
def _sampling_case(B, V, seed, kind):
    g = torch.Generator().manual_seed(seed)
    r = np.random.RandomState(seed)
    x = torch.randn(B, V, generator=g) * 2.3
    if kind == "peaked":
        x.scatter_add_(1, torch.randint(0, V, (B, min(V, 40)), generator=g), torch.rand(B, min(V, 40), generator=g) * 16)
    if kind == "rounded":
        x = (x * 2).round() / 2                                                 # thousands of equal logits
    if kind == "equal":
        x = torch.full((B, V), -3.25)
    if kind == "flat":
        x = x * 0.01
    if kind == "masked":
        x[:, ::3] = torch.finfo(torch.float32).min
        x[:, 1::3] = -math.inf
        x[:, min(4, V - 1)] = math.nan
    if kind == "wide":
        x = x * 1e3
    f = lambda a: torch.tensor(np.asarray(a), dtype=torch.float32)              # noqa: E731
    i = lambda a: torch.tensor(np.asarray(a), dtype=torch.int32)                # noqa: E731
    return dict(logits=x, u=torch.rand(B, generator=g), inv_temp=f(1 / r.choice([0.3, 0.7, 1.0, 1.0, 2.0], B)), top_k=i(r.choice([0, 0, 1, 5, 50, 3000, 10 ** 8], B)),
                top_p=f(r.choice([1.0, 1.0, 0.0, 0.3, 0.9, 0.95, 0.999], B)), min_p=f(r.choice([0.0, 0.0, 0.001, 0.1, 1.0], B)), greedy=i(r.rand(B) < 0.1))


def _check_sampling(c):
    tok, lp = SO.sample_filtered_ref(**c)
    got, glp = SO.sample_filtered(**{k: v.cuda() for k, v in c.items()})
    assert torch.equal(got.cpu(), tok), [(int(a), int(b)) for a, b in zip(got.cpu(), tok) if a != b][:5]
    # both in 64 bits, rounded once to fp32 (half a step each); sums in other orders move the log by less than 1e-9
    fin = torch.isfinite(lp)
    assert torch.equal(fin, torch.isfinite(glp.cpu()))
    assert torch.all((glp.cpu()[fin].double() - lp[fin].double()).abs() <= 2.0 ** -23 * lp[fin].abs().double() + 1e-9)
    _no_kernel_error()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["normal", "peaked", "rounded", "equal", "flat", "masked", "wide"])
@pytest.mark.parametrize("B,V", [(40, 1), (40, 2), (40, 37), (60, 1024), (40, 5000), (40, 20481), (24, 50001), (24, 151936)])
def test_sampling_matches_the_statement(kind, B, V):
    _check_sampling(_sampling_case(B, V, V % 97 + B, kind))


@pytest.mark.gpu
def test_sampling_one_filter_at_a_time():
    for name, value in (("top_p", 0.9), ("top_p", 0.5), ("top_k", 20), ("top_k", 2500), ("top_k", 30000), ("min_p", 0.05), ("min_p", 1e-6), ("none", 0), ("greedy", 1)):
        for kind in ("normal", "peaked", "rounded"):
            c = _sampling_case(16, 65536, 3, kind)
            c["top_k"].zero_(); c["top_p"].fill_(1.0); c["min_p"].zero_(); c["greedy"].zero_()
            if name != "none":
                c[name].fill_(value)
            _check_sampling(c)


@pytest.mark.gpu
def test_sampling_top_p_behind_a_long_top_k():
    for kind in ("normal", "rounded", "flat", "equal"):
        for k in (2049, 4096, 20000):
            for p in (0.2, 0.9, 0.9999):
                c = _sampling_case(6, 32768, k, kind)
                c["top_k"].fill_(k); c["top_p"].fill_(p); c["min_p"].zero_(); c["greedy"].zero_()
                _check_sampling(c)


@pytest.mark.gpu
def test_sampling_rows_at_the_edges():
    V = 700
    x = torch.randn(8, V)
    x[0] = -math.inf
    x[1] = math.nan
    x[2, 5] = x[2, 9] = math.inf
    x[3] = -math.inf
    x[3, V - 1] = -1e38
    x[4, :] = 0
    f = torch.ones(8)
    c = dict(logits=x, u=torch.tensor([0.5, 0.5, 0.75, 0.0, 1 - 2.0 ** -24, 0.0, 0.999999, 0.3]), inv_temp=f, top_k=torch.zeros(8, dtype=torch.int32), top_p=f.clone(),
             min_p=torch.zeros(8), greedy=torch.zeros(8, dtype=torch.int32))
    c["logits"] = torch.where(torch.isposinf(x), torch.full_like(x, 0.0), x)     # the statement for row 2: two equal logits, all others without weight
    c["logits"][2] = torch.where(torch.isposinf(x[2]), 0.0, -math.inf)
    tok, lp = SO.sample_filtered_ref(**c)
    c["logits"] = x
    got, glp = SO.sample_filtered(**{k: v.cuda() for k, v in c.items()})
    assert torch.equal(got.cpu(), tok) and int(got[2]) == 9 and int(got[0]) == -1 and int(got[1]) == -1 and int(got[4]) == V - 1
    assert torch.isneginf(glp[:2]).all() and torch.allclose(glp.cpu()[2:], lp[2:], rtol=1e-6, atol=1e-9)
    c["logits"] = x[4:5]                                                        # uniform: the exclusive sum of token i is i / V, kept up to equality
    for p, u, want in ((0.25, 0.999999, 175), (0.0, 0.9, 0), (0.25, 0.0, 0)):
        got, _ = SO.sample_filtered(x[4:5].cuda(), torch.tensor([u]).cuda(), f[:1].cuda(), c["top_k"][:1].cuda(), torch.tensor([p]).cuda(), c["min_p"][:1].cuda())
        assert int(got) == want


def _masked_rows(V, low, offset, kind, u, **filters):
    """Rows in which all but a window of tokens stand at ``low`` (its first two rows: the window at the front and at the end)."""
    g = torch.Generator().manual_seed(V)
    B = 6
    x = torch.full((B, V), low)
    n = max(1, min(V // 3, 5000) if kind == "long" else min(V // 3, 90))
    for b in range(B):
        at = (0, V - n)[b] if b < 2 else int(torch.randint(0, V - n + 1, (1,), generator=g))
        x[b, at:at + n] = (torch.randn(n, generator=g) * 2 if kind != "equal" else torch.zeros(n)) + offset
    f = lambda v: torch.full((B,), float(v))                                    # noqa: E731
    i = lambda v: torch.full((B,), int(v), dtype=torch.int32)                   # noqa: E731
    return dict(logits=x, u=f(u), inv_temp=f(filters.get("inv_temp", 1.0)), top_k=i(filters.get("top_k", 0)), top_p=f(filters.get("top_p", 1.0)),
                min_p=f(filters.get("min_p", 0.0)), greedy=i(0))


FILTERS_AT_ZERO = [{}, dict(top_k=50), dict(top_k=2000), dict(top_k=30000), dict(top_p=0.9), dict(top_p=0.9999999), dict(min_p=0.1), dict(min_p=1e-30), dict(top_k=4000, top_p=0.999),
                   dict(top_k=40, min_p=1e-9), dict(top_p=0.99999, min_p=1e-20), dict(inv_temp=50.0), dict(inv_temp=50.0, top_k=3000)]


def test_the_statement_draws_no_masked_token():
    for low, offset in ((torch.finfo(torch.float32).min, 0.0), (-1e4, 1000.0), (-math.inf, 0.0), (-690.0, 12.0)):
        for filters in FILTERS_AT_ZERO:
            c = _masked_rows(300, low, offset, "short", 0.0, **filters)
            tok, lp = SO.sample_filtered_ref(**c)
            assert torch.all(c["logits"].gather(1, tok[:, None].long()) > low) and torch.all(lp > -700), (low, filters)


@pytest.mark.gpu
@pytest.mark.parametrize("low,offset", [(torch.finfo(torch.float32).min, 0.0), (-1e4, 0.0), (-690.0, 12.0), (torch.finfo(torch.float32).min, 1000.0), (-math.inf, 0.0)])
@pytest.mark.parametrize("V", [37, 1024, 5000, 50001, 151936])
def test_sampling_at_u_zero_takes_no_masked_token(V, low, offset):
    for kind in ("short", "long", "equal"):
        for filters in FILTERS_AT_ZERO:
            for u in (0.0, 2.0 ** -24):
                _check_sampling(_masked_rows(V, low, offset, kind, u, **filters))


@pytest.mark.gpu
@pytest.mark.parametrize("V", [131072, 151936, 393216])
@pytest.mark.parametrize("first,at,end", [(16.61, 16.7, 16.85), (16.7, 18.0, 20.0), (30.0, 31.0, 33.0)])
def test_sampling_of_nuclei_that_end_far_below_the_largest(V, first, at, end):
    """One large logit and thousands of small ones, most of them ``first`` to ``at`` nats down and 6000 from there to ``end``, where the nucleus ends. Together they are a small part of the
    total and each is 6e-8 of it or less: the border, and the token drawn next to the end of the sum, are those of a total in 64 bits, in
    whatever order the tokens stand."""
    g = torch.Generator().manual_seed(V)
    it = torch.tensor([1 / 0.7]).float()
    down = torch.cat([torch.linspace(first, at, V - 6001, dtype=torch.float64), torch.linspace(at, end, 6000, dtype=torch.float64)]).float() / it
    x = torch.empty(16, V)
    x[:, 0] = 195.0625 + 0.4375 * (torch.arange(16) % 8)                        # (times 64 / 0.7 it is rounded by nearly half a step of 32 bits, always upwards)
    x[:, 1:] = x[:, :1] - down
    w = torch.exp((x[0].double() - x[0, 0].double()) * it.double())
    p = torch.tensor([float(w[:V - a].sum() / w.sum()) for a in (5000, 4000, 3000, 2500, 2000, 1500, 1000, 500)] * 2).clamp(max=1 - 2.0 ** -24).float()
    for b in range(8, 16):
        x[b] = x[b, torch.randperm(V, generator=g)]
    c = dict(logits=x, u=torch.full((16,), 1 - 2.0 ** -24), inv_temp=it.expand(16).contiguous(), top_k=torch.zeros(16, dtype=torch.int32), top_p=p,
             min_p=torch.zeros(16), greedy=None)
    tok, lp = SO.sample_filtered_ref(**c)
    got, glp = SO.sample_filtered(**{k: v if v is None else v.cuda() for k, v in c.items()})
    assert torch.equal(got.cpu(), tok), (got.cpu() - tok).tolist()
    assert torch.all((glp.cpu().double() - lp.double()).abs() <= 2.0 ** -23 * lp.abs().double() + 1e-9)
    _no_kernel_error()


@pytest.mark.gpu
@pytest.mark.parametrize("V", [3, 37, 1024, 5000, 50001])
def test_sampling_takes_both_zeros_for_one_value(V):
    """Logits of plus and minus zero tie, as the largest value, at the end of a top-k and at the border of a nucleus: the lowest indices come first."""
    g = torch.Generator().manual_seed(V)
    B = 24
    for top in (0.0, 3.0):
        x = (torch.randn(B, V, generator=g) * 1.2 + top / 2).round().clamp(max=top)
        x = torch.where(x == 0, torch.where(torch.rand(B, V, generator=g) < 0.5, 0.0, -0.0), x)
        above = (x > 0).sum(1)
        for filters in (dict(top_k=above + 1), dict(top_k=above + V // 8 + 1), dict(top_p=0.0), dict(top_p=0.5), dict(top_p=0.7, top_k=torch.full((B,), V - 1)), dict(top_k=above + 3, top_p=0.6)):
            p = filters.get("top_p", 1.0)
            _check_sampling(dict(logits=x, u=torch.rand(B, generator=g), inv_temp=torch.ones(B), top_k=filters.get("top_k", torch.zeros(B)).int(), top_p=torch.full((B,), p),
                                 min_p=torch.zeros(B), greedy=(torch.arange(B) % 6 == 5).int()))


@pytest.mark.gpu
def test_sampling_slices_streams_and_graphs():
    c = {k: v.cuda() for k, v in _sampling_case(33, 9973, 2, "peaked").items()}
    first = SO.sample_filtered(**c)
    wide = torch.full((33, 10007), 50.0, device="cuda")
    wide[:, 11:11 + 9973] = c["logits"]
    again = SO.sample_filtered(**{**c, "logits": wide[:, 11:11 + 9973]})
    out = torch.empty(33, dtype=torch.int32, device="cuda"), torch.empty(33, device="cuda")
    g = torch.cuda.CUDAGraph()
    s = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=s):
        SO.sample_filtered(**c, out=out)
    g.replay()
    torch.cuda.synchronize()
    for r in (again, out):
        assert torch.equal(r[0], first[0]) and torch.equal(r[1], first[1])
    c["u"].copy_(torch.rand(33))
    g.replay()
    new = SO.sample_filtered(**c)
    torch.cuda.synchronize()
    assert torch.equal(new[0], out[0]) and torch.equal(new[1], out[1])

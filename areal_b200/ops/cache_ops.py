"""Paged key/value cache in 8 bits: rows quantised into it, attention of single tokens over it, and copies of pages of either
cache.

Layout of one layer (:class:`QuantPages`): codes e4m3 ``[pages, Hkv, page_size, D]``, fp32 scales ``[pages, Hkv]``, powers of two, one
for the tokens of a page and head; value = code * scale. The scale of a page that receives rows is the smallest power of two that
holds its largest finite element (|x| <= 448 * scale), never smaller than what the page already has; where it grows, the page's other
codes are rounded again to the new one. Writing slot 0 starts a page: what stood in it counts for nothing.

As in :mod:`.functional`, CUDA tensors run the sm_100a kernels and CPU tensors the plain statements (``*_ref``), computed in 64 bits.
The engine takes this cache with ``NativeInferConfig.kv_cache_dtype = "float8_e4m3"``. There are no gradients: rows, queries or logits that require them are refused
unless they are switched off.
"""
from __future__ import annotations

import functools
import struct
from dataclasses import dataclass
from typing import Optional, Sequence

import torch

from . import lib as _lib

F8 = torch.float8_e4m3fn
KV8_MAX = 448.0
KV8_E_MIN, KV8_E_MAX = -100, 120
PAGE_SIZES = (16, 32, 64, 128)
WIDEST = (1 << 31) - 64                      # tokens of a page table: positions up to the end of a page or tile are counted in 32 bits

_V, _I, _F, _L = _lib.c_void_p, _lib.c_int, _lib.c_float, _lib.c_ll


@dataclass
class QuantPages:
    """The 8-bit pages of one layer."""

    k: torch.Tensor              # [pages, Hkv, page_size, D] e4m3
    v: torch.Tensor
    k_scale: torch.Tensor        # [pages, Hkv] fp32
    v_scale: torch.Tensor

    @staticmethod
    def empty(pages: int, kv_heads: int, page_size: int, dim: int, device) -> "QuantPages":
        k, v = (torch.zeros(pages, kv_heads, page_size, dim, device=device, dtype=torch.uint8).view(F8) for _ in range(2))
        ks, vs = (torch.zeros(pages, kv_heads, device=device) for _ in range(2))
        return QuantPages(k, v, ks, vs)

    def dense(self, dtype=torch.float32) -> tuple[torch.Tensor, torch.Tensor]:
        """Keys and values as numbers."""
        return tuple(c.to(dtype) * s.to(dtype)[:, :, None, None] for c, s in ((self.k, self.k_scale), (self.v, self.v_scale)))


def _need(ok: bool, what: str) -> None:
    if not ok:
        raise ValueError(what)


def _no_gradients(*tensors) -> None:
    """Refuses what a backward pass would expect a gradient for: the result would be cut off from it without a word."""
    if torch.is_grad_enabled() and any(t.requires_grad for t in tensors):
        raise ValueError("serving operators have no gradients: call them under torch.no_grad()")


def _check_pages(p: QuantPages, dim: int, dev: int) -> tuple:
    """(pages, Hkv, page size) of a cache on device number ``dev`` (-1: the host), after its checks."""
    k, v, ks, vs = p.k, p.v, p.k_scale, p.v_scale
    s = k.shape
    if (len(s) == 4 and v.shape == s and k.dtype is F8 and v.dtype is F8 and ks.dtype is torch.float32 and vs.dtype is torch.float32 and ks.shape == s[:2]
            and vs.shape == s[:2] and k.is_contiguous() and v.is_contiguous() and ks.is_contiguous() and vs.is_contiguous() and s[2] in PAGE_SIZES
            and s[3] == dim and (dim == 128 or dim == 64) and s[0] > 0 and s[1] > 0
            and k.get_device() == v.get_device() == ks.get_device() == vs.get_device() == dev and not (k.data_ptr() | v.data_ptr()) & 15):
        return s[0], s[1], s[2]
    # which of them it is
    _need(k.dtype == F8 and v.dtype == F8 and len(s) == 4 and v.shape == s, "codes: two e4m3 tensors [pages, Hkv, page_size, D]")
    _need(k.is_contiguous() and v.is_contiguous(), "codes have to be contiguous")
    _need(ks.dtype == torch.float32 and vs.dtype == torch.float32 and ks.shape == s[:2] and vs.shape == s[:2] and ks.is_contiguous() and vs.is_contiguous(),
          "scales: two contiguous fp32 tensors [pages, Hkv]")
    _need(s[3] == dim and dim in (64, 128), f"head size {dim} with a cache of {s[3]}: 64 or 128 are built")
    _need(s[2] in PAGE_SIZES, f"page size {s[2]}: one of {PAGE_SIZES}")
    _need(s[0] > 0 and s[1] > 0, "a cache without pages or heads")
    _need(not (k.data_ptr() | v.data_ptr()) & 15, "codes have to start on 16 bytes")
    raise ValueError("cache on another device than the rows")


def _check_table(table, lens, B: int, dev: int) -> int:
    """The table's width, after its checks."""
    t = table.shape
    if (len(t) == 2 and t[0] == B and t[1] > 0 and table.dtype is torch.int32 and lens.dtype is torch.int32 and lens.shape == t[:1] and table.is_contiguous()
            and lens.is_contiguous() and table.get_device() == lens.get_device() == dev):
        return t[1]
    _need(len(t) == 2 and table.dtype == torch.int32 and table.is_contiguous() and t[1] > 0, "page table: contiguous int32 [B, width]")
    _need(t[0] == B, f"a table of {t[0]} sequences for {B}")
    _need(lens.dtype == torch.int32 and lens.is_contiguous() and lens.shape == t[:1], "lengths: contiguous int32 [B]")
    raise ValueError("page table or lengths on another device")


def _launch(dev: int, name: str, *args) -> None:
    """Calls a launcher on device number ``dev`` and its current stream."""
    if dev == torch._C._cuda_getDevice():
        rc = getattr(_lib.get_lib(), name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            rc = getattr(_lib.get_lib(), name)(*args, torch._C._cuda_getCurrentRawStream(dev))
    if rc:
        _lib.check(rc, name)


# ----------------------------------------------------------------------------- append
def _exponent(amax: torch.Tensor) -> torch.Tensor:
    m, e = torch.frexp(amax)                                     # amax = m * 2^e, m in [1/2, 1)
    e = torch.where(m <= KV8_MAX / 512, e - 9, e - 8)
    return torch.where(amax > 0, e, torch.full_like(e, KV8_E_MIN)).clamp(KV8_E_MIN, KV8_E_MAX)


def round_e4m3(x: torch.Tensor) -> torch.Tensor:
    """The nearest e4m3 value of each element (halves to even, beyond 448 the largest), in the type of ``x``."""
    a = x.abs().clamp(max=KV8_MAX)
    e = torch.frexp(a)[1].clamp(min=-5) - 4                      # steps of 2^-3 of the leading power, 2^-9 below 2^-6
    step = torch.ldexp(torch.ones_like(a), e)
    return torch.copysign(torch.round(a / step) * step, x)


def kv8_append_ref(k, v, pages: QuantPages, page_table, seq_lens, cu_seqlens=None) -> None:
    """Plain statement of :func:`kv8_append`, page by page in 64 bits."""
    P, _, ps, _ = pages.k.shape
    B, width = page_table.shape
    cu = cu_seqlens.tolist() if cu_seqlens is not None else None
    for b, end in enumerate(seq_lens.tolist()):
        lo_row, hi_row = (cu[b], cu[b + 1]) if cu else (b, b + (end > 0))
        start = end - (hi_row - lo_row)
        if hi_row <= lo_row:
            continue
        _need(start >= 0 and end <= width * ps and hi_row <= k.shape[0], f"sequence {b}: {hi_row - lo_row} rows at the end of {end} tokens do not fit")
        for j in range(start // ps, (end - 1) // ps + 1):
            page = int(page_table[b, j])
            _need(0 <= page < P, f"page {page} of sequence {b} is not in the cache")
            lo, hi = max(start, j * ps), min(end, (j + 1) * ps)
            slot = lo - j * ps
            for x, codes, scales in ((k, pages.k, pages.k_scale), (v, pages.v, pages.v_scale)):
                rows = x[lo_row + lo - start:lo_row + hi - start].double().transpose(0, 1)          # [Hkv, n, D]
                old = scales[page].double() if slot else torch.zeros_like(scales[page], dtype=torch.float64)
                amax = torch.where(torch.isfinite(rows), rows.abs(), torch.zeros_like(rows)).amax((1, 2))
                s = torch.maximum(old, torch.ldexp(torch.ones_like(amax), _exponent(amax)))
                ratio = torch.where((old > 0) & (s > old), old / s, torch.ones_like(s))
                block = round_e4m3(codes[page].double() * ratio[:, None, None])
                block[:, slot:slot + hi - lo] = round_e4m3(rows / s[:, None, None])
                codes[page] = block.float().to(F8)
                scales[page] = s.float()


def kv8_append(k: torch.Tensor, v: torch.Tensor, pages: QuantPages, page_table: torch.Tensor, seq_lens: torch.Tensor,
               cu_seqlens: Optional[torch.Tensor] = None) -> None:
    """Quantises rows ``k``, ``v`` ``[rows, Hkv, D]`` bf16 into the pages of their sequences, behind what those hold.

    Without ``cu_seqlens`` row ``b`` is the last token of sequence ``b``, at position ``seq_lens[b] - 1``; a row of length 0 has none. With it
    sequence ``b`` brings the rows ``cu_seqlens[b] .. cu_seqlens[b + 1]`` as its last ones; rows behind ``cu_seqlens[B]`` are left out. Rows
    may be a part of a wider projection (``k.stride(0)`` a multiple of 8 elements, heads dense). A page that gets rows belongs to one
    sequence. ``page_table`` ``[B, width]`` int32; entries of a sequence beyond its length are not read. An entry out of the cache, or a
    length beyond the table, sets the device error word (code 6) and writes nothing for that page (on the host: a ``ValueError``)."""
    shape = k.shape
    if not (len(shape) == 3 and v.shape == shape and k.dtype is torch.bfloat16 and v.dtype is torch.bfloat16):
        raise ValueError("keys and values: bf16 [rows, Hkv, D]")
    dev, (rows, Hkv, D) = k.get_device(), shape
    if v.get_device() != dev:
        raise ValueError("keys and values on different devices")
    _no_gradients(k, v)
    P, heads, ps = _check_pages(pages, D, dev)
    if heads != Hkv:
        raise ValueError(f"rows of {Hkv} heads into a cache of {heads}")
    if cu_seqlens is None:
        B, cu = rows, None
    else:
        B, cu = cu_seqlens.numel() - 1, cu_seqlens.data_ptr()
        _need(B >= 0 and cu_seqlens.dtype is torch.int32 and cu_seqlens.dim() == 1 and cu_seqlens.is_contiguous() and cu_seqlens.get_device() == dev,
              "cu_seqlens: contiguous int32 [B + 1]")
    width = _check_table(page_table, seq_lens, B, dev)
    if width * ps >= WIDEST:
        raise ValueError("a table wider than 2^31 tokens")
    if dev < 0:
        return kv8_append_ref(k, v, pages, page_table, seq_lens, cu_seqlens)
    if rows == 0 or B == 0:
        return
    ks, vs = k.stride(), v.stride()
    kr, vr = (ks[0], vs[0]) if rows > 1 else (0, 0)
    kp, vp = k.data_ptr(), v.data_ptr()
    if not (ks[2] == 1 and vs[2] == 1 and (Hkv == 1 or (ks[1] == D and vs[1] == D))):
        raise ValueError("heads of a row have to be dense")
    if (kr | vr) & 7 or (kp | vp) & 15:
        raise ValueError("rows have to start on 16 bytes")
    _launch(dev, "ab2_kv8_append", kp, vp, pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr(), page_table.data_ptr(),
            seq_lens.data_ptr(), cu, B, rows, Hkv, D, ps, width, P, kr, vr)


# ----------------------------------------------------------------------------- attention of single tokens
def kv8_decode_ref(q, pages: QuantPages, page_table, seq_lens, scale: Optional[float] = None) -> torch.Tensor:
    """Plain statement of :func:`kv8_decode` in 64 bits (returned in 64 bits)."""
    B, Hq, D = q.shape
    Hkv, ps = pages.k.shape[1:3]
    scale = D ** -0.5 if scale is None else scale
    out = torch.zeros(B, Hq, D, dtype=torch.float64, device=q.device)
    for b, n in enumerate(seq_lens.tolist()):
        if n <= 0:
            continue
        _need(n <= page_table.shape[1] * ps, f"sequence {b}: {n} tokens are more than its table holds")
        pg = page_table[b, :-(-n // ps)].long()
        _need(bool(((pg >= 0) & (pg < pages.k.shape[0])).all()), f"a page of sequence {b} is not in the cache")
        K, V = ((c.view(torch.uint8)[pg].view(F8).double() * s[pg].double()[:, :, None, None]).transpose(0, 1).reshape(Hkv, -1, D)[:, :n]
                for c, s in ((pages.k, pages.k_scale), (pages.v, pages.v_scale)))
        z = torch.einsum("hgd,htd->hgt", q[b].double().view(Hkv, Hq // Hkv, D), K) * scale
        out[b] = torch.einsum("hgt,htd->hgd", torch.softmax(z, -1), V).reshape(Hq, D)
    return out


@functools.lru_cache(maxsize=256)
def _decode_workspace(dev: int, *sizes: int) -> int:
    with torch.cuda.device(dev):
        return int(_lib.get_lib().ab2_kv8_decode_workspace(*sizes))


_SCRATCH: dict = {}         # (device, stream) -> workspace of the calls on that stream


def _scratch(dev: int, size: int) -> torch.Tensor:
    """A workspace of ``size`` bytes. Calls on one stream run one after the other and share it: a call reads of it only what it has written. A
    captured call gets one of its graph's own."""
    if torch.cuda.is_current_stream_capturing():
        return torch.empty(size, dtype=torch.uint8, device=f"cuda:{dev}")
    key = dev, torch._C._cuda_getCurrentRawStream(dev)
    c = _SCRATCH.get(key)
    if c is None or c.numel() < size:
        c = _SCRATCH[key] = torch.empty(size, dtype=torch.uint8, device=f"cuda:{dev}")
    return c


def kv8_decode(q: torch.Tensor, pages: QuantPages, page_table: torch.Tensor, seq_lens: torch.Tensor, scale: Optional[float] = None,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Attention of one query token per sequence over its first ``seq_lens[b]`` cached tokens: ``softmax(scale q K^T) V``.

    ``q`` ``[B, Hq, D]`` bf16, heads dense, rows a multiple of 8 elements apart (the query part of a wider projection); ``Hq`` a multiple of the cache's
    heads, any number of query heads for each. ``scale`` defaults to ``1 / sqrt(D)``. Returns bf16 ``[B, Hq, D]`` (``out``, contiguous and apart from
    ``q``, where given); a sequence of length 0 gets zeros. Codes behind a sequence's last token may be anything. An entry of the table out of the cache, or a
    length beyond the table, sets the device error word (code 6); the row's result is not to be used (on the host: a ``ValueError``). The workspace
    belongs to the current stream or, in a captured call, to its graph: calls on several streams and graphs do not share one, and calls of several threads on
    one stream go one after the other. At most 8192 sequences."""
    shape = q.shape
    if not (len(shape) == 3 and q.dtype is torch.bfloat16):
        raise ValueError("queries: bf16 [B, Hq, D]")
    _no_gradients(q)
    dev, (B, Hq, D) = q.get_device(), shape
    P, Hkv, ps = _check_pages(pages, D, dev)
    width = _check_table(page_table, seq_lens, B, dev)
    if Hq <= 0 or Hq % Hkv:
        raise ValueError(f"{Hq} query heads over {Hkv} cached ones")
    if B > 8192 or width * ps >= WIDEST:
        raise ValueError("more than 8192 sequences, or a table wider than 2^31 tokens")
    if out is not None:
        _need(out.shape == shape and out.dtype == torch.bfloat16 and out.is_contiguous() and out.get_device() == dev, "out: contiguous bf16 like the queries")
        o, first = out.data_ptr(), q.data_ptr()
        _need(not o & 15, "out has to start on 16 bytes")
        _need(not out.numel() or o + 2 * out.numel() <= first or first + 2 * (1 + sum((n - 1) * st for n, st in zip(shape, q.stride()))) <= o,
              "out overlaps the queries, which other blocks may still read")
    if scale is None:
        scale = D ** -0.5
    if dev < 0:
        o = kv8_decode_ref(q, pages, page_table, seq_lens, scale).to(torch.bfloat16)
        return o if out is None else out.copy_(o)
    if dev != torch._C._cuda_getDevice():
        with torch.cuda.device(dev):                 # whose stream it is that may be captured, and that the workspace belongs to
            return kv8_decode(q, pages, page_table, seq_lens, scale, out)
    if out is None:
        out = torch.empty_like(q, memory_format=torch.contiguous_format)             # half the host time of torch.empty
    if B == 0:
        return out
    st = q.stride()
    row = st[0] if B > 1 else 0
    if not (st[2] == 1 and (Hq == 1 or st[1] == D)):
        raise ValueError("heads of a row have to be dense")
    if row & 7 or q.data_ptr() & 15:
        raise ValueError("rows have to start on 16 bytes")
    ws = _scratch(dev, _decode_workspace(dev, B, Hq, Hkv, D, ps, width))
    _launch(dev, "ab2_kv8_decode", q.data_ptr(), pages.k.data_ptr(), pages.v.data_ptr(), pages.k_scale.data_ptr(), pages.v_scale.data_ptr(),
            page_table.data_ptr(), seq_lens.data_ptr(), out.data_ptr(), ws.data_ptr(), B, Hq, Hkv, D, ps, width, P, scale, row)
    return out


# ----------------------------------------------------------------------------- page copies
def copy_pages_ref(buffers, src, dst, tokens=None) -> None:
    """Plain statement of :func:`copy_pages`."""
    for t, page_dim, token_dim in buffers:
        t = t.view(torch.uint8) if t.dtype == F8 else t
        for i, (s, d) in enumerate(zip(src, dst)):
            a, b = t.select(page_dim, int(s)), t.select(page_dim, int(d))
            if tokens is not None and token_dim is not None:
                a, b = a.narrow(token_dim - 1, 0, int(tokens[i])), b.narrow(token_dim - 1, 0, int(tokens[i]))
            b.copy_(a)


def copy_pages(buffers: Sequence[tuple], src, dst, tokens=None) -> None:
    """Copies pages ``src[i]`` to ``dst[i]`` in every buffer, all in one launch (256 pairs each): requests that fork from a prompt's partial last
    page, or pages that move.

    ``buffers``: up to four ``(tensor, page_dim, token_dim)``. The tensor is contiguous; its dims before ``page_dim`` (layers, keys and values) are copied
    for every page; ``token_dim`` (behind ``page_dim``) counts the tokens of a page, or is None for what belongs to a page as a whole (scales).
    ``src``, ``dst``, ``tokens``: host sequences of ints or integer arrays; ``tokens[i]`` leading tokens of page i are copied, the rest of the
    destination stays as it is (None: whole pages). They are arguments of the launch: a captured call copies the same pages in every replay. A source may stand for several destinations; no page may be a destination twice, or source and
    destination at once."""
    src, dst = _ints(src), _ints(dst)
    n = len(src)
    if len(dst) != n or not 0 < len(buffers) <= 4:
        raise ValueError("one destination for each source, one to four buffers")
    dev, pages, slots = buffers[0][0].get_device(), None, None
    desc = []
    for t, page_dim, token_dim in buffers:
        shape, st, es = t.shape, t.stride(), t.element_size()
        if not (t.get_device() == dev and t.is_contiguous() and t.numel() > 0):
            raise ValueError("buffers: contiguous, on one device")
        if not (0 <= page_dim < len(shape) and (token_dim is None or page_dim < token_dim < len(shape))):
            raise ValueError("no such dims")
        p = shape[page_dim]
        if pages is None:
            pages = p
        elif pages != p:
            raise ValueError("buffers of different numbers of pages")
        whole = st[page_dim] * es
        rows, row, tok = 1, whole, 0
        if token_dim is not None:
            if slots is None:
                slots = shape[token_dim]
            elif slots != shape[token_dim]:
                raise ValueError("buffers of different page sizes")
            if tokens is not None:
                tok = st[token_dim] * es
                row = tok * slots
                rows = whole // row
        if whole >= (1 << 31) - (1 << 15):
            raise ValueError("a page of 2 GB")
        desc += (t.data_ptr(), whole * p, whole, row, t.numel() * es // (whole * p), rows, row, tok, p, 0)
    if n == 0:
        return
    to = set(dst)
    if min(src) < 0 or max(src) >= pages or min(dst) < 0 or max(dst) >= pages:
        raise ValueError(f"pages outside of 0 .. {pages - 1}")
    if len(to) != n:
        raise ValueError("a page is the destination of two copies")
    if not to.isdisjoint(src):
        raise ValueError("a page is source and destination")
    if tokens is not None:
        tokens = _ints(tokens)
        if not (len(tokens) == n and slots is not None and min(tokens) >= 0 and max(tokens) <= slots):
            raise ValueError("tokens: 0 to the page size, one for each pair")
    if dev < 0:
        return copy_pages_ref(buffers, src, dst, tokens)
    pairs = src + dst + (tokens if tokens is not None else [-1] * n)
    _launch(dev, "ab2_copy_pages", struct.pack(f"{len(desc)}q", *desc), len(buffers), struct.pack(f"{3 * n}i", *pairs), n)


def _ints(x) -> list:
    return x.tolist() if hasattr(x, "tolist") else list(x)


_lib.declare("ab2_kv8_append", [_V] * 9 + [_I] * 7 + [_L, _L, _V])
def _decode_kernels(*a) -> int:
    return 1 + (a[13] * a[14] > 4 * 64)          # the join, where the table holds more than the smallest unit's four chunks of 64 tokens


_lib.declare("ab2_kv8_decode", [_V] * 9 + [_I] * 7 + [_F, _L, _V], kernels=_decode_kernels)
_lib.declare("ab2_kv8_decode_workspace", [_I] * 6, _L)
_lib.declare("ab2_copy_pages", [_V, _I, _V, _I, _V], kernels=lambda *a: -(-a[3] // 256))           # pairs travel 256 at a time

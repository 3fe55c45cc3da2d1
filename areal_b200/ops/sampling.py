"""The next token under temperature, top-k, top-p and min-p, drawn from given uniform numbers.

As in :mod:`.functional`, CUDA tensors run the sm_100a kernel and CPU tensors the plain statement. Weights and sums are held in 64 bits in
both: a token next to a border of the nucleus, or of the number drawn, does not depend on the order of a sum.
"""
from __future__ import annotations

from typing import Optional

import torch

from . import lib as _lib
from .cache_ops import _launch, _need, _no_gradients

_V, _I, _L = _lib.c_void_p, _lib.c_int, _lib.c_ll
NO_WEIGHT = -(700 + 2.0 ** -11)          # from here down a token has no weight: e^-700 is next to the smallest number of 64 bits
MAX_VOCAB = 8 * 49152        # the kernel holds a row in the shared memory of eight SMs


def sample_filtered_ref(logits, u, inv_temp, top_k, top_p, min_p, greedy=None):
    """Plain statement of :func:`sample_filtered`, row by row in 64 bits."""
    B, V = logits.shape
    tok = torch.full((B,), -1, dtype=torch.int32, device=logits.device)
    lp = torch.full((B,), float("-inf"), device=logits.device)
    for b in range(B):
        x = logits[b].double()
        x = torch.where(torch.isnan(x), torch.full_like(x, float("-inf")), x)
        order = torch.sort(x, descending=True, stable=True).indices
        top = x[order[0]]
        if top == float("-inf"):
            continue
        it = float(inv_temp[b])
        w = torch.where(x == top, torch.ones_like(x), torch.where((x == float("-inf")) | ((x - top) * it <= NO_WEIGHT), torch.zeros_like(x), torch.exp((x - top) * it)))
        if greedy is not None and int(greedy[b]):
            tok[b], lp[b] = int(order[0]), -torch.log(w.sum())
            continue
        k, p, m = int(top_k[b]), float(top_p[b]), float(min_p[b])
        if 0 < k < V:
            order = order[:k]
        ws = w[order]
        keep = ws > 0
        if p < 1:
            cum = torch.cumsum(ws, 0)
            keep &= cum - ws <= max(p, 0.0) * cum[-1]
        keep &= ws >= min(m, 1.0)
        kept = torch.sort(order[keep]).values
        run = torch.cumsum(w[kept], 0)
        i = min(int(torch.searchsorted(run, float(u[b]) * run[-1], right=True)), len(kept) - 1)
        tok[b], lp[b] = int(kept[i]), torch.log(w[kept[i]] / run[-1])
    return tok, lp


def sample_filtered(logits: torch.Tensor, u: torch.Tensor, inv_temp: torch.Tensor, top_k: torch.Tensor, top_p: torch.Tensor, min_p: torch.Tensor,
                    greedy: Optional[torch.Tensor] = None, out: Optional[tuple] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """One token for each row of ``logits`` ``[B, V]`` fp32, and its log-prob: ``(int32 [B], fp32 [B])`` (``out``, contiguous, where given).

    Row by row, with ``w_i = exp((x_i - max) * inv_temp)`` and the order by falling logit (equal ones: the lowest index first): ``top_k`` keeps the first
    k; ``top_p`` keeps those before which the weights of the order sum to no more than ``top_p`` times the total of what top-k left;
    ``min_p`` keeps ``w_i >= min_p``. The token is the lowest index at which the kept weights, summed by index, pass ``u`` times their
    sum ``W`` (``u`` in [0, 1)); its log-prob is ``ln(w / W)``. A row with ``greedy`` set takes the first of the order, with its log-prob
    over all tokens. ``top_k <= 0`` (or >= V), ``top_p >= 1`` and ``min_p <= 0`` switch a filter off; ``inv_temp`` is positive. Logits of minus
    infinity and NaN have no weight, nor have those more than 700 nats below the largest; infinite ones share all of it. A row in which nothing has weight gives token -1 and minus infinity.

    ``u``, ``inv_temp``, ``top_p``, ``min_p``: fp32 ``[B]``; ``top_k``, ``greedy``: int32 ``[B]``. Rows of logits may lie apart (a slice of a wider
    tensor). The log-prob has no gradient: logits that require one are refused unless gradients are switched off. At most 393216 tokens in the vocabulary on CUDA."""
    shape = logits.shape
    if not (len(shape) == 2 and logits.dtype is torch.float32 and shape[1] > 0 and (logits.stride(1) == 1 or shape[1] == 1)):
        raise ValueError("logits: fp32 [B, V], dense rows")
    _no_gradients(logits, u, inv_temp, top_p, min_p)
    B, V = shape
    dev, one = logits.get_device(), shape[:1]
    for t, d, name in ((u, torch.float32, "u"), (inv_temp, torch.float32, "inv_temp"), (top_p, torch.float32, "top_p"), (min_p, torch.float32, "min_p"),
                       (top_k, torch.int32, "top_k"), (greedy, torch.int32, "greedy")):
        if t is not None and not (t.dtype is d and t.shape == one and t.is_contiguous() and t.get_device() == dev):
            raise ValueError(f"{name}: contiguous {d} [{B}] beside the logits")
    if out is not None:
        _need(out[0].dtype == torch.int32 and out[1].dtype == torch.float32 and all(t.shape == one and t.is_contiguous() and t.get_device() == dev for t in out),
              "out: int32 and fp32, contiguous [B]")
    if dev < 0:
        r = sample_filtered_ref(logits, u, inv_temp, top_k, top_p, min_p, greedy)
        return r if out is None else (out[0].copy_(r[0]), out[1].copy_(r[1]))
    if V > MAX_VOCAB:
        raise ValueError(f"a vocabulary of {V}: at most {MAX_VOCAB}")
    ld = logits.stride(0) if B > 1 else V
    if ld < V:
        raise ValueError("rows of logits overlap")
    if out is None:
        out = torch.empty_like(top_k), torch.empty_like(u)
    _launch(dev, "ab2_sample_filtered", logits.data_ptr(), ld, B, V, u.data_ptr(), inv_temp.data_ptr(), top_k.data_ptr(), top_p.data_ptr(),
            min_p.data_ptr(), None if greedy is None else greedy.data_ptr(), out[0].data_ptr(), out[1].data_ptr())
    return out


_lib.declare("ab2_sample_filtered", [_V, _L, _I, _I] + [_V] * 9)

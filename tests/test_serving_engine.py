"""The rollout engine on its 8-bit cache and with sampling filters on the device."""
import asyncio

import numpy as np
import pytest
import torch

from areal_b200.api.cli_args import GenerationHyperparameters, InferenceEngineConfig, NativeInferConfig
from areal_b200.api.io_struct import ModelRequest
from areal_b200.engine import infer_engine as IE
from areal_b200.engine.infer_engine import NativeInferenceEngine, PagedKVCache
from areal_b200.engine.remote_backends import _sampling
from areal_b200.engine.server import gconfig_from_sampling_params
from areal_b200.models.config import preset
from areal_b200.models.decoder import build_model
from areal_b200.ops import lib as oplib


def _engine(model, device="cuda", **kw):
    ic = NativeInferConfig(max_running_requests=16, page_size=16, context_length=512, **kw)
    ic.num_pages = 400
    return NativeInferenceEngine(InferenceEngineConfig(), ic, model=model).initialize(device=device, start_executor=False)


def _run(e, prompts, g):
    async def go():
        return await asyncio.gather(*[e.agenerate(ModelRequest(rid=f"r{i}", input_ids=p, gconfig=g)) for i, p in enumerate(prompts)])
    return asyncio.run(go())


# ----------------------------------------------------------------------------- on the host
def test_numbers_of_requests_are_spread_and_belong_to_seed_and_position():
    u = np.array([[IE._uniform01(s, n) for n in range(200)] for s in range(50)])
    assert u.min() >= 0 and u.max() < 1 and abs(u.mean() - 0.5) < 0.02 and abs(np.corrcoef(u[:, :-1].ravel(), u[:, 1:].ravel())[0, 1]) < 0.05
    assert np.unique(u).size > 0.99 * u.size and IE._uniform01(7, 3) == IE._uniform01(7, 3)
    assert np.all(u * (1 << 24) == np.floor(u * (1 << 24)))                     # exact in 32 bits


def test_min_p_travels_with_a_request_and_filters_on_the_host():
    g = GenerationHyperparameters(min_p=0.2)
    assert _sampling(g, 5, 0)["min_p"] == 0.2 and "min_p" not in _sampling(GenerationHyperparameters(), 5, 0)
    assert gconfig_from_sampling_params({"min_p": 0.2}).min_p == 0.2 and gconfig_from_sampling_params({}).min_p == 0.0
    model = build_model(preset("tiny-qwen3"), dtype=torch.float32, device="cpu", seed=3)
    e = _engine(model, "cpu")
    s = IE._Seq(rid="a", tokens=[1], prompt_len=1, max_new=1, min_new=0, temperature=1.0, greedy=False, stop_ids=set(), ignore_eos=True, seed=1, min_p=0.5)
    logits = torch.tensor([3.0, 2.9, 2.0, 0.0])
    for n in range(40):
        s.tokens = [1] * (n + 1)
        tok, lp = e._sample_cpu(logits, s)
        assert tok in (0, 1) and abs(lp - float(torch.log_softmax(logits[:2], -1)[tok])) < 1e-6
    e.destroy()


def test_tokens_that_tie_with_the_last_of_a_top_k():
    """The host keeps them all, the device the lowest indices up to k: log-probs differ by the tokens more, and agree where nothing ties."""
    model = build_model(preset("tiny-qwen3"), dtype=torch.float32, device="cpu", seed=3)
    e = _engine(model, "cpu")
    s = IE._Seq(rid="a", tokens=[1], prompt_len=1, max_new=1, min_new=0, temperature=1.0, greedy=False, stop_ids=set(), ignore_eos=True, seed=1, top_k=3)
    for logits, host, device in ((torch.tensor([1.0, 2.0, 3.0, 2.0, 2.0, -1.0]), {1, 2, 3, 4}, {1, 2, 3}), (torch.tensor([1.0, 2.5, 3.0, 2.0, 1.5, -1.0]), {1, 2, 3}, {1, 2, 3})):
        seen = {}
        for n in range(200):
            s.tokens = [1] * (n + 1)
            tok, lp = e._sample_cpu(logits, s)
            seen[tok] = lp
        assert set(seen) == host
        u = (torch.arange(200) + 0.5) / 200
        one = torch.ones(200)
        tok, lp = IE.OS.sample_filtered(logits.expand(200, 6).contiguous(), u, one, (one * 3).int(), one, one * 0)
        assert set(tok.tolist()) == device
        for kept, got in ((host, seen), (device, dict(zip(tok.tolist(), lp.tolist())))):
            want = torch.log_softmax(logits[sorted(kept)], 0)
            assert max(abs(got[t] - float(want[i])) for i, t in enumerate(sorted(kept))) < 1e-6
    e.destroy()


def test_unknown_sampling_places_are_refused():
    with pytest.raises(ValueError):
        NativeInferenceEngine(InferenceEngineConfig(), NativeInferConfig(filtered_sampling="gpu"), model_config=preset("tiny-qwen3"))


def test_an_eight_bit_cache_that_cannot_be_had_is_said(monkeypatch):
    said = []
    monkeypatch.setattr(IE.logger, "warning", lambda text, *a: said.append(text % a))
    model = build_model(preset("tiny-qwen3"), dtype=torch.float32, device="cpu", seed=3)
    for kind, n in (("bfloat16", 0), ("fp8_e4m3", 1)):
        _engine(model, "cpu", kv_cache_dtype=kind).destroy()
        assert len([x for x in said if "kv_cache_dtype" in x]) == n


def test_an_eight_bit_pool_holds_nearly_twice_the_pages():
    cfg = preset("qwen3-8b")
    a, b = PagedKVCache.bytes_per_page(cfg, 64), PagedKVCache.bytes_per_page(cfg, 64, True)
    assert a == 36 * 2 * 8 * 64 * 128 * 2 and b == 36 * 2 * 8 * (64 * 128 + 4)
    small = preset("tiny-qwen3")
    c = PagedKVCache(small, 6, 16, "cpu", torch.bfloat16, eight_bit=True)
    assert c.data.numel() + 4 * c.scales.numel() == 6 * PagedKVCache.bytes_per_page(small, 16, True)
    p = c.layer(1)
    p.k.view(torch.uint8)[3] = 5
    c.scales[1, 0, 3] = 2.0
    c.copy([3], [4], [10])
    assert torch.all(c.data[1, 0, 4, :, :10] == 5) and torch.all(c.data[1, 0, 4, :, 10:] == 0) and torch.all(c.scales[1, 0, 4] == 2)
    assert torch.all(c.data[0] == 0) and p.k.data_ptr() == c.data[1, 0].data_ptr()


# ----------------------------------------------------------------------------- on the GPU
def _recomputed(model, r):
    """Log-softmax of every generated position by the training forward."""
    seq = r.input_tokens + r.output_tokens
    T = len(seq)
    Tp = (T + 127) // 128 * 128
    ids = torch.tensor(seq + [0] * (Tp - T), dtype=torch.int32, device="cuda")
    cu = torch.tensor([0, T] + ([Tp] if Tp > T else []), dtype=torch.int32, device="cuda")
    with torch.no_grad():
        h = model(ids, cu)
        return model.logits(h[len(r.input_tokens) - 1:T - 1].contiguous()).float().cpu()


@pytest.mark.gpu
@pytest.mark.parametrize("graph", [True, False])
@pytest.mark.parametrize("pausable", [False, True])
def test_rollout_on_the_eight_bit_cache(graph, pausable):
    """Prompts and answers over several pages; log-probs follow the training forward as far as codes of four significant bits allow on
    this small model (the 16-bit cache is held to 0.1 there)."""
    model = build_model(preset("tiny-qwen3"), dtype=torch.bfloat16, device="cuda", seed=13)
    e = _engine(model, kv_cache_dtype="float8_e4m3", use_cuda_graph=graph, pausable_kv_cache=pausable)
    assert e.cache.eight_bit and e.cache.data.dtype == torch.uint8
    prompts = [list(range(3 + i, 20 + 7 * i)) for i in range(12)]
    rs = _run(e, prompts, GenerationHyperparameters(max_new_tokens=40, max_tokens=400, temperature=1.0, ignore_eos=True))
    again = _run(e, prompts[:3], GenerationHyperparameters(max_new_tokens=20, max_tokens=400, greedy=True, ignore_eos=True))
    assert oplib.kernel_error() == 0
    e.offload()
    e.onload()
    after = _run(e, prompts[:3], GenerationHyperparameters(max_new_tokens=20, max_tokens=400, greedy=True, ignore_eos=True))
    graphs = len(e._graphs)                              # (gone with the engine)
    e.destroy()
    assert [r.output_tokens for r in after] == [r.output_tokens for r in again]
    off = []
    for r in rs:
        assert len(r.output_tokens) == 40
        lp = torch.log_softmax(_recomputed(model, r), -1)
        off.append((lp.gather(1, torch.tensor(r.output_tokens)[:, None])[:, 0] - torch.tensor(r.output_logprobs)).abs())
    assert float(torch.cat(off).mean()) < 0.1, float(torch.cat(off).mean())
    assert (graphs > 0) == graph


@pytest.mark.gpu
@pytest.mark.parametrize("prompt_len", [64, 75])
@pytest.mark.parametrize("kv", ["bfloat16", "fp8_e4m3"])
def test_forks_of_a_prompt_continue_as_requests_of_their_own(prompt_len, kv):
    model = build_model(preset("tiny-qwen3"), dtype=torch.bfloat16, device="cuda", seed=11)
    g = GenerationHyperparameters(max_new_tokens=40, max_tokens=400, greedy=True, ignore_eos=True)
    prompts = [list(range(7, 7 + prompt_len))] * 6 + [list(range(90, 90 + prompt_len - 3))] * 2
    alone = _engine(model, kv_cache_dtype=kv)
    want = _run(alone, prompts, g)
    alone.destroy()
    e = _engine(model, kv_cache_dtype=kv, enable_prefix_sharing=True)
    got = _run(e, prompts, g)
    assert e.stats["prefix_hits"] == 6
    e.destroy()
    assert oplib.kernel_error() == 0
    assert [r.output_tokens for r in got] == [r.output_tokens for r in want]


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(top_k=1), dict(top_k=5), dict(top_p=0.6, temperature=0.8), dict(min_p=0.3), dict(top_k=20, top_p=0.9, min_p=0.05)])
def test_filtered_sampling_on_the_device(kw):
    """Every token lies within its request's filters, as the training forward sees them (bf16 noise moves a border by a little), its log-prob is
    the one under the filtered distribution, and the same requests draw the same tokens again."""
    model = build_model(preset("tiny-qwen3"), dtype=torch.bfloat16, device="cuda", seed=13)
    e = _engine(model, filtered_sampling="device")
    prompts = [list(range(3 + i, 30 + 2 * i)) for i in range(9)]
    g = GenerationHyperparameters(**{"max_new_tokens": 24, "max_tokens": 400, "ignore_eos": True, **kw})
    rs, again = _run(e, prompts, g), _run(e, prompts, g)
    mixed = _run(e, prompts[:2], GenerationHyperparameters(max_new_tokens=24, max_tokens=400, ignore_eos=True))
    e.destroy()
    assert oplib.kernel_error() == 0
    assert [r.output_tokens for r in rs] == [r.output_tokens for r in again] and all(len(r.output_tokens) == 24 for r in mixed)
    for r in rs:
        z = _recomputed(model, r) / g.temperature
        p = torch.softmax(z, -1)
        for t, tok in enumerate(r.output_tokens):
            share = p[t] / p[t].max()
            assert g.top_k >= 10 ** 7 or int((z[t] > z[t, tok] + 0.1).sum()) < g.top_k
            assert float(share[tok]) >= g.min_p * 0.85
            assert float(p[t][z[t] > z[t, tok] + 0.1].sum()) <= g.top_p + 0.05
            assert r.output_logprobs[t] <= 1e-6 and r.output_logprobs[t] >= float(torch.log(p[t, tok])) - 0.1
        if g.top_k == 1:
            assert max(abs(x) for x in r.output_logprobs) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("place", ["host", "device"])
def test_a_request_without_a_number_to_draw_by_is_an_error_and_no_token(place):
    model = build_model(preset("tiny-qwen3"), dtype=torch.bfloat16, device="cuda", seed=5)
    e = _engine(model, filtered_sampling=place)
    s = IE._Seq(rid="a", tokens=[1], prompt_len=1, max_new=1, min_new=0, temperature=1.0, greedy=False, stop_ids=set(), ignore_eos=True, seed=1, top_p=0.9)
    with torch.cuda.stream(e.stream):
        logits = torch.randn(2, 1024, device="cuda")
        assert min(e._sample_cuda(logits, [s, s])[0]) >= 0
        logits[1] = float("nan")
        with pytest.raises(RuntimeError):
            e._sample_cuda(logits, [s, s])
    e.destroy()


@pytest.mark.gpu
def test_device_and_host_filters_leave_the_same_distribution():
    """Next-token counts of many seeds on one prompt, both places: each token's share differs by less than five standard deviations."""
    model = build_model(preset("tiny-qwen3"), dtype=torch.bfloat16, device="cuda", seed=5)
    counts = []
    for place in ("host", "device"):
        e = _engine(model, filtered_sampling=place)
        async def go():
            return await asyncio.gather(*[e.agenerate(ModelRequest(rid=f"r{i}", input_ids=list(range(5, 40)), gconfig=GenerationHyperparameters(
                max_new_tokens=2, max_tokens=400, top_k=8, top_p=0.95, temperature=0.7, ignore_eos=True, seed=i))) for i in range(600)])
        rs = asyncio.run(go())
        e.destroy()
        counts.append(np.bincount([r.output_tokens[0] for r in rs], minlength=1024))
    a, b = counts
    assert set(np.nonzero(a)[0]) <= set(np.nonzero(a + b)[0]) and np.count_nonzero(a + b) <= 8
    p = (a + b) / 1200
    assert np.all(np.abs(a - b) <= 5 * np.sqrt(2 * 600 * p * (1 - p)) + 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_filters_on_the_device_serve_a_mixer_stack(monkeypatch, dtype):
    """Requests of a mixer stack with filters, without and greedy, side by side: every draw is the statement's on the step's own logits, with the numbers that
    belong to the requests' seeds and positions, and the tokens are those drawn; top-k 1 and greedy agree."""
    model = build_model(preset("tiny-kagolix"), dtype=dtype, device="cuda", seed=7)
    e = _engine(model, filtered_sampling="device")
    calls, inner = [], IE.OS.sample_filtered

    def watched(*a, **kw):
        calls.append([x.clone() for x in a])
        r = inner(*a, **kw)
        calls[-1].append([x.clone() for x in r])
        return r
    monkeypatch.setattr(IE.OS, "sample_filtered", watched)
    kinds = [dict(top_k=5), dict(top_p=0.8, temperature=0.7), {}, dict(greedy=True), dict(min_p=0.1, top_k=40), dict(top_k=1), dict(top_p=0.95, top_k=9, seed=77)]
    prompts = [list(range(3, 40))] * len(kinds)

    async def go():
        return await asyncio.gather(*[e.agenerate(ModelRequest(rid=f"r{i}", input_ids=p, gconfig=GenerationHyperparameters(
            **{"max_new_tokens": 20, "max_tokens": 400, "ignore_eos": True, **k}))) for i, (p, k) in enumerate(zip(prompts, kinds))])
    rs = asyncio.run(go())
    e.destroy()
    assert oplib.kernel_error() == 0
    assert rs[3].output_tokens == rs[5].output_tokens and max(abs(x) for x in rs[5].output_logprobs) == 0
    assert sum(c[0].shape[0] for c in calls) >= 20 * sum(bool(k) and k != dict(greedy=True) for k in kinds)
    drawn = set()
    for *a, (tok, lp) in calls:
        want, wlp = IE.OS.sample_filtered_ref(*(x.cpu() for x in a))
        assert torch.equal(tok.cpu(), want) and torch.all((lp.cpu().double() - wlp.double()).abs() <= 2.0 ** -23 * wlp.abs().double() + 1e-9)
        drawn |= {(float(u), int(t), float(p)) for u, t, p in zip(a[1].cpu(), tok.cpu(), lp.cpu())}
    for n, (tok, lp) in enumerate(zip(rs[6].output_tokens, rs[6].output_logprobs)):
        assert (IE._uniform01(77, len(prompts[6]) + n), tok, lp) in drawn


@pytest.mark.gpu
def test_a_cache_the_kernels_do_not_take_is_refused():
    model = build_model(preset("tiny-qwen3"), dtype=torch.bfloat16, device="cuda", seed=5)
    with pytest.raises(ValueError):
        NativeInferenceEngine(InferenceEngineConfig(), NativeInferConfig(kv_cache_dtype="fp8", page_size=48, context_length=480, num_pages=20),
                              model=model).initialize(device="cuda", start_executor=False)

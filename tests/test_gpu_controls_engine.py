"""Logit controls and adapters through the engine and the speculative decoder: token streams
checked token by token against the 64-bit restatement, in one shared batch."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle.controls import control_row

from .test_gpu_model import device_model, tiny_model_cfg

pytestmark = pytest.mark.gpu

DEV = "cuda"


@pytest.fixture(autouse=True)
def no_device_error():
    from microserve_b200 import _lib

    yield
    assert _lib.device_error() == 0


def _engine(golden, gamma: int = 0, target=None, blocks: int = 128, **sched):
    from microserve_b200.config import (CacheConfig, EngineConfig, SchedulerConfig,
                                        SpeculativeConfig)
    from microserve_b200.engine import LLMEngine

    target = target if target is not None else device_model(golden, "target")
    cfg = EngineConfig(model=tiny_model_cfg(golden, "target"),
                       cache=CacheConfig(block_size=8, num_blocks=blocks),
                       scheduler=SchedulerConfig(max_batch_size=8, **sched),
                       speculative=SpeculativeConfig(enabled=gamma > 0, gamma=max(gamma, 1)))
    return LLMEngine(target, cfg, draft_model=device_model(golden, "draft") if gamma else None)


def _logits(model, tokens: list[int]) -> np.ndarray:
    """The last row's logits of one sequence, computed alone."""
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig

    cache = PagedKVCache(model.cfg, CacheConfig(8, 32, model.cfg.dtype), DEV)
    batch = build_paged_batch(cache, [0], [tokens], [0])
    return model.forward_paged(batch, cache)[-1].cpu().numpy()


def assert_greedy(model, prompt: list[int], cfg, got: list[int]) -> None:
    """Every token of ``got`` is the best one after the tokens before it, with the controls
    applied by the 64-bit restatement to logits computed alone.  Those agree with the
    engine's to 1e-4 relative + 1e-5 (the float32 models' bound), so a token may be behind the
    best by twice that, times a repetition penalty below 2."""
    V = model.cfg.vocab_size
    assert len(got) == cfg.max_new_tokens
    for i, token in enumerate(got):
        out = got[:i]
        x = _logits(model, prompt + out)
        seen = np.zeros(V, bool)
        seen[prompt + out] = True
        allowed = cfg.allowed_tokens(out) if cfg.allowed_tokens else None
        y, _ = control_row(x, np.bincount(out, minlength=V), seen, [],
                           (cfg.repetition_penalty, cfg.presence_penalty, cfg.frequency_penalty),
                           cfg.logit_bias or {}, allowed)
        assert y[token] >= y.max() - 4 * (1e-4 * np.abs(x).max() + 1e-5), (i, token, int(y.argmax()))


def _settings(V: int) -> list:
    from microserve_b200.config import SamplingConfig

    def even_after_odd(out: list[int]) -> np.ndarray | None:
        if len(out) % 3 == 2:
            return None
        ok = np.zeros(V, bool)
        ok[len(out) % 2 :: 2] = True
        return ok

    return [
        SamplingConfig(temperature=0.0, max_new_tokens=24, repetition_penalty=1.7),
        SamplingConfig(temperature=0.0, max_new_tokens=24, frequency_penalty=0.9, presence_penalty=0.6),
        SamplingConfig(temperature=0.0, max_new_tokens=24, logit_bias={3: 4.0, 7: -float("inf"), 11: 2.5}),
        SamplingConfig(temperature=0.0, max_new_tokens=24),
        SamplingConfig(temperature=0.0, max_new_tokens=24, repetition_penalty=0.8,
                       frequency_penalty=1.5, logit_bias={5: 1.0, 0: -2.0}),
        SamplingConfig(temperature=0.0, max_new_tokens=24, allowed_tokens=even_after_odd,
                       presence_penalty=1.0),
    ]


def _prompts(golden, n: int) -> list[list[int]]:
    rng = np.random.default_rng(8)
    V = int(golden["target_cfg"][0])
    return [rng.integers(0, V, 5 + 3 * i).tolist() for i in range(n)]


@pytest.mark.parametrize("gamma", [0, 1, 4])
def test_controlled_streams_match_greedy_by_hand(golden, gamma: int) -> None:
    """Every kind of control in one batch, beside a request without any; without speculation,
    and in chained speculative rounds (no request restricts its tokens there)."""
    eng = _engine(golden, gamma)
    V = eng.model.cfg.vocab_size
    settings = [s for s in _settings(V) if gamma == 0 or s.allowed_tokens is None]
    prompts = _prompts(golden, len(settings))
    reqs = [eng.add_request(p, s) for p, s in zip(prompts, settings)]
    got = {o.request_id: o.output_ids for o in eng.run()}
    for r, p, s in zip(reqs, prompts, settings):
        assert_greedy(eng.model, p, s, got[r.request_id])
    if gamma:
        assert eng.stats.num_spec_rounds > 0 and eng.spec.lookahead_hits > 0
    assert not eng.controls._slot and not eng.controls._counted  # all given back


def test_restricted_requests_take_ordinary_passes_beside_speculation(golden) -> None:
    eng = _engine(golden, 3)
    V = eng.model.cfg.vocab_size
    settings = _settings(V)
    prompts = _prompts(golden, len(settings))
    settings[-1].max_new_tokens = 6  # then the others speculate
    reqs = [eng.add_request(p, s) for p, s in zip(prompts, settings)]
    got = {o.request_id: o.output_ids for o in eng.run()}
    for r, p, s in zip(reqs, prompts, settings):
        assert_greedy(eng.model, p, s, got[r.request_id])
    assert eng.stats.num_spec_rounds > 0


@pytest.mark.parametrize("gamma", [0, 3])
def test_controls_survive_preemption_and_chunked_prefill(golden, gamma: int) -> None:
    eng = _engine(golden, gamma, blocks=12, prefill_chunk=4)
    settings = [s for s in _settings(eng.model.cfg.vocab_size) if s.allowed_tokens is None]
    prompts = _prompts(golden, len(settings))
    reqs = [eng.add_request(p, s) for p, s in zip(prompts, settings)]
    got = {o.request_id: o.output_ids for o in eng.run()}
    for r, p, s in zip(reqs, prompts, settings):
        assert_greedy(eng.model, p, s, got[r.request_id])
    assert eng.stats.num_preemptions > 0


def test_a_caller_that_changes_the_tokens_gets_them_counted_afresh(golden) -> None:
    """The decoder used directly: the caller keeps one token of each round and appends another."""
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, SamplingConfig
    from microserve_b200.scheduler import Request
    from microserve_b200.speculative import SpeculativeDecoder

    target, draft = device_model(golden, "target"), device_model(golden, "draft")
    dec = SpeculativeDecoder(target, draft, CacheConfig(8, 64), gamma=3)
    dec.lookahead = False  # chained rounds need every token kept
    cache = PagedKVCache(target.cfg, CacheConfig(8, 64, target.cfg.dtype), DEV)
    cfg = SamplingConfig(temperature=0.0, max_new_tokens=500, repetition_penalty=1.4, frequency_penalty=0.7)
    req = Request(0, _prompts(golden, 1)[0], cfg)
    gens = {0: torch.Generator().manual_seed(0)}
    V = target.cfg.vocab_size
    for step in range(6):
        new = dec.step([req], cache, gens)[0]
        x = _logits(target, req.all_ids)
        seen = np.zeros(V, bool)
        seen[req.all_ids] = True
        y, _ = control_row(x, np.bincount(req.output_ids, minlength=V), seen, [], (1.4, 0.0, 0.7), {}, None)
        assert y[new[0]] >= y.max() - 4 * (1e-4 * np.abs(x).max() + 1e-5)
        req.output_ids.append(new[0])
        if step % 2 and len(new) > 1:
            req.output_ids.extend(new[1:])
        keep = min(cache.num_tokens(0), req.num_tokens - 1)
        cache.truncate(0, keep)
        dec.draft_cache.truncate(0, min(dec.draft_cache.num_tokens(0), keep))
        req.num_computed = keep
    seen = np.zeros(V, bool)
    dec.controls.prepare([req])
    slot = dec.controls._slot[0]
    assert np.array_equal(dec.controls.counts.counts[slot].cpu().numpy(),
                          np.bincount(req.output_ids, minlength=V))


def test_an_id_used_again_starts_without_counts(golden) -> None:
    """The decoder used directly: a freed id's next request has the length that was counted."""
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, SamplingConfig
    from microserve_b200.scheduler import Request
    from microserve_b200.speculative import SpeculativeDecoder

    target, draft = device_model(golden, "target"), device_model(golden, "draft")
    dec = SpeculativeDecoder(target, draft, CacheConfig(8, 64), gamma=2)
    cache = PagedKVCache(target.cfg, CacheConfig(8, 64, target.cfg.dtype), DEV)
    cfg = SamplingConfig(temperature=0.0, max_new_tokens=500, repetition_penalty=1.4)
    first = Request(7, _prompts(golden, 1)[0], cfg)
    new = dec.step([first], cache, {7: torch.Generator().manual_seed(0)})[0]
    cache.free(7)
    dec.free(7)
    second = Request(7, [3] * (first.num_tokens + len(new)), cfg)
    dec.controls.prepare([second])
    slot = dec.controls._slot[7]
    assert not dec.controls.counts.counts[slot].any()
    seen = dec.controls.counts.seen[slot].cpu().tolist()
    assert seen[0] == 1 << 3 and not any(seen[1:])


def test_sampled_speculation_follows_the_controlled_distribution(golden) -> None:
    """Chi-square of the first token of 4096 requests against the controlled softmax: the accept
    rule has to use controlled draft and target rows alike."""
    from microserve_b200.config import SamplingConfig

    eng = _engine(golden, 2, blocks=4096)
    eng.config.scheduler.max_batch_size = 512
    V = eng.model.cfg.vocab_size
    prompt = _prompts(golden, 1)[0]
    bias = {i: 1.5 for i in range(0, V, 4)}
    n = 1024
    for i in range(n):
        eng.add_request(prompt, SamplingConfig(temperature=1.0, max_new_tokens=2, seed=1000 + i,
                                               repetition_penalty=1.5, logit_bias=bias))
    outs = eng.run()
    # the second token comes from a speculative round; condition on the most common first one
    first = np.array([o.output_ids[0] for o in outs])
    common = int(np.bincount(first).argmax())
    second = np.array([o.output_ids[1] for o in outs if o.output_ids[0] == common])
    x = _logits(eng.model, prompt + [common])
    seen = np.zeros(V, bool)
    seen[prompt + [common]] = True
    y, _ = control_row(x, np.bincount([common], minlength=V), seen, [], (1.5, 0.0, 0.0), bias, None)
    p = np.exp(y - y.max())
    p /= p.sum()
    order = np.argsort(-p)
    # pool tokens so that each cell expects at least 5
    cells, mass, members = [], 0.0, []
    for v in order:
        members.append(v)
        mass += p[v]
        if mass * len(second) >= 5:
            cells.append(members)
            mass, members = 0.0, []
    cells[-1] += members
    exp = np.array([p[c].sum() for c in cells]) * len(second)
    got = np.array([np.isin(second, c).sum() for c in cells])
    chi = ((got - exp) ** 2 / exp).sum()
    df = len(cells) - 1
    assert len(cells) >= 2 and chi < df + 5 * np.sqrt(2 * df) + 10  # mean df, sd sqrt(2 df)


def test_engine_refusals(golden) -> None:
    from microserve_b200.config import SamplingConfig

    eng = _engine(golden, 2)
    V = eng.model.cfg.vocab_size
    for bad in (dict(repetition_penalty=0.0), dict(repetition_penalty=-1.0),
                dict(repetition_penalty=float("inf")), dict(presence_penalty=float("nan")),
                dict(frequency_penalty=float("inf")), dict(logit_bias={V: 1.0}),
                dict(logit_bias={-1: 1.0}), dict(logit_bias={1: float("nan")}),
                dict(logit_bias={1: float("inf")}), dict(logit_bias={1.5: 1.0})):
        with pytest.raises(ValueError):
            eng.add_request([1, 2], SamplingConfig(**bad))
    with pytest.raises(ValueError, match="adapter"):
        eng.add_request([1, 2], adapter="nobody")
    assert not eng.has_unfinished
    for fn in (lambda out: np.zeros(V, bool), lambda out: np.ones(V + 1, bool),
               lambda out: np.ones(V)):
        eng.reset()
        r = eng.add_request([1, 2], SamplingConfig(allowed_tokens=fn))
        with pytest.raises(ValueError, match="allowed_tokens"):
            eng.step()
        assert r.num_computed == 0 and eng.cache.num_tokens(r.request_id) == 0
    from microserve_b200.scheduler import Request

    spec = eng.spec
    with pytest.raises(ValueError, match="speculative"):
        spec.step([Request(0, [1], SamplingConfig(allowed_tokens=lambda o: None))], eng.cache,
                  {0: torch.Generator()})
    with pytest.raises(ValueError, match="adapter"):
        spec.step([Request(0, [1], SamplingConfig(), adapter="x")], eng.cache, {0: torch.Generator()})


# ---- adapters --------------------------------------------------------------------------


def adapter_state(cfg, rank: int, seed: int, parts: tuple[str, ...], size: float = 1.0) -> dict[str, torch.Tensor]:
    g = torch.Generator().manual_seed(seed)
    d, ff = cfg.d_model, cfg.ffn_hidden
    q, kv = cfg.n_heads * cfg.d_head, cfg.kv_heads * cfg.d_head
    shape = {"attn.q_proj": (d, q), "attn.k_proj": (d, kv), "attn.v_proj": (d, kv), "attn.o_proj": (q, d),
             "ffn.gate_proj": (d, ff), "ffn.up_proj": (d, ff), "ffn.down_proj": (ff, d)}
    out = {}
    for i in range(cfg.n_layers):
        for p in parts:
            k, n = shape[p]
            out[f"blocks.{i}.{p}.lora_A.weight"] = torch.randn(rank, k, generator=g) * k ** -0.5
            out[f"blocks.{i}.{p}.lora_B.weight"] = torch.randn(n, rank, generator=g) * (size * rank ** -0.5 * 0.1)
    return out


def merged(model, adapter: dict[str, torch.Tensor], scale: float):
    """A model with the adapter's product added into its weights."""
    from microserve_b200.model import Transformer

    state = {k: v.clone() for k, v in model.state_dict().items()}
    for key in adapter:
        if key.endswith("lora_A.weight"):
            stem = key[: -len(".lora_A.weight")]
            state[stem + ".weight"] += scale * (adapter[stem + ".lora_B.weight"] @ adapter[key])
    return Transformer.from_state_dict(model.cfg, state, DEV)


ALL = ("attn.q_proj", "attn.k_proj", "attn.v_proj", "attn.o_proj", "ffn.gate_proj", "ffn.up_proj", "ffn.down_proj")


def test_adapters_in_one_batch_match_merged_models(golden) -> None:
    """float32: requests with three adapters and without one in one batch, prompts and single
    tokens alike, give the logits of models with the adapters merged in (1e-4, as the models'
    other logits) and, in the engine with and without speculation, their greedy streams."""
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, SamplingConfig
    from microserve_b200.lora import LoraAdapters

    model = device_model(golden, "target")
    ads = LoraAdapters(model, rank_capacity=4)
    states = {"a": adapter_state(model.cfg, 3, 1, ALL), "b": adapter_state(model.cfg, 8, 2, ("attn.q_proj", "attn.v_proj")),
              "c": adapter_state(model.cfg, 5, 3, ("attn.o_proj", "ffn.gate_proj", "ffn.down_proj"))}
    for name, st in states.items():
        ads.load(name, st, alpha=2.0 * st[next(iter(st))].shape[0])
    who = ["a", None, "b", "c", "a", None]
    models = {None: model, **{n: merged(model, st, 2.0) for n, st in states.items()}}
    prompts = _prompts(golden, len(who))
    cache = PagedKVCache(model.cfg, CacheConfig(8, 64, model.cfg.dtype), DEV)
    batch = build_paged_batch(cache, list(range(6)), prompts, [0] * 6)
    got = model.forward_paged(batch, cache, lora=ads.plan(who, [len(p) for p in prompts]))
    rows = np.cumsum([len(p) for p in prompts]) - 1
    for i, n in enumerate(who):
        want = _logits(models[n], prompts[i])
        np.testing.assert_allclose(got[rows[i]].cpu().numpy(), want, rtol=1e-4, atol=1e-4)
    cfg = SamplingConfig(temperature=0.0, max_new_tokens=20)
    for gamma in (0, 3):
        eng = _engine(golden, gamma, target=model)
        reqs = [eng.add_request(p, cfg, adapter=n) for p, n in zip(prompts, who)]
        with pytest.raises(ValueError, match="held"):
            ads.unload("a")
        outs = {o.request_id: o.output_ids for o in eng.run()}
        for r, p, n in zip(reqs, prompts, who):
            assert_greedy(models[n], p, cfg, outs[r.request_id])
        assert ads._users == {"a": 0, "b": 0, "c": 0}
    # unloading frees its part; the others keep working, and the gap is used again
    ads.unload("b")
    ads.load("d", states["b"], alpha=16.0)
    got = model.forward_paged(*_again(model, prompts[2]), lora=ads.plan(["d"], [len(prompts[2])]))
    np.testing.assert_allclose(got[-1].cpu().numpy(), _logits(models["b"], prompts[2]), rtol=1e-4, atol=1e-4)


def _again(model, tokens):
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig

    cache = PagedKVCache(model.cfg, CacheConfig(8, 32, model.cfg.dtype), DEV)
    return build_paged_batch(cache, [0], [tokens], [0]), cache


def test_adapters_on_the_tensor_core_path() -> None:
    """bf16: tokens without an adapter agree with the shared weights, the others with a merged
    model, to the bf16 models' 2e-2 of the row's scale."""
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, ModelConfig
    from microserve_b200.lora import LoraAdapters
    from microserve_b200.model import Transformer

    from .test_gpu_model import assert_bf16_close

    cfg = ModelConfig(vocab_size=512, n_layers=2, d_model=512, n_heads=8, n_kv_heads=2, d_ff=1024,
                      max_seq_len=512, dtype="bfloat16")
    model = Transformer(cfg, DEV, seed=3)
    ads = LoraAdapters(model)
    states = {"a": adapter_state(cfg, 16, 1, ALL), "b": adapter_state(cfg, 40, 2, ALL)}
    for n, st in states.items():
        ads.load(n, st)
    who, lens = ["a", None, "b", None], [37, 64, 130, 1]
    rng = np.random.default_rng(0)
    prompts = [rng.integers(0, 512, n).tolist() for n in lens]

    def run(m, lora=None):
        cache = PagedKVCache(cfg, CacheConfig(16, 64, "bfloat16"), DEV)
        return m.forward_paged(build_paged_batch(cache, list(range(4)), prompts, [0] * 4), cache, lora=lora)

    plain = run(model)
    got = run(model, ads.plan(who, lens))
    start = np.cumsum([0] + lens)
    mm = {n: run(merged(model, st, 1.0)) for n, st in states.items()}
    for i, n in enumerate(who):
        rows = slice(start[i], start[i + 1])
        want = plain if n is None else mm[n]
        assert_bf16_close(got[rows].cpu().numpy(), want[rows].cpu().numpy())
        if n is not None:  # and the adapter does something
            assert (got[rows] - plain[rows]).abs().max() > 0.05


def test_an_array_of_a_without_b_is_refused(golden) -> None:
    import ctypes

    from microserve_b200 import _lib
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig
    from microserve_b200.lora import LoraAdapters

    model = device_model(golden, "target")
    ads = LoraAdapters(model)
    ads.load("a", adapter_state(model.cfg, 4, 1, ALL))
    cache = PagedKVCache(model.cfg, CacheConfig(8, 64, model.cfg.dtype), DEV)
    batch = build_paged_batch(cache, [0], [_prompts(golden, 1)[0]], [0])
    n = batch.n_tokens
    ads.c_struct().b_o = ctypes.POINTER(ctypes.c_void_p)()
    with pytest.raises(_lib.MicroserveError, match="without its B"):
        model.forward_paged(batch, cache, lora=ads.plan(["a"], [n]))
    assert _lib.device_error() == 0


def test_loading_refusals_change_nothing(golden) -> None:
    from microserve_b200.lora import LoraAdapters

    model = device_model(golden, "target")
    ads = LoraAdapters(model)
    good = adapter_state(model.cfg, 4, 1, ("attn.q_proj",))
    key = "blocks.0.attn.q_proj.lora_A.weight"
    bad = [{}, {**good, "blocks.9.attn.q_proj.lora_A.weight": good[key]}, {k: v for k, v in good.items() if k != key},
           {**good, key: good[key][:3]}, {**good, key: good[key][:, 1:]}, {**good, key: good[key][0]}]
    for st in bad:
        with pytest.raises(ValueError):
            ads.load("x", st)
    with pytest.raises(ValueError):
        ads.load("x", good, alpha=float("nan"))
    big = adapter_state(model.cfg, 257, 1, ("attn.q_proj",))
    with pytest.raises(ValueError):
        ads.load("x", big)
    assert ads.names == [] and ads._rank == []
    ads.load("x", good)
    with pytest.raises(ValueError, match="already"):
        ads.load("x", good)
    with pytest.raises(ValueError):
        ads.unload("y")
    with pytest.raises(ValueError):
        ads.plan(["y"], [3])
    with pytest.raises(ValueError):
        ads.acquire("y")
    from microserve_b200.lora import LoraPlan

    with pytest.raises(ValueError):  # a plan of another batch
        model.forward_paged(*_again(model, [1, 2, 3]), lora=LoraPlan.build([0, 0], DEV))
    other = device_model(golden, "target")
    with pytest.raises(ValueError, match="no adapters"):
        other.forward_paged(*_again(other, [1, 2, 3]), lora=LoraPlan.build([0, 0, 0], DEV))

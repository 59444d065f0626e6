"""Trees of drafted tokens: masks, the walk, and whole verify rounds through a model."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .form_check import DEV, pack_bits, tree_of

pytestmark = pytest.mark.gpu


def _i32(a) -> torch.Tensor:
    return torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(DEV)


@pytest.mark.parametrize("lens", [[1], [7, 1, 33], [64, 0, 65, 2], [300, 5], [1024, 31], [3] * 500])
@pytest.mark.parametrize("extra", [0, 3])
def test_masks_and_depths(lens, extra) -> None:
    from microserve_b200 import _lib
    from microserve_b200.tree import tree_masks

    rng = np.random.default_rng(len(lens))
    parents, depths = [], []
    top = max(lens)
    flags = np.zeros((sum(lens), (-(-top // 32) + extra) * 32), bool)
    at = 0
    for n in lens:
        p, d, sees = tree_of(n, rng)
        if n > 4:  # a second root
            p[3] = -1
            sees = np.eye(n, dtype=bool)
            for i in range(1, n):
                if p[i] >= 0:
                    sees[i] |= sees[p[i]]
            d = sees.sum(1) - 1
        parents.append(p)
        depths.append(d)
        flags[at : at + n, :n] = sees
        at += n
    q_start = np.concatenate([[0], np.cumsum(lens)])
    masks, got = tree_masks(_i32(np.concatenate(parents)), _i32(q_start), top, -(-top // 32) + extra)
    assert np.array_equal(masks.cpu().numpy().view(np.uint32), pack_bits(flags))
    assert np.array_equal(got.cpu().numpy(), np.concatenate(depths))
    assert _lib.device_error() == 0


def test_bad_parents_are_reported_and_count_as_roots() -> None:
    from microserve_b200 import _lib
    from microserve_b200.tree import tree_masks

    for bad in (2, 7, -2, 1 << 30):
        masks, depths = tree_masks(_i32([-1, 0, bad, 2]), _i32([0, 4]), 4)
        assert _lib.device_error() == 10
        assert masks.flatten().tolist() == [1, 3, 4, 12] and depths.tolist() == [0, 1, 0, 1]
    tree_masks(_i32([-1, 0, 0]), _i32([0, 5]), 5)
    assert _lib.device_error() == 9
    tree_masks(_i32([-1, 0, 0]), _i32([0, 3]), 2)
    assert _lib.device_error() == 9


def _case(seed: int, lens: list[int], vocab: int, bs: int, agree: float):
    from microserve_b200.model import PagedBatch

    rng = np.random.default_rng(seed)
    T = sum(lens)
    q_start = np.concatenate([[0], np.cumsum(lens)])
    parents = np.concatenate([tree_of(n, rng)[0] for n in lens])
    ids = rng.integers(0, min(vocab, 4), T)  # siblings repeat one another
    target = np.where(rng.random(T) < agree, rng.integers(0, min(vocab, 4), T), rng.integers(0, vocab, T))
    cached = rng.integers(0, 50, len(lens))
    context = cached + lens
    width = int(-(-context.max() // bs))
    blocks = len(lens) * width
    tables = rng.permutation(blocks).reshape(len(lens), width)
    z = _i32(np.zeros(T))
    batch = PagedBatch(input_ids=_i32(ids), positions=z, slot_mapping=z, block_tables=_i32(tables),
                       context_lens=_i32(context), q_lens=_i32(lens), q_start=_i32(q_start), max_q=max(lens),
                       n_tokens=T, max_context=int(context.max()))
    return batch, parents, ids, target, cached, tables, q_start, blocks


def _walk(lens, parents, ids, target, cached, tables, q_start, bs, most):
    B = len(lens)
    said, nodes = np.full((B, most + 1), -1), np.full((B, most), -1)
    src, dst, num = np.full((B, most), -1), np.full((B, most), -1), np.zeros(B, int)
    for b, n in enumerate(lens):
        at, t0 = 0, q_start[b]
        slot = lambda j, b=b: tables[b, j // bs] * bs + j % bs  # noqa: E731
        for k in range(most + 1):
            if n == 0:
                break
            token = said[b, k] = target[t0 + at]
            fits = [i for i in range(n) if parents[t0 + i] == at and ids[t0 + i] == token]
            if k == most or not fits:
                break
            at = nodes[b, k] = fits[0]
            src[b, k], dst[b, k] = slot(cached[b] + at), slot(cached[b] + k + 1)
            num[b] += 1
    return said, num, nodes, src, dst


@pytest.mark.parametrize("lens,most", [([1], 3), ([7] * 8, 4), ([33, 1, 0, 64, 9], 9), ([300, 1024], 40), ([5, 6], 0),
                                       ([12] * 300, 5)])
@pytest.mark.parametrize("vocab", [3, 65, 4099, 32000, 128256])
@pytest.mark.parametrize("by_logits", [False, True])
def test_the_walk(lens, most, vocab, by_logits) -> None:
    from microserve_b200 import _lib
    from microserve_b200.tree import accept_trees

    if by_logits and sum(lens) * vocab > 2 ** 28:
        pytest.skip("logits beyond 1 GB")
    bs = 16
    batch, parents, ids, target, cached, tables, q_start, blocks = _case(most + vocab, lens, vocab, bs, 0.9)
    T = sum(lens)
    if by_logits:
        pad = 1 if vocab % 2 else 0
        g = torch.Generator(device=DEV).manual_seed(1)
        t = torch.randn((T, vocab + pad), generator=g, device=DEV)[:, :vocab]
        # the target's token twice: the lowest of equals counts; NaN and -inf never
        t[:, -1] = float("nan") if vocab > 65 else t[:, -1]
        t[torch.arange(T, device=DEV), _i32(target).long()] = 9.0
        t[torch.arange(T, device=DEV), _i32(np.minimum(target + 7, vocab - 2 if vocab > 65 else vocab - 1)).long()] = 9.0
        if vocab > 65:
            target = np.minimum(target, vocab - 2)
            t[torch.arange(T, device=DEV), _i32(target).long()] = 9.0
            t[:, -1] = float("nan")
        target = np.array([int(torch.nonzero(r == 9.0)[0]) for r in t.cpu()])
    else:
        t = _i32(target)
    got = accept_trees(t, batch, _i32(parents), most, bs, blocks)
    want = _walk(lens, parents, ids, target, cached, tables, q_start, bs, most)
    for name, w in zip(("tokens", "num_accepted", "nodes", "src_slots", "dst_slots"), want):
        assert np.array_equal(getattr(got, name).cpu().numpy(), w), name
    assert _lib.device_error() == 0


def test_a_walk_without_moves_needs_no_cache() -> None:
    """The C call with neither slots nor a cache's sizes: contexts are not looked at."""
    from microserve_b200 import _lib
    from microserve_b200.attention import pack_batch
    from microserve_b200.tree import accept_trees

    lens, most = [7, 33, 1], 5
    batch, parents, ids, target, cached, tables, q_start, blocks = _case(5, lens, 65, 16, 0.9)
    want = accept_trees(_i32(target), batch, _i32(parents), most, 16, blocks)
    batch.context_lens = _i32([2 ** 30, -5, 0])
    batch.block_tables = _i32(np.zeros((3, 0)))
    target, parents = _i32(target), _i32(parents)
    tokens, nodes, num = (torch.empty(n, dtype=torch.int32, device=DEV) for n in (18, 15, 3))
    _lib.launch_on(_lib.cuda_index(tokens), "ms_tree_accept", None, 0, 0, target.data_ptr(),
                   pack_batch(batch, _lib.cuda_index(tokens), True), parents.data_ptr(), most, 0, 0, tokens.data_ptr(),
                   num.data_ptr(), nodes.data_ptr(), None, None)
    assert torch.equal(tokens.view(3, 6), want.tokens) and torch.equal(num, want.num_accepted)
    assert torch.equal(nodes.view(3, 5), want.nodes) and _lib.device_error() == 0


@pytest.mark.parametrize("vocab", [65, 32000])
def test_the_walk_of_a_padded_batch(vocab) -> None:
    """Rows behind the last sequence are not read, and sequences without nodes emit nothing."""
    from microserve_b200 import _lib
    from microserve_b200.tree import accept_trees, tree_masks

    lens, most = [7, 0, 12], 4
    batch, parents, ids, target, cached, tables, q_start, blocks = _case(9, lens, vocab, 16, 0.9)
    want = _walk(lens, parents, ids, target, cached, tables, q_start, 16, most)
    plain = tree_masks(_i32(parents), batch.q_start, batch.max_q)
    T, extra = sum(lens), 5
    parents, target = np.append(parents, [10 ** 6] * extra), np.append(target, [-7] * extra)
    batch.input_ids = _i32(np.append(ids, [-1] * extra))
    batch.positions = batch.slot_mapping = _i32(np.zeros(T + extra))
    batch.n_tokens = T + extra
    logits = torch.full((T + extra, vocab), float("nan"), device=DEV)
    logits[:T] = 0.0
    logits[torch.arange(T, device=DEV), _i32(target[:T]).long()] = 1.0
    for t in (_i32(target), logits):
        got = accept_trees(t, batch, _i32(parents), most, 16, blocks)
        for name, w in zip(("tokens", "num_accepted", "nodes", "src_slots", "dst_slots"), want):
            assert np.array_equal(getattr(got, name).cpu().numpy(), w), name
    masks, depths = tree_masks(_i32(parents), batch.q_start, batch.max_q)
    assert torch.equal(masks[:T], plain[0]) and torch.equal(depths[:T], plain[1])
    assert _lib.device_error() == 0


def test_rows_of_infinities() -> None:
    """A row of -inf alone, or of NaN alone, gives token 0; +inf is the largest."""
    from microserve_b200.tree import accept_trees

    batch, *_ = _case(0, [1, 1, 1], 5000, 16, 1.0)
    t = torch.full((3, 5000), -float("inf"), device=DEV)
    t[1] = float("nan")
    t[2, 4777] = float("inf")
    got = accept_trees(t, batch, _i32([-1, -1, -1]), 2, 16)
    assert got.tokens[:, 0].tolist() == [0, 0, 4777] and got.num_accepted.tolist() == [0, 0, 0]


def test_refusals() -> None:
    from microserve_b200.tree import accept_trees, tree_masks

    batch, parents, *_ = _case(0, [3, 4], 65, 16, 1.0)
    t, p = torch.zeros((7, 65), device=DEV), _i32(parents)
    for args in ((t[:-1], batch, p, 2, 16), (t.half(), batch, p, 2, 16), (t.t(), batch, p, 2, 16),
                 (t, batch, p[:-1], 2, 16), (t, batch, p.long(), 2, 16), (t, batch, p, -1, 16), (t, batch, p, 2, 0),
                 (_i32(np.zeros(6)), batch, p, 2, 16), (torch.zeros(7, device=DEV), batch, p, 2, 16),
                 (t[:, :0], batch, p, 2, 16)):
        with pytest.raises(ValueError):
            accept_trees(*args)
    for args in ((p.long(), batch.q_start, 4), (p, batch.q_start, 1025), (p, batch.q_start, 40, 1),
                 (p, batch.q_start.long(), 4)):
        with pytest.raises(ValueError):
            tree_masks(*args)


# ------------------------------------------------------------------------------------- whole rounds


def _model(dtype: str = "float32", **kw):
    from microserve_b200.config import ModelConfig
    from microserve_b200.model import Transformer

    kw = {"vocab_size": 61, "n_layers": 3, "d_model": 64, "n_heads": 4, "n_kv_heads": 2, "max_seq_len": 256, **kw}
    return Transformer(ModelConfig(dtype=dtype, **kw), DEV, seed=3)


def _cache(model, blocks: int = 200, bs: int = 8):
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig

    return PagedKVCache(model.cfg, CacheConfig(bs, blocks, model.cfg.dtype), DEV)


def _prefill(model, cache, prompts) -> None:
    """Everything but each prompt's last token."""
    from microserve_b200.batching import build_paged_batch

    ids = [i for i, p in enumerate(prompts) if len(p) > 1]
    if ids:
        model.forward_paged(build_paged_batch(cache, ids, [prompts[i][:-1] for i in ids], [0] * len(ids)), cache)


def _ordinary(model, prompts, n, sampling=None, seeds=None):
    """The streams of ordinary passes, one token at a time."""
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.sampling import make_params, params_to_device
    from microserve_b200 import _lib

    cache = _cache(model)
    _prefill(model, cache, prompts)
    last, out = [p[-1] for p in prompts], [[] for _ in prompts]
    B = len(prompts)
    for step in range(n):
        batch = build_paged_batch(cache, list(range(B)), [[t] for t in last], [cache.num_tokens(i) for i in range(B)])
        logits = model.forward_paged(batch, cache)
        if sampling is None:
            last = logits.argmax(-1).tolist()
        else:
            params = params_to_device(make_params(sampling, seeds, [step] * B), logits.device)
            tokens = torch.empty(B, dtype=torch.int32, device=DEV)
            _lib.call("ms_sample", logits.data_ptr(), logits.shape[1], B, logits.shape[1], params.data_ptr(), None, 0,
                      tokens.data_ptr(), None, None, None, None, _lib.stream_ptr())
            last = tokens.tolist()
        for o, t in zip(out, last):
            o.append(t)
    return out


def _trees_for(rng, streams, done, last, vocab, size):
    """Trees that hold the next tokens of each stream on some path, among wrong ones."""
    trees = []
    for s, k, t in zip(streams, done, last):
        tokens, parents, at = [t], [-1], 0
        right = int(rng.integers(0, size))
        follow = list(s[k : k + right])
        while len(tokens) < size:
            if follow and rng.random() < 0.5:
                tokens.append(follow.pop(0))
                parents.append(at)
                at = len(tokens) - 1
            else:
                tokens.append(int(rng.integers(0, vocab)))
                parents.append(int(rng.integers(0, len(parents))))
        trees.append((tokens, parents))
    return trees


def _rounds(model, prompts, streams, n, seed, size, sampling=None, seeds=None):
    from microserve_b200.tree import verify_trees

    rng = np.random.default_rng(seed)
    cache = _cache(model)
    _prefill(model, cache, prompts)
    B = len(prompts)
    got, last, rounds = [[] for _ in prompts], [p[-1] for p in prompts], 0
    while min(map(len, got)) < n:
        trees = _trees_for(rng, streams, [len(g) for g in got], last, model.cfg.vocab_size, size)
        out = verify_trees(model, cache, list(range(B)), trees, sampling, seeds,
                           None if sampling is None else [len(g) for g in got])
        rounds += 1
        for i, o in enumerate(out):
            assert o
            got[i] += o
            last[i] = o[-1]
            assert cache.num_tokens(i) == len(prompts[i]) - 1 + len(got[i])
        cache.allocator.check_invariants()
    return got, rounds, cache


PROMPTS = [[5, 9, 2], [7], list(range(20)), [3] * 9]


@pytest.mark.parametrize("size", [1, 2, 9, 40])
def test_greedy_rounds_give_the_ordinary_streams(size) -> None:
    model = _model()
    n = 24
    want = _ordinary(model, PROMPTS, n + 41)
    got, rounds, _ = _rounds(model, PROMPTS, want, n, size, size)
    for g, w in zip(got, want):
        assert g[:n] == w[:n]
    assert rounds == n if size == 1 else rounds < n


def test_sampled_rounds_give_the_ordinary_streams() -> None:
    """The uniforms go by draw step, so the streams are those of ordinary passes."""
    from microserve_b200.config import SamplingConfig

    model = _model()
    sampling = [SamplingConfig(temperature=1.0), SamplingConfig(temperature=0.7, top_k=20),
                SamplingConfig(temperature=0.0), SamplingConfig(temperature=1.2, top_p=0.9)]
    seeds = [11, 12, 13, 14]
    want = _ordinary(model, PROMPTS, 60, sampling, seeds)
    got, rounds, _ = _rounds(model, PROMPTS, want, 20, 5, 12, sampling, seeds)
    for g, w in zip(got, want):
        assert g[:20] == w[:20]
    assert rounds < 20


def test_the_cache_after_a_round_is_that_of_ordinary_passes() -> None:
    """The kept path's keys and values are, position by position, those that ordinary passes write."""
    from microserve_b200.batching import build_paged_batch

    model = _model()
    want = _ordinary(model, PROMPTS, 70)
    got, _, cache = _rounds(model, PROMPTS, want, 20, 9, 16)
    plain = _cache(model)
    B = len(PROMPTS)
    tokens = [p + g[:-1] for p, g in zip(PROMPTS, got)]
    model.forward_paged(build_paged_batch(plain, list(range(B)), tokens, [0] * B), plain)
    for i in range(B):
        n = cache.num_tokens(i)
        assert plain.num_tokens(i) == n
        for layer in range(model.cfg.n_layers):
            a, b = (c.gather(layer, c.build_block_tables([i])[0], n) for c in (cache, plain))
            for x, y in zip(a, b):
                torch.testing.assert_close(x, y, rtol=1e-4, atol=1e-5)


@pytest.mark.parametrize("heads,kv,d", [(4, 2, 256), (8, 1, 512), (2, 2, 256)])
def test_bf16_logits_of_a_tree_are_those_of_its_paths(heads, kv, d) -> None:
    """Each node's logits against a float32 model's over the node's own path."""
    from microserve_b200.attention import AttentionForm
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.config import ModelConfig
    from microserve_b200.model import Transformer
    from microserve_b200.tree import tree_masks

    model = _model("bfloat16", d_model=d, n_heads=heads, n_kv_heads=kv)
    f32 = Transformer.from_state_dict(ModelConfig(**{**model.cfg.__dict__, "dtype": "float32"}), model.state_dict(), DEV)
    rng = np.random.default_rng(0)
    prompt = rng.integers(0, 61, 50).tolist()
    parents, depths, _ = tree_of(14, rng)
    tokens = rng.integers(0, 61, 14).tolist()
    cache = _cache(model, bs=16)
    model.forward_paged(build_paged_batch(cache, [0], [prompt], [0]), cache)
    batch = build_paged_batch(cache, [0], [tokens], [50])
    batch.positions = _i32(50 + depths)
    masks, got_depths = tree_masks(_i32(parents), batch.q_start, 14)
    assert got_depths.tolist() == depths.tolist()
    logits = model.forward_paged(batch, cache, form=AttentionForm(tree_mask=masks))
    for i in range(14):
        path, at = [], i
        while at >= 0:
            path.insert(0, tokens[at])
            at = parents[at]
        ref_cache = _cache(f32, bs=16)
        ref = f32.forward_paged(build_paged_batch(ref_cache, [0], [prompt + path], [0]), ref_cache)[-1]
        assert float((logits[i] - ref).abs().max()) <= 2e-2 * max(1.0, float(ref.abs().max()))


def test_no_form_in_a_forward_is_the_plain_forward() -> None:
    from microserve_b200.attention import AttentionForm
    from microserve_b200.batching import build_paged_batch

    model = _model()
    logits = []
    for form in (None, AttentionForm()):
        cache = _cache(model)
        logits.append(model.forward_paged(build_paged_batch(cache, [0, 1], [[1, 2, 3], [4]], [0, 0]), cache, form=form))
    torch.testing.assert_close(logits[0], logits[1], rtol=1e-4, atol=1e-5)


def test_forwards_with_a_form_in_two_graphs() -> None:
    """Each graph has a workspace of its own, whatever runs between, larger passes among it."""
    from microserve_b200.attention import AttentionForm
    from microserve_b200.batching import build_paged_batch

    model = _model()
    rng = np.random.default_rng(3)
    form = AttentionForm(softcap=2.0, window=9)
    runs = []
    for n in (5, 60):
        prompts = [rng.integers(0, 61, n).tolist() for _ in range(3)]
        cache = _cache(model)
        batch = build_paged_batch(cache, [0, 1, 2], prompts, [0, 0, 0])
        want = model.forward_paged(batch, cache, form=form).clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = model.forward_paged(batch, cache, form=form)
        runs.append((g, got, want, batch, cache))
    big = _cache(model, blocks=400)
    model.forward_paged(build_paged_batch(big, list(range(12)), [[1] * 200] * 12, [0] * 12), big, form=form)
    junk = [torch.full((1 << 20,), 7.0, device=DEV) for _ in range(8)]  # over whatever was freed
    for _ in range(2):
        for g, got, *_ in runs:
            got.zero_()
            g.replay()
        for _, got, want, batch, cache in runs:
            torch.testing.assert_close(got, want, rtol=1e-4, atol=1e-5)
            torch.testing.assert_close(model.forward_paged(batch, cache, form=form), want, rtol=1e-4, atol=1e-5)
    assert all(bool((j == 7).all()) for j in junk)


def test_a_tree_with_adapters() -> None:
    """Forms and adapters in one pass: a chain as a tree is the plain forward with the same adapters."""
    from microserve_b200.attention import AttentionForm
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.lora import LoraAdapters
    from microserve_b200.tree import tree_masks

    from .test_gpu_controls_engine import adapter_state

    model = _model()
    ads = LoraAdapters(model)
    ads.load("a", adapter_state(model.cfg, 4, 1, ("attn.q_proj", "attn.v_proj", "ffn.down_proj"), 8.0))
    prompts = [[1, 2, 3, 4, 5, 6, 7], [4, 5], [9] * 40]
    lens = [len(p) for p in prompts]
    logits = []
    for adapter, tree in ((None, False), ("a", False), ("a", True)):
        cache = _cache(model)
        batch = build_paged_batch(cache, [0, 1, 2], prompts, [0, 0, 0])
        parents = _i32(np.concatenate([np.arange(n) - 1 for n in lens]))
        form = AttentionForm(tree_mask=tree_masks(parents, batch.q_start, batch.max_q)[0]) if tree else None
        lora = ads.plan([adapter] * 3, lens) if adapter else None
        logits.append(model.forward_paged(batch, cache, lora=lora, form=form).clone())
    torch.testing.assert_close(logits[1], logits[2], rtol=1e-4, atol=1e-5)
    assert float((logits[0] - logits[1]).abs().max()) > 0.01


def test_masks_walk_and_moves_in_a_graph() -> None:
    """A captured round on a side stream, replayed with other target tokens and another tree."""
    from microserve_b200 import _lib
    from microserve_b200.cache import move_tokens
    from microserve_b200.tree import accept_trees, tree_masks

    lens, most, bs, vocab = [9, 40, 1, 17], 6, 16, 65
    case = _case(31, lens, vocab, bs, 0.9)
    batch, blocks = case[0], case[-1]
    pool = torch.randn((2, 2, blocks, 2, bs, 16), device=DEV)
    parents, target = _i32(case[1]), _i32(case[3])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            masks, depths = tree_masks(parents, batch.q_start, max(lens))
            got = accept_trees(target, batch, parents, most, bs, blocks)
            move_tokens(pool, got.src_slots, got.dst_slots)
    torch.cuda.synchronize()
    for seed in (31, 32, 33):
        other = _case(seed, lens, vocab, bs, 0.9)
        parents.copy_(_i32(other[1]))
        target.copy_(_i32(other[3]))
        batch.input_ids.copy_(_i32(other[2]))
        before = pool.clone()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g.replay()
        side.synchronize()
        want = _walk(lens, other[1], other[2], other[3], case[4], case[5], case[6], bs, most)
        for name, w in zip(("tokens", "num_accepted", "nodes", "src_slots", "dst_slots"), want):
            assert np.array_equal(getattr(got, name).cpu().numpy(), w), name
        for s, d in zip(want[3].ravel(), want[4].ravel()):
            if s >= 0:
                assert torch.equal(pool[:, :, d // bs, :, d % bs], before[:, :, s // bs, :, s % bs])
        plain = tree_masks(parents, batch.q_start, max(lens))
        assert torch.equal(masks, plain[0]) and torch.equal(depths, plain[1])
    assert _lib.device_error() == 0


def test_verify_trees_refuses_and_leaves_the_cache() -> None:
    from microserve_b200.config import SamplingConfig
    from microserve_b200.tree import verify_trees

    model = _model(max_seq_len=64)
    cache = _cache(model, blocks=12)
    _prefill(model, cache, [[1, 2, 3, 4, 5]])
    good = ([5, 6, 7], [-1, 0, 0])
    cases = [
        dict(trees=[good, good]), dict(trees=[([], [])]), dict(trees=[([5, 6], [-1])]), dict(trees=[([5, 6], [-1, -1])]),
        dict(trees=[([5, 6], [0, 0])]), dict(trees=[([5, 6], [-1, 1])]), dict(trees=[([5, 61], [-1, 0])]),
        dict(trees=[([5] * 61, [-1, *range(60)])]), dict(trees=[good], sampling=[SamplingConfig()]),
        dict(trees=[good], sampling=[SamplingConfig(presence_penalty=1.0)], seeds=[0], steps=[0]),
    ]
    for kw in cases:
        with pytest.raises(ValueError):
            verify_trees(model, cache, [0], **kw)
    with pytest.raises(ValueError):
        verify_trees(model, cache, [0, 0], [good, good])
    cache.fork(0, 1)
    with pytest.raises(ValueError, match="unshare"):
        verify_trees(model, cache, [0], [good])
    assert cache.num_tokens(0) == 4
    cache.unshare_many([0])
    assert verify_trees(model, cache, [0], [good]) and verify_trees(model, cache, [], []) == []
    cache.allocator.check_invariants()


def test_forked_sequences_verify_their_own_trees() -> None:
    """Forks of one prompt take different trees in one pass; compaction in between changes nothing."""
    model = _model()
    prompts = [PROMPTS[2]] * 3
    from microserve_b200.tree import verify_trees

    want = _ordinary(model, prompts, 40)
    cache = _cache(model)
    cache.append(99, 30)  # in the way, so that compaction has something to do
    _prefill(model, cache, prompts[:1])
    cache.fork_many(0, [1, 2])
    cache.free(99)
    rng = np.random.default_rng(0)
    got, last = [[], [], []], [prompts[0][-1]] * 3
    for _ in range(6):
        out = verify_trees(model, cache, [0, 1, 2], _trees_for(rng, want, [len(g) for g in got], last, 61, 8))
        for i, o in enumerate(out):
            got[i] += o
            last[i] = o[-1]
        cache.compact()
    for g, w in zip(got, want):
        assert g == w[: len(g)]

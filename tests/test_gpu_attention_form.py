"""Attention with score forms against the plain implementation in 64 bits (form_check.py says
where the tolerances come from).  Everything that no sequence holds is NaN in the pools."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from .form_check import DEV, Inputs, check, make, reference, run, visible

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32

# dtype, hq, hkv, dh, block size
SHAPES = [
    (F32, 4, 4, 32, 16), (F32, 4, 2, 8, 4), (F32, 6, 2, 64, 5), (F32, 2, 1, 128, 16), (F32, 8, 1, 16, 8),
    (BF16, 32, 4, 64, 16), (BF16, 8, 2, 128, 16), (BF16, 6, 2, 64, 8), (BF16, 5, 1, 128, 64),
    (BF16, 4, 4, 64, 32), (BF16, 4, 2, 128, 128), (BF16, 4, 2, 32, 16), (BF16, 4, 2, 64, 12), (BF16, 3, 3, 128, 2),
]
FORMS = {
    "plain": {},
    "cap": dict(softcap=3.0),
    "slopes": dict(alibi=True),
    "window": dict(window=37),
    "all": dict(softcap=5.0, alibi=True, window=50),
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,hq,hkv,dh,bs", SHAPES)
def test_trees(dtype, hq, hkv, dh, bs, form) -> None:
    x = make(hq + dh + bs, dtype, hq, hkv, dh, bs, [0, 1, 63, 64, 200, 131], [1, 7, 9, 33, 16, 5], tree=True,
             **FORMS[form])
    check(run(x), x)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype,hq,hkv,dh,bs", SHAPES)
def test_single_tokens(dtype, hq, hkv, dh, bs, form) -> None:
    x = make(hq + dh + bs, dtype, hq, hkv, dh, bs, [0, 1, 15, 16, 63, 64, 127, 300], [1] * 8, **FORMS[form])
    check(run(x), x)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("prefix", [False, True])
@pytest.mark.parametrize("dtype,hq,hkv,dh,bs", SHAPES)
def test_prompts(dtype, hq, hkv, dh, bs, prefix, form) -> None:
    cached, q = [0, 70, 0, 129], [140, 33, 1, 65]
    x = make(hq + dh + bs, dtype, hq, hkv, dh, bs, cached, q, prefix=[100, 0, 1, 20] if prefix else None, **FORMS[form])
    check(run(x), x)


@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("hkv,hq", [(2, 16), (1, 16), (2, 4)])
@pytest.mark.parametrize("nodes", [[64, 3], [128], [61, 65], [200, 17]])
def test_wide_trees(dh, hkv, hq, nodes) -> None:
    """Trees whose rows fill several tiles, mask rows of several words."""
    x = make(dh + hq, BF16, hq, hkv, dh, 16, [300, 77][: len(nodes)], nodes, tree=True, softcap=20.0, alibi=True)
    check(run(x), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("window", [0, 100, 4000])
def test_long_context_of_few_rows(dtype, window) -> None:
    """The KV axis is split and joined again; ragged lengths leave some ranges empty."""
    x = make(3, dtype, 8, 2, 64, 16, [5000, 1, 900], [3, 2, 4], tree=True, window=window)
    check(run(x), x)
    x = make(4, dtype, 4, 1, 128, 16, [9001], [1], alibi=True, window=window)
    check(run(x), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dh", [64, 128])
def test_window_behind_a_prefix_leaves_a_hole(dtype, dh) -> None:
    x = make(dh, dtype, 4, 2, dh, 16, [700, 300, 40], [9, 1, 5], window=20, prefix=[33, 290, 45])
    check(run(x), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("hq", [2, 16])
@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_flat_and_sharp_scores(dtype, hq, spread) -> None:
    x = make(11, dtype, hq, 2, 64, 16, [200, 17], [9, 12], tree=True, spread=spread)
    check(run(x), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("dh,nodes", [(64, 5), (128, 5), (64, 70), (128, 70)])
def test_rows_that_see_nothing_give_zero(dtype, dh, nodes) -> None:
    masks = np.zeros((nodes + 3, nodes), bool)
    masks[1, 1] = masks[2, [0, nodes - 1]] = True
    masks[nodes + 1, 1] = True
    x = make(5, dtype, 8, 2, dh, 16, [0, 0], [nodes, 3], tree=True, masks=masks)
    got = run(x)
    check(got, x)
    assert not got[0].any() and not got[nodes].any() and not got[nodes + 2].any()
    # a window that lets a row see nothing of the context, and a mask nothing of the tree
    x = make(6, dtype, 8, 2, dh, 16, [100, 90], [nodes, 3], tree=True, masks=masks, window=1)
    got = run(x)
    check(got, x)
    assert not got[0].any()


@pytest.mark.parametrize("value", [float("inf"), -float("inf"), float("nan")])
@pytest.mark.parametrize("dtype,dh,hq,n", [(F32, 32, 4, 9), (BF16, 64, 4, 9), (BF16, 128, 4, 9), (BF16, 64, 16, 40),
                                           (BF16, 128, 16, 40)])
@pytest.mark.parametrize("tree", [False, True])
def test_what_a_row_does_not_see_cannot_reach_it(value, dtype, dh, hq, n, tree) -> None:
    """A key and another value of the pass's own tokens are not finite: rows that see them get the
    formula's result, all others are as if nothing were wrong."""
    x = make(8, dtype, hq, 2, dh, 16, [50, 130], [n, n], tree=tree)
    t = lambda b, j: (int(x.tables[b, j // 16]), slice(None), j % 16)  # noqa: E731
    x.v[t(0, 50 + n - 3)][:, 5] = value  # one dimension of one value
    x.k[t(1, 130 + n - 2)] = value
    ref, tol = reference(x)
    hurt = {int(x.q_start[b]) + i for b, j in ((0, 50 + n - 3), (1, 130 + n - 2)) for i in range(n)
            if j in visible(x, b, i)[0]}
    assert hurt and len(hurt) < n
    got = run(x).double().cpu()
    rows = [r for r in range(2 * n) if r not in hurt]
    assert bool(got[rows].isfinite().all())
    assert bool(((got - ref).abs() <= tol)[rows].all())
    for r in hurt:
        if r < n:  # the value: its own dimension only
            other = [d for d in range(dh) if d != 5]
            assert bool(((got - ref).abs() <= tol)[r][:, other].all())
            assert torch.equal(got[r, :, 5].isnan(), ref[r, :, 5].isnan())
            assert torch.equal(got[r, :, 5].nan_to_num(), ref[r, :, 5].nan_to_num())


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_of_queries_and_results(dtype) -> None:
    x = make(9, dtype, 8, 2, 64, 16, [33, 90], [3, 6], tree=True)
    T = 9
    for extra, shift in ((2 * 2 * 64, 0), (7, 0), (9, 1), (8, 8)):
        wide = torch.randn((T, 8 * 64 + extra + shift), device=DEV).to(dtype)
        q = wide[:, shift : shift + 512].view(T, 8, 64)
        q.copy_(x.q.to(DEV))
        holder = torch.full((T, 512 + extra + shift), 7.0, device=DEV, dtype=dtype)
        out = holder[:, shift : shift + 512].view(T, 8, 64)
        assert run(x, q=q, out=out) is out
        check(out, x)
        assert bool((holder[:, :shift] == 7).all()) and bool((holder[:, shift + 512 :] == 7).all())


def test_results_do_not_depend_on_the_rest_of_the_batch() -> None:
    """A sequence gives the same bits twice, and rows of other sequences do not change with its content."""
    x = make(10, BF16, 8, 2, 64, 16, [333, 90, 20], [9, 6, 17], tree=True)
    a = run(x)
    assert torch.equal(a, run(x))
    x.q[:9] = 0.5
    b = run(x)
    assert torch.equal(a[9:], b[9:]) and not torch.equal(a[:9], b[:9])


def test_stream_and_graph() -> None:
    from microserve_b200.attention import paged_attention

    x = make(12, BF16, 8, 2, 128, 16, [900, 90], [9, 6], tree=True)
    want = reference(x)
    q, k, v, batch, form = x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), x.batch(), x.form()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = paged_attention(q, k, v, batch, form)
    torch.cuda.current_stream().wait_stream(side)
    check(got, x, want)
    out, out2 = torch.zeros_like(q), torch.zeros_like(q)
    graphs = []
    for o in (out, out2):  # two graphs with workspaces of their own
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            paged_attention(q, k, v, batch, form, o)
        graphs.append(g)
    for g, o in zip(graphs, (out, out2)):
        g.replay()
    torch.cuda.synchronize()
    check(out, x, want)
    check(out2, x, want)
    q.mul_(0.5)
    x.q.mul_(0.5)
    graphs[0].replay()
    check(out, x)


def test_bad_lengths_and_blocks_are_reported_and_stay_inside() -> None:
    from microserve_b200 import _lib
    from microserve_b200.attention import paged_attention

    def error(change) -> int:
        x = make(13, BF16, 8, 2, 64, 16, [300, 90], [9, 6], tree=True)
        batch = x.batch()
        change(batch)
        paged_attention(x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), batch, x.form())
        return _lib.device_error()

    def set_(name, i, value):
        return lambda b: getattr(b, name).view(-1).__setitem__(i, value)

    assert error(lambda b: None) == 0
    assert error(set_("block_tables", 3, 10 ** 6)) == 2
    assert error(set_("block_tables", 3, -5)) == 2
    assert error(set_("context_lens", 1, 10 ** 8)) == 9
    assert error(set_("context_lens", 1, -4)) == 9
    assert error(set_("q_start", 2, 10 ** 6)) == 9
    assert error(set_("q_start", 1, -1)) == 9
    assert error(lambda b: setattr(b, "max_q", 7)) == 9


def test_a_batch_without_tokens() -> None:
    x = make(14, F32, 4, 2, 32, 16, [5], [2])
    from microserve_b200.attention import paged_attention
    from microserve_b200.model import PagedBatch

    z = torch.zeros(0, dtype=torch.int32, device=DEV)
    one = torch.zeros(1, dtype=torch.int32, device=DEV)
    empty = PagedBatch(input_ids=z, positions=z, slot_mapping=z, block_tables=z.view(0, 1), context_lens=z, q_lens=z,
                       q_start=one, max_q=0, n_tokens=0)
    q = torch.zeros((0, 4, 32), device=DEV)
    assert paged_attention(q, x.k.to(DEV), x.v.to(DEV), empty).shape == (0, 4, 32)
    # a sequence without tokens between others
    x = make(15, F32, 4, 2, 32, 16, [5, 9], [2, 3])
    b = x.batch()
    b.q_start = torch.tensor([0, 2, 2, 5], dtype=torch.int32, device=DEV)
    b.q_lens = torch.tensor([2, 0, 3], dtype=torch.int32, device=DEV)
    b.context_lens = torch.tensor([7, 0, 12], dtype=torch.int32, device=DEV)
    b.block_tables = b.block_tables[[0, 0, 1]].contiguous()
    got = paged_attention(x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), b)
    check(got, x)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_no_form_is_plain_causal_attention(dtype) -> None:
    from microserve_b200.attention import paged_attention

    x = make(16, dtype, 8, 4, 64, 16, [30, 0, 400], [4, 20, 1])
    got = paged_attention(x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), x.batch())
    check(got, x)


def test_positions_other_than_the_usual_ones() -> None:
    """Causality goes by the positions given, not by the order of the rows."""
    x = make(17, BF16, 8, 2, 64, 16, [40, 300], [6, 80])
    x.positions[:6] = [45, 3, 44, 0, 41, 20]
    rng = np.random.default_rng(1)
    x.positions[6:] = 300 + rng.permutation(80)
    check(run(x), x)


def _refused(match: str, **kw) -> None:
    from microserve_b200.attention import paged_attention

    x: Inputs = make(18, BF16, 8, 2, 64, 16, [30, 20], [4, 2], tree=True)
    args = dict(q=x.q.to(DEV), k_pool=x.k.to(DEV), v_pool=x.v.to(DEV), batch=x.batch(), form=x.form(), out=None)
    for name, f in kw.items():
        if name in args:
            args[name] = f(args[name])
        else:
            setattr(args["form"], name, f(getattr(args["form"], name)))
    with pytest.raises(ValueError, match=match):
        paged_attention(**args)


def test_refusals() -> None:
    _refused("q must be", q=lambda t: t.half())
    _refused("k_pool must be", k_pool=lambda t: t.float())
    _refused("v_pool must be", v_pool=lambda t: t[:-1])
    _refused("k_pool must be", k_pool=lambda t: t.transpose(1, 2))
    _refused("the batch", q=lambda t: t[:-1])
    _refused("heads", q=lambda t: t[:, :7].contiguous())
    _refused("contiguous heads", q=lambda t: t.transpose(0, 1).contiguous().transpose(0, 1))
    _refused("out must", out=lambda _: torch.empty((6, 8, 64), device=DEV))
    _refused("slopes", slopes=lambda _: torch.zeros(7, device=DEV))
    _refused("prefix_lens", prefix_lens=lambda _: torch.zeros(3, dtype=torch.int32, device=DEV))
    _refused("tree_mask", tree_mask=lambda t: t[:-1])
    _refused("tree_mask", tree_mask=lambda t: t.long())
    _refused("tree_mask", tree_mask=lambda t: t[:, :0])
    _refused("softcap", softcap=lambda _: float("nan"))
    _refused("softcap", softcap=lambda _: -1.0)
    _refused("softcap", scale=lambda _: float("inf"))
    _refused("window", window=lambda _: -1)
    x = make(19, BF16, 4, 2, 64, 16, [30], [4])
    q = torch.zeros((8, 4, 64), device=DEV, dtype=BF16)
    with pytest.raises(ValueError, match="overlap"):
        run(x, q=q[:4], out=q[2:6])


@pytest.mark.parametrize("dh,hq,n", [(64, 4, 9), (128, 4, 9), (64, 16, 40), (128, 16, 40), (128, 16, 10), (64, 16, 10)])
@pytest.mark.parametrize("tree", [False, True])
def test_the_largest_values_in_unseen_places(dh, hq, n, tree) -> None:
    """Stale places hold the type's largest finite value: an unseen key's weight is exactly 0."""
    big = float(torch.finfo(BF16).max)
    x = make(21, BF16, hq, 2, dh, 16, [50, 130, 0], [n, n - 1, 1], tree=tree, stale=big, window=0 if tree else 30)
    for _ in range(2):
        check(run(x), x)
    for b, c in enumerate((50, 130)):  # and so do other branches' values, and keys that come later
        page = int(x.tables[b, (c + 2) // 16])
        x.v[page, :, (c + 2) % 16] = big
    seen = [r for b in range(2) for r in range(int(x.q_start[b]), int(x.q_start[b + 1]))
            if x.context[b] - x.q_lens[b] + 2 not in visible(x, b, r - int(x.q_start[b]))[0]]
    got = run(x).double().cpu()
    ref, tol = reference(x)
    assert seen and bool(((got - ref).abs() <= tol)[seen].all())


@pytest.mark.parametrize("dtype,hq,dh", [(F32, 2, 64), (BF16, 2, 64), (BF16, 16, 128), (BF16, 2, 32)])
def test_pools_beyond_four_gigabytes(dtype, hq, dh) -> None:
    """Pages whose offsets pass 32 bits, in bytes and in elements."""
    from microserve_b200.attention import paged_attention

    x = make(22, dtype, hq, 1, dh, 16, [40, 100], [5, 9], tree=True)
    blocks = x.k.shape[0]
    total = (2 ** 32 + 2 ** 28) // (16 * dh)
    big = torch.empty((2, total, 1, 16, dh), dtype=dtype, device=DEV)  # (not filled: only the pages in use are)
    batch = x.batch()
    high = total - blocks
    batch.block_tables += high
    big[0, high:].copy_(x.k)
    big[1, high:].copy_(x.v)
    check(paged_attention(x.q.to(DEV), big[0], big[1], batch, x.form()), x)


@pytest.mark.parametrize("dtype,shift", [(F32, 1), (F32, 2), (BF16, 1), (BF16, 4)])
@pytest.mark.parametrize("n", [1, 40])
def test_pools_that_start_anywhere(dtype, shift, n) -> None:
    """Pools that are not aligned to 16 bytes."""
    from microserve_b200.attention import paged_attention

    x = make(23, dtype, 4, 2, 64, 16, [70, 20], [n, n], tree=True)
    pools = []
    for t in (x.k, x.v):
        flat = torch.empty(t.numel() + shift, dtype=dtype, device=DEV)
        pools.append(flat[shift:].view(t.shape).copy_(t))
    check(paged_attention(x.q.to(DEV), *pools, x.batch(), x.form()), x)


def test_a_cap_far_below_the_scale_is_refused() -> None:
    from microserve_b200._lib import MicroserveError

    for dtype, dh in ((F32, 32), (BF16, 64)):
        x = make(24, dtype, 2, 2, dh, 16, [30], [4], softcap=1e-38, scale=1.0)
        with pytest.raises(MicroserveError, match="too small"):
            run(x)
        x.softcap = 1e-20  # still a cap: scores of +-1e-20, every key alike
        check(run(x), x)


def test_calls_on_two_streams_at_once() -> None:
    """Many sequences in order of their length, a long context in ranges, and a model's forward (other
    tensor-core kernels) side by side."""
    from microserve_b200.attention import paged_attention
    from microserve_b200.batching import build_paged_batch
    from microserve_b200.cache import PagedKVCache
    from microserve_b200.config import CacheConfig, ModelConfig
    from microserve_b200.model import Transformer

    rng = np.random.default_rng(0)
    xs = [make(25, BF16, 8, 4, 64, 16, rng.integers(1, 300, 130).tolist(), rng.integers(17, 33, 130).tolist(), tree=True),
          make(26, BF16, 16, 2, 128, 16, [3000, 40], [30, 16], tree=True),
          make(27, BF16, 8, 8, 64, 16, rng.integers(1, 300, 90).tolist(), [1] * 90, softcap=20.0)]
    wants = [reference(x) for x in xs]
    held = [(x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), x.batch(), x.form()) for x in xs]
    model = Transformer(ModelConfig(vocab_size=512, n_layers=2, d_model=512, n_heads=8, n_kv_heads=4, max_seq_len=256,
                                    dtype="bfloat16"), DEV, seed=1)
    cache = PagedKVCache(model.cfg, CacheConfig(16, 64, "bfloat16"), DEV)
    prompts = [rng.integers(0, 512, 200).tolist() for _ in range(3)]
    batch = build_paged_batch(cache, [0, 1, 2], prompts, [0, 0, 0])
    logits = model.forward_paged(batch, cache).clone()
    streams = [torch.cuda.Stream() for _ in range(4)]
    torch.cuda.synchronize()
    results = []
    for _ in range(6):
        for s, h in zip(streams, held):
            with torch.cuda.stream(s):
                results.append(paged_attention(*h))
        with torch.cuda.stream(streams[3]):
            again = model.forward_paged(batch, cache)
    torch.cuda.synchronize()
    # (split sums of the projections are added in no fixed order: two passes alone differ too; each
    # is within 2e-2 of its scale of the float32 model's, so they are within twice that)
    assert float((again - logits).abs().max()) <= 4e-2 * max(1.0, float(logits.abs().max()))
    for i, got in enumerate(results):
        assert torch.equal(got, results[i % 3])
    for got, x, want in zip(results, xs, wants):
        check(got, x, want)


@pytest.mark.parametrize("nodes", [1, 20])
def test_a_captured_batch_takes_other_lengths(nodes) -> None:
    """A graph of an ordered call, replayed with shorter contexts: nothing of the capture's lengths stays."""
    from microserve_b200.attention import paged_attention

    rng = np.random.default_rng(1)
    n = 160
    x = make(28, BF16, 8, 4, 64, 16, rng.integers(200, 400, n).tolist(), [nodes] * n)
    q, k, v, batch, form = x.q.to(DEV), x.k.to(DEV), x.v.to(DEV), x.batch(), x.form()
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        paged_attention(q, k, v, batch, form, out)
    g.replay()
    check(out, x)
    x.context = [int(c) for c in rng.integers(nodes, 200, n)]
    x.positions = np.concatenate([np.arange(c - nodes, c) for c in x.context]).astype(np.int32)
    batch.context_lens.copy_(torch.tensor(x.context, dtype=torch.int32))
    batch.positions.copy_(torch.from_numpy(x.positions))
    g.replay()
    check(out, x)


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dh,hq,bs", [(64, 32, 16), (128, 32, 64), (64, 48, 8)])
@pytest.mark.parametrize("tree", [False, True])
def test_many_sequences_of_few_tokens(tree, dh, hq, bs, form) -> None:
    """More sequences and kv heads than run at once, of up to 64 rows a sequence and kv head."""
    rng = np.random.default_rng(2)
    n = 45
    q_lens = [int(t) for t in rng.integers(0, 64 // (hq // 8) + 1, n)]
    q_lens[:3] = [64 // (hq // 8), 1, 64 // (hq // 8)]
    cached = rng.integers(0, 150, n).tolist()
    x = make(30, BF16, hq, 8, dh, bs, cached, q_lens, tree=tree, **FORMS[form])
    check(run(x), x)


@pytest.mark.parametrize("value", [float("inf"), float("nan"), 3.3e38])
@pytest.mark.parametrize("dh", [64, 128])
@pytest.mark.parametrize("tree", [False, True])
def test_many_sequences_of_which_some_hold_anything(tree, dh, value) -> None:
    """What a row does not see, or sees, beside many others: as for few sequences."""
    n = 40
    x = make(31, BF16, 32, 8, dh, 16, [37, 5] * (n // 2), [9, 14] * (n // 2), tree=tree, prefix=[3, 0] * (n // 2))
    page, at = x.tables[4, (37 + 2) // 16], (37 + 2) % 16  # the third of the pass's own tokens
    x.v[page, :, at, 5] = value
    x.k[page, :, at] = value
    own = [r for r in range(int(x.q_start[4]), int(x.q_start[5]))
           if 37 + 2 in visible(x, 4, r - int(x.q_start[4]))[0]]
    got = run(x).double().cpu()
    ref, tol = reference(x)
    keep = torch.ones(len(ref), dtype=torch.bool)
    keep[own] = False
    assert own and len(own) < 9 and bool(((got - ref).abs() <= tol)[keep].all())
    # a key alone is as other sequences' are: only its value is out of the ordinary
    x.k[page, :, at] = 0.25
    got, (ref, tol) = run(x).double().cpu(), reference(x)
    rest = [d for d in range(dh) if d != 5]
    assert bool(((got - ref).abs() <= tol)[:, :, rest].all())
    if not np.isfinite(value):
        assert torch.equal(got[own][:, :, 5].isfinite(), ref[own][:, :, 5].isfinite())
        assert torch.equal(got[own][:, :, 5].isnan(), ref[own][:, :, 5].isnan())


@pytest.mark.parametrize("dh", [64, 128])
def test_many_sequences_that_see_nothing(dh) -> None:
    n = 44
    x = make(32, BF16, 32, 8, dh, 16, [0, 20] * (n // 2), [7, 12] * (n // 2), tree=True)
    x.masks[:] = False
    x.window = 5  # of the cached keys only the last few remain
    x.positions += 100  # (and those are out of the window)
    got = run(x)
    assert not bool(got.any())
    check(got, x)


@pytest.mark.parametrize("dtype,hq,hkv,dh,n,cached", [
    (F32, 4, 2, 32, 3, [40, 900]), (BF16, 8, 2, 64, 1, [40, 2000]), (BF16, 16, 2, 128, 9, [40, 3000]),
    (BF16, 16, 2, 64, 16, [40, 90]), (BF16, 16, 2, 128, 40, [40, 2500]), (BF16, 16, 8, 64, 17, [30] * 40)])
@pytest.mark.parametrize("tree", [False, True])
def test_padded_batches(tree, dtype, hq, hkv, dh, n, cached) -> None:
    """Rows behind the last sequence keep what they held; sequences without tokens, whose tables hold no
    block at all, do nothing; nor is any of it read."""
    from microserve_b200.attention import paged_attention

    x = make(33, dtype, hq, hkv, dh, 16, cached, [n] * len(cached), tree=tree, alibi=True)
    B, T, extra = len(cached), n * len(cached), 21
    b, form = x.batch(), x.form()
    behind = lambda t, count, value: torch.cat([t, torch.full((count, *t.shape[1:]), value, dtype=t.dtype, device=DEV)])  # noqa: E731
    b.positions = behind(b.positions, extra, -(1 << 31))
    b.input_ids, b.slot_mapping = behind(b.input_ids, extra, -1), behind(b.slot_mapping, extra, -1)
    b.q_start = behind(b.q_start, 2, T)
    b.q_lens, b.context_lens = behind(b.q_lens, 2, 0), behind(b.context_lens, 2, 0)
    b.block_tables = behind(b.block_tables, 2, -1)
    b.n_tokens = T + extra
    if tree:
        form.tree_mask = behind(form.tree_mask, extra, -1)
    q = behind(x.q.to(DEV), extra, float("nan"))
    out = torch.full_like(q, 7.0)
    paged_attention(q, x.k.to(DEV), x.v.to(DEV), b, form, out)
    assert bool((out[T:] == 7).all())
    check(out[:T], x)


@pytest.mark.parametrize("dtype,hq,hkv,dh", [(F32, 2, 1, 32), (BF16, 4, 1, 64), (BF16, 2, 2, 128)])
def test_the_largest_tree(dtype, hq, hkv, dh) -> None:
    x = make(34, dtype, hq, hkv, dh, 16, [33, 500], [1024, 3], tree=True, alibi=True, window=300)
    check(run(x), x)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n", [1, 30, 200])
def test_prefixes_of_any_length(dtype, n) -> None:
    """Longer than the context, and below zero: as the whole context, and as none."""
    x = make(35, dtype, 4, 2, 64, 16, [50, 50, 50, 0], [n] * 4, prefix=[10 ** 9, -3, 51, n + 1], window=7)
    check(run(x), x)

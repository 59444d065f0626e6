"""The operators of tree speculation and of other score forms over the paged cache, as cases to be measured.

Four operators:

* ``attention`` over one layer's paged keys and values, with a tree of drafted tokens behind each cached context
  (each node sees the context, its ancestors and itself) or with causal queries, and with any of: scores capped
  by a tanh, a bias that falls with the distance, a sliding window, a prefix that every query sees;
* ``copy`` -- pages of every layer copied to others (a fork's own pages, a pool made compact);
* ``move`` -- tokens of every layer moved inside their sequences (the accepted path of a tree made contiguous);
* ``accept`` -- the walk down each tree along the target's tokens, with what it emits and the moves it leaves.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through the package.
"""

import numpy as np
import torch

own = False

# ---------------------------------------------------------------------------------------------- cases


def _attention(name, requests, cached, q, heads, dh, block, dtype, tree, softcap=0.0, alibi=False, window=0,
               prefix=False):
    case = dict(op="attention", requests=requests, cached_lo=cached[0], cached_hi=cached[1], q_lo=q[0], q_hi=q[1],
                hq=heads[0], hkv=heads[1], dh=dh, block=block, dtype=dtype, tree=tree, softcap=softcap, alibi=alibi,
                window=window, prefix=prefix)
    return dict(case, name=name) if name else case


def listed():
    return [
        # the character-level model with a small tree for each of 8 requests: launch latency
        _attention("tree_char_f32", 8, (20, 90), (7, 7), (4, 4), 32, 16, "float32", True),
        # one user of the 8B shape with a long context: few rows, a long axis
        _attention("tree_single_long", 1, (32751, 32751), (16, 16), (32, 8), 128, 16, "bfloat16", True),
        # the verify pass of the default workload with trees of 8 tokens instead of chains of 5
        _attention("tree_verify_1b", 256, (512, 2048), (8, 8), (32, 4), 64, 16, "bfloat16", True),
        # wide ragged trees of the 8B shape: as much arithmetic as traffic
        _attention("tree_verify_8b_wide", 64, (1001, 4090), (33, 61), (32, 8), 128, 16, "bfloat16", True),
        # one request decoding alone with a distance bias: launch latency
        _attention("decode_single_alibi", 1, (332, 332), (1, 1), (32, 4), 64, 16, "bfloat16", False, alibi=True),
        # a decode step of long contexts through a capped layer with a sliding window
        _attention("decode_window_capped", 128, (700, 8191), (1, 1), (32, 8), 128, 16, "bfloat16", False, softcap=50.0,
                   window=2048),
        # prompts of the 8B shape through a capped layer, a prefix of each seen by all its tokens: the largest
        _attention("prompts_prefix_capped", 4, (0, 0), (1111, 4096), (32, 8), 128, 16, "bfloat16", False, softcap=30.0,
                   prefix=True),
        # a fork that is about to append takes its own last page, 22 layers of the 1.1B shape: latency
        dict(name="fork_one_page", op="copy", pairs=1, blocks=2048, layers=22, hkv=4, dh=64, block=16, dtype="bfloat16"),
        # a pool made compact: pages from its upper end to free places below
        dict(name="compact_pool", op="copy", pairs=4001, blocks=10000, layers=22, hkv=4, dh=64, block=16,
             dtype="bfloat16"),
        # accepted paths of a batch made contiguous, 8B shape (what lies before the paths is not touched: short)
        dict(name="keep_paths_8b", op="move", requests=192, cached_lo=40, cached_hi=150, nodes=31, accept=5, layers=32,
             hkv=8, dh=128, block=16, dtype="bfloat16"),
        # the walk of the character-level model's small trees: launch latency
        dict(name="accept_char", op="accept", requests=8, nodes=7, accept=4, vocab=65, block=16),
        # the walk of a full batch of the 8B shape over the target's logits
        dict(name="accept_8b", op="accept", requests=192, nodes=16, accept=5, vocab=128256, block=16),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["attention"] * 5 + ["copy", "move", "accept"])
    if op == "accept":
        vocab = _log_int(rng, 65, 131072)
        nodes = _log_int(rng, 1, 64)
        requests = min(_log_int(rng, 1, 256), max(1, 192 * 16 * 128256 // (nodes * vocab)))
        return dict(op=op, requests=requests, nodes=nodes, accept=rng.choice([1, 2, 4, 5, 9]), vocab=vocab,
                    block=rng.choice([8, 16, 32, 64]))
    if op != "attention":
        f32 = rng.random() < 0.2
        layers, hkv = rng.choice([2, 4, 16, 22, 32]), rng.choice([1, 2, 4, 8])
        dh, block = rng.choice([8, 16, 32, 64] if f32 else [32, 64, 128]), rng.choice([8, 16, 32, 64])
        shape = dict(layers=layers, hkv=hkv, dh=dh, block=block, dtype="float32" if f32 else "bfloat16")
        token = layers * hkv * dh * (4 if f32 else 2)
        most = 10000 * 16 * 22 * 4 * 64 * 2 // token  # tokens of the largest listed pool
        if op == "copy":
            blocks = max(2, min(_log_int(rng, 2, 20000), most // block))
            pairs = min(_log_int(rng, 1, 4001), blocks // 2, 4001 * 16 * 22 * 4 * 64 * 2 // (block * token))
            return dict(op=op, pairs=max(1, pairs), blocks=blocks, **shape)
        nodes, cached = _log_int(rng, 1, 64), _log_int(rng, 1, 900)
        requests = max(1, min(_log_int(rng, 1, 256), most // (2 * (cached + nodes + block))))
        return dict(op=op, requests=requests, cached_lo=(cached + 1) // 2, cached_hi=cached, nodes=nodes,
                    accept=rng.choice([1, 2, 4, 5, 9]), **shape)
    f32 = rng.random() < 0.15
    if f32:  # the small models
        (hq, hkv), dh = rng.choice([(4, 4), (4, 2), (8, 1), (6, 2)]), rng.choice([8, 16, 32, 64])
        requests, cached = _log_int(rng, 1, 64), _log_int(rng, 1, 1024) - 1
    else:
        (hq, hkv), dh = rng.choice([(32, 4), (32, 8), (16, 16), (12, 4), (8, 1)]), rng.choice([64, 128])
        requests, cached = _log_int(rng, 1, 256), _log_int(rng, 1, 32768) - 1
    kind = rng.choice(["tree", "tree", "decode", "prompt"])
    q = _log_int(rng, 2, 96) if kind == "tree" else 1 if kind == "decode" else _log_int(rng, 2, 512 if f32 else 4096)
    if kind == "prompt":
        requests, cached = min(requests, 8), rng.choice([0, cached])
    # keys and scores in all, as the plain form pads them: at most those of the largest cases
    requests = max(1, min(requests, 80 * 8192 * 8 * 128 // ((cached + q) * hkv * dh)))
    requests = max(1, min(requests, 4 * 4096 * 4096 * 32 // (q * (cached + q) * hq)))
    while requests * q * (cached + q) * hq > 4 * 4096 * 4096 * 32:
        cached //= 2
    return _attention("", requests, (cached // rng.choice([1, 2, 4]), cached), (max(1, q // rng.choice([1, 2])), q),
                      (hq, hkv), dh, rng.choice([8, 16, 32, 64]), "float32" if f32 else "bfloat16", kind == "tree",
                      softcap=rng.choice([0.0, 0.0, 30.0, 50.0]), alibi=rng.random() < 0.4,
                      window=rng.choice([0, 0, 7, 129, 1024]), prefix=kind == "prompt" and rng.random() < 0.5)


# ------------------------------------------------------------------------------------- lengths and trees


def _spread(n, lo, hi, salt):
    """n lengths from lo to hi, the first of them hi; the same for every seed."""
    lens = np.random.RandomState(salt).randint(lo, hi + 1, n)
    lens[0] = hi
    return lens


def _trees(lens, salt):
    """Parents inside each tree (-1: the root, node 0), breadth first with two to four children a node, and depths."""
    r = np.random.RandomState(salt)
    parents, depths = [], []
    for n in lens:
        p, d = np.full(n, -1), np.zeros(n, np.int64)
        for i in range(1, n):
            p[i] = r.randint((i - 1) // 4, (i - 1) // 2 + 1)
            d[i] = d[p[i]] + 1
        parents.append(p)
        depths.append(d)
    return parents, depths


def _shapes(case):
    """Query lengths, cached lengths, prefix lengths and the trees' parents and depths of an attention case."""
    n = case["requests"]
    q = _spread(n, case["q_lo"], case["q_hi"], n)
    cached = _spread(n, case["cached_lo"], case["cached_hi"], n + 1)
    prefix = (cached + q) * (1 + np.arange(n) % 4) // 8 if case["prefix"] else np.zeros(n, np.int64)
    parents, depths = _trees(q, n + 2) if case["tree"] else (None, [np.arange(k) for k in q])
    return q, cached, prefix, parents, depths


# --------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _i32(v):
    return torch.from_numpy(np.ascontiguousarray(v).astype(np.int32)).cuda()


def _pages(context, block, g, spare=3):
    """A pool's block count and tables whose pages lie in it in any order."""
    need = -(-context // block)
    total = int(need.sum())
    order = torch.randperm(total + spare, generator=g, device="cuda")[:total].to(torch.int32)
    start = torch.from_numpy(np.cumsum(need) - need).cuda()
    col = torch.arange(int(need.max()), device="cuda")
    held = col < torch.from_numpy(need).cuda().unsqueeze(1)
    tables = torch.where(held, order[(start.unsqueeze(1) + col).clamp(max=total - 1)], 0)
    return total + spare, tables.contiguous()


def _batch(q, cached, depths, block, g, vocab=32000):
    """The arrays of a paged pass: q[b] tokens behind cached[b] ones."""
    context = cached + q
    blocks, tables = _pages(context, block, g)
    q_start = np.concatenate([[0], np.cumsum(q)])
    seq = np.repeat(np.arange(len(q)), q)
    at = _i32(np.arange(q.sum()) - q_start[seq] + cached[seq]).long()
    rows = torch.from_numpy(seq).cuda()
    slots = tables[rows, at // block] * block + (at % block).to(torch.int32)
    ids = torch.randint(0, vocab, (int(q.sum()),), generator=g, device="cuda", dtype=torch.int32)
    return blocks, {
        "ids": ids, "positions": _i32(np.concatenate([c + d for c, d in zip(cached, depths)])),
        "slots": slots.contiguous(), "q_start": _i32(q_start), "context": _i32(context), "q_lens": _i32(q),
        "tables": tables, "max_q": int(q.max()), "tokens": int(q.sum()), "max_context": int(context.max()),
    }


def _ancestor_words(parents, width):
    """Bit i % 32 of word i / 32 of a node: it sees node i of its tree (its ancestors and itself)."""
    words = np.zeros((sum(len(p) for p in parents), width), np.uint32)
    at = 0
    for p in parents:
        for i, up in enumerate(p):
            if up >= 0:
                words[at + i] = words[at + up]
            words[at + i, i // 32] |= np.uint32(1 << i % 32)
        at += len(p)
    return torch.from_numpy(words.view(np.int32)).cuda()


def _prepare_attention(case, seed):
    g = _generator(seed)
    dt = getattr(torch, case["dtype"])
    q, cached, prefix, parents, depths = _shapes(case)
    hq, hkv, dh, block = case["hq"], case["hkv"], case["dh"], case["block"]
    blocks, s = _batch(q, cached, depths, block, g)
    draw_ = lambda *shape: torch.randn(shape, generator=g, device="cuda").to(dt)  # noqa: E731
    s |= {
        "op": "attention", "softcap": case["softcap"], "window": case["window"],
        # queries come as the first columns of the fused q | k | v projection
        "qkv": draw_(s["tokens"], (hq + 2 * hkv) * dh) * 2, "hq": hq, "dh": dh,
        "k": draw_(blocks, hkv, block, dh), "v": draw_(blocks, hkv, block, dh),
        "slopes": 2.0 ** (-8.0 * torch.arange(1, hq + 1, device="cuda") / hq) if case["alibi"] else None,
        "prefix": _i32(prefix) if case["prefix"] else None,
        "mask": _ancestor_words(parents, -(-int(q.max()) // 32)) if case["tree"] else None,
    }
    return s


def _pool(case, blocks, g):
    # page by page of one random layer: a whole pool of random numbers takes too long to make
    shape = (blocks, case["hkv"], case["block"], case["dh"])
    dt = getattr(torch, case["dtype"])
    pool = torch.empty((2, case["layers"], *shape), dtype=dt, device="cuda")
    one = torch.randn(shape, generator=g, device="cuda").to(dt)
    for i in range(2 * case["layers"]):
        pool[i % 2, i // 2] = one * (1 + i)
    return pool


def _prepare_copy(case, seed):
    g = _generator(seed)
    at = torch.randperm(case["blocks"], generator=g, device="cuda").to(torch.int32)
    src, dst = at[: case["pairs"]].contiguous(), at[case["pairs"] : 2 * case["pairs"]].contiguous()
    return {"op": "copy", "pool": _pool(case, case["blocks"], g), "src": src, "dst": dst}


def _paths(parents, accept, seed):
    """For each tree a path from a child of its root downwards, of 0 to `accept` nodes."""
    r = np.random.RandomState(seed % (1 << 31))
    paths = np.full((len(parents), accept), -1)
    for b, p in enumerate(parents):
        at = 0
        for k in range(b % (accept + 1)):
            children = np.flatnonzero(p == at)
            if not len(children):
                break
            at = paths[b, k] = r.choice(children)
    return paths


def _prepare_move(case, seed):
    g = _generator(seed)
    n = case["requests"]
    cached = _spread(n, case["cached_lo"], case["cached_hi"], n + 1)
    parents, _ = _trees(np.full(n, case["nodes"]), n + 2)
    blocks, tables = _pages(cached + case["nodes"], case["block"], g)
    paths = torch.from_numpy(_paths(parents, case["accept"], seed)).cuda()
    base = torch.from_numpy(cached).cuda().unsqueeze(1)

    def slots(at):
        return tables.gather(1, at // case["block"]) * case["block"] + (at % case["block"]).to(torch.int32)

    to = (1 + torch.arange(case["accept"], device="cuda")).expand_as(paths)
    src = torch.where(paths >= 0, slots(base + paths.clamp(min=0)), -1)
    dst = torch.where(paths >= 0, slots(base + torch.where(paths >= 0, to, 0)), -1)
    return {"op": "move", "pool": _pool(case, blocks, g), "src": src.to(torch.int32).contiguous(),
            "dst": dst.to(torch.int32).contiguous()}


def _prepare_accept(case, seed):
    g = _generator(seed)
    n, V, N = case["requests"], case["vocab"], case["nodes"]
    q, cached = np.full(n, N), _spread(n, 1, 900, n + 1)
    parents, depths = _trees(q, n + 2)
    _, s = _batch(q, cached, depths, case["block"], g, V)
    logits = torch.randn((n * N, V), generator=g, device="cuda") * 3.0
    # the target agrees with the draft along a path of each tree
    paths = _paths(parents, case["accept"], seed)
    b, k = np.nonzero(paths >= 0)
    before = np.where(k > 0, paths[b, k - 1], 0)
    rows, nodes = (torch.from_numpy(b * N + i).cuda() for i in (before, paths[b, k]))
    logits[rows, s["ids"][nodes].long()] = 30.0
    return s | {"op": "accept", "logits": logits, "parents": _i32(np.concatenate(parents)), "accept": case["accept"],
                "block": case["block"]}


def prepare(case, seed):
    return {"attention": _prepare_attention, "copy": _prepare_copy, "move": _prepare_move,
            "accept": _prepare_accept}[case["op"]](case, seed)


# ------------------------------------------------------------------------------------------------ run


def _unpack_bits(words):
    bits = (words.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1
    return bits.flatten(1).bool()


def _plain_attention(s):
    B, S, Q, hq, dh, T = s["context"].numel(), s["max_context"], s["max_q"], s["hq"], s["dh"], s["tokens"]
    _, hkv, block, _ = s["k"].shape
    dev = s["k"].device
    q_start, q_lens, context = s["q_start"].long(), s["q_lens"].long(), s["context"].long()
    # queries and their positions, padded to (B, Q)
    row = (q_start[:-1].unsqueeze(1) + torch.arange(Q, device=dev)).clamp(max=T - 1)
    live = torch.arange(Q, device=dev) < q_lens.unsqueeze(1)
    q = s["qkv"][:, : hq * dh].float()[row].view(B, Q, hkv, hq // hkv, dh)
    at = s["positions"].long()[row]
    # keys and values of each sequence in order: (B, S, hkv, dh)
    j = torch.arange(S, device=dev)
    page = s["tables"].long()[:, j // block]
    k, v = (t[page, :, j % block].float() for t in (s["k"], s["v"]))
    base = (context - q_lens).unsqueeze(1)
    node = (j - base).clamp(min=0)  # of a key behind the cached context
    drafted = j >= base
    key_at = torch.where(drafted, at.gather(1, node.clamp(max=Q - 1)), j) if s["mask"] is not None else j.expand(B, S)
    distance = at.unsqueeze(2) - key_at.unsqueeze(1)  # (B, Q, S)
    seen = distance >= 0
    if s["mask"] is not None:
        bits = _unpack_bits(s["mask"])[row]
        seen = torch.where(drafted.unsqueeze(1), bits.gather(2, node.clamp(max=bits.shape[2] - 1).unsqueeze(1)
                                                             .expand(B, Q, S)), True)
    if s["window"]:
        seen = seen & (distance < s["window"])
    if s["prefix"] is not None:
        seen = seen | (j < s["prefix"].unsqueeze(1)).unsqueeze(1)
    seen = (seen & (j < context.unsqueeze(1)).unsqueeze(1)).unsqueeze(1).unsqueeze(1)
    x = torch.einsum("bqhgd,bshd->bhgqs", q, k) * dh ** -0.5
    if s["softcap"]:
        x = s["softcap"] * torch.tanh(x / s["softcap"])
    if s["slopes"] is not None:
        x = x - s["slopes"].view(1, hkv, -1, 1, 1) * distance.abs().unsqueeze(1).unsqueeze(1)
    x = torch.where(seen, x, float("-inf"))
    p = torch.exp(x - x.amax(-1, keepdim=True).clamp(min=-3e38))
    del x
    total = p.sum(-1).clamp(min=1e-38)
    out = torch.einsum("bhgqs,bshd->bhgqd", p, v) / total.unsqueeze(-1)
    return out.permute(0, 3, 1, 2, 4).reshape(B, Q, hq, dh)[live].to(s["qkv"].dtype)


def _plain_copy(s):
    pool = s["pool"]
    pool[:, :, s["dst"].long()] = pool[:, :, s["src"].long()]
    return pool


def _plain_move(s):
    pool = s["pool"]
    block = pool.shape[4]
    moved = (s["src"] >= 0) & (s["src"] != s["dst"])
    src, dst = s["src"][moved].long(), s["dst"][moved].long()
    pool[:, :, dst // block, :, dst % block] = pool[:, :, src // block, :, src % block]
    return pool


def _plain_accept(s):
    B, Q, D, dev = s["context"].numel(), s["max_q"], s["accept"], s["logits"].device
    row = s["q_start"][:-1].long().unsqueeze(1) + torch.arange(Q, device=dev)
    target = s["logits"].argmax(-1)[row]
    tokens, parents = s["ids"].long()[row], s["parents"].long()[row]
    i = torch.arange(Q, device=dev)
    at = torch.zeros((B, 1), dtype=torch.long, device=dev)
    going = torch.ones((B, 1), dtype=torch.bool, device=dev)
    said, nodes = [target[:, :1]], []
    for _ in range(D):
        fits = (parents == at) & (tokens == target.gather(1, at)) & going
        first = torch.where(fits, i, Q).amin(1, keepdim=True)
        going = first < Q
        at = torch.where(going, first, at)
        nodes.append(torch.where(going, at, -1))
        said.append(torch.where(going, target.gather(1, at), -1))
    nodes = torch.cat(nodes, 1)
    base = (s["context"] - s["q_lens"]).long().unsqueeze(1)
    slot = lambda p: s["tables"].gather(1, p // s["block"]) * s["block"] + p % s["block"]  # noqa: E731
    src = torch.where(nodes >= 0, slot(base + nodes.clamp(min=0)), -1)
    to = torch.where(nodes >= 0, 1 + torch.arange(D, device=dev), 0)
    dst = torch.where(nodes >= 0, slot(base + to), -1)
    return [t.to(torch.int32) for t in (torch.cat(said, 1), (nodes >= 0).sum(1), nodes, src, dst)]


def _own_batch(s):
    from microserve_b200.model import PagedBatch

    return PagedBatch(input_ids=s["ids"], positions=s["positions"], slot_mapping=s["slots"], block_tables=s["tables"],
                      context_lens=s["context"], q_lens=s["q_lens"], q_start=s["q_start"], max_q=s["max_q"],
                      n_tokens=s["tokens"], max_context=s["max_context"])


def _own_attention(s):
    from microserve_b200.attention import AttentionForm, paged_attention

    form = AttentionForm(softcap=s["softcap"], slopes=s["slopes"], window=s["window"], prefix_lens=s["prefix"],
                         tree_mask=s["mask"])
    q = s["qkv"][:, : s["hq"] * s["dh"]].view(s["tokens"], s["hq"], s["dh"])
    return paged_attention(q, s["k"], s["v"], _own_batch(s), form)


def _own_copy(s):
    from microserve_b200.cache import copy_blocks

    copy_blocks(s["pool"], s["src"], s["dst"])
    return s["pool"]


def _own_move(s):
    from microserve_b200.cache import move_tokens

    move_tokens(s["pool"], s["src"], s["dst"])
    return s["pool"]


def _own_accept(s):
    from microserve_b200.tree import accept_trees

    a = accept_trees(s["logits"], _own_batch(s), s["parents"], s["accept"], s["block"])
    return [a.tokens, a.num_accepted, a.nodes, a.src_slots, a.dst_slots]


def run(state):
    if own:
        return {"attention": _own_attention, "copy": _own_copy, "move": _own_move,
                "accept": _own_accept}[state["op"]](state)
    return {"attention": _plain_attention, "copy": _plain_copy, "move": _plain_move,
            "accept": _plain_accept}[state["op"]](state)


# ----------------------------------------------------------------------------------------------- work


def work(case):
    if case["op"] == "accept":
        parents, _ = _trees(np.full(case["requests"], case["nodes"]), case["requests"] + 2)
        rows = case["requests"] + (_paths(parents, case["accept"], 0) >= 0).sum()  # the rows on the paths
        return {"bytes": float(rows * case["vocab"] * 4 + case["requests"] * case["nodes"] * 8), "flops": 0}
    wide = 4 if case["dtype"] == "float32" else 2
    if case["op"] != "attention":
        token = 2 * case["layers"] * case["hkv"] * case["dh"] * wide
        if case["op"] == "copy":
            return {"bytes": float(2 * case["pairs"] * case["block"] * token), "flops": 0}
        parents, _ = _trees(np.full(case["requests"], case["nodes"]), case["requests"] + 2)
        paths = _paths(parents, case["accept"], 0)
        moved = ((paths >= 0) & (paths != 1 + np.arange(case["accept"]))).sum()
        return {"bytes": float(2 * moved * token + 8 * paths.size), "flops": 0}
    q, cached, prefix, _, depths = _shapes(case)
    keys = pairs = 0
    for n, c, f, d in zip(q, cached, prefix, depths):
        w = case["window"] or c + n
        low = np.maximum(0, c + d + 1 - w)  # the first key in a query's window
        last = c + d + 1  # context, ancestors and itself: one key at each position up to the query's own
        seen = last - low
        pairs += (seen + np.maximum(0, np.minimum(f, low)) + np.maximum(0, f - last)).sum()
        keys += c + n - max(0, min(low.min(), c) - min(f, low.min()))
    T = int(q.sum())
    total = keys * 2 * case["hkv"] * case["dh"] * wide + 2 * T * case["hq"] * case["dh"] * wide
    if case["tree"]:
        total += T * 4 * -(-int(q.max()) // 32)
    return {"bytes": float(total), "flops": float(4 * pairs * case["hq"] * case["dh"])}


# ---------------------------------------------------------------------------------------------- exact


def _exact_attention(case, s):
    q, cached, prefix, parents, depths = _shapes(case)
    hq, hkv, dh, block, group = case["hq"], case["hkv"], case["dh"], case["block"], case["hq"] // case["hkv"]
    if 4 * hq * dh * sum((c + n) * n for c, n in zip(cached, q)) > 3e13:
        return None
    out = torch.empty((int(q.sum()), hq, dh), dtype=torch.float64, device="cuda")
    start = 0
    for b, n in enumerate(q):
        n, c, f = int(n), int(cached[b]), int(prefix[b])
        at = c + torch.from_numpy(np.asarray(depths[b])).cuda()
        key_at = torch.cat([torch.arange(c, device="cuda"), at])
        if parents is None:
            sees = key_at.unsqueeze(0) <= at.unsqueeze(1)
        else:
            tree = np.eye(n, dtype=bool)
            for i in range(1, n):
                tree[i] |= tree[parents[b][i]]
            sees = torch.cat([torch.ones((n, c), dtype=torch.bool), torch.from_numpy(tree)], 1).cuda()
        away = (at.unsqueeze(1) - key_at.unsqueeze(0)).double()
        if case["window"]:
            sees = sees & (away < case["window"])
        sees[:, :f] = True
        pages = s["tables"][b, : -(-(c + n) // block)].long()
        for h in range(hkv):
            k, v = (t[pages, h].reshape(-1, dh)[: c + n].double() for t in (s["k"], s["v"]))
            for i in range(h * group, (h + 1) * group):
                x = s["qkv"][start : start + n, i * dh : (i + 1) * dh].double() @ k.t() / dh ** 0.5
                if case["softcap"]:
                    x = torch.tanh(x / case["softcap"]) * case["softcap"]
                if case["alibi"]:
                    x -= s["slopes"][i].double() * away.abs()
                x[~sees] = float("-inf")
                p = torch.softmax(x, -1)
                out[start : start + n, i] = torch.nan_to_num(p) @ v
        start += n
    return out


def exact(case, seed):
    if case["op"] == "accept":
        return None  # whole numbers: the plain form's are exact
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    before = s["pool"].clone()
    block = case["block"] if case["op"] == "move" else 1
    pairs = torch.stack([s["src"].flatten(), s["dst"].flatten()], 1).tolist()
    for src, dst in pairs:
        if src >= 0 and src != dst:
            at = lambda t, i: t[:, :, i // block, :, i % block] if case["op"] == "move" else t[:, :, i]  # noqa: E731
            at(s["pool"], dst).copy_(at(before, src))
    return s["pool"].double()

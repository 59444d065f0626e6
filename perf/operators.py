"""The operators a request sets for itself inside a shared batch, as cases to be measured.

Two operators:

* ``logits`` -- penalties for repeated tokens, per-request biases and grammar masks, over the logits of one
  draw (one row per request) or of a speculative verify pass (several rows per request, each seeing the
  proposals before it as already said);
* ``lora`` -- the low-rank adapters of many requests beside one shared projection, optionally with the
  SwiGLU that follows the gate/up projection.

``run`` computes them in elementary torch operations, or, where ``own`` is true, through the package.
"""

import numpy as np
import torch

own = False

NEG_INF = float("-inf")

# ---------------------------------------------------------------------------------------------- cases


def listed():
    return [
        # one request of the character-level model decoding alone: launch latency
        dict(name="logits_char_single", op="logits", requests=1, rows=1, vocab=65, history=48, penalties=True,
             bias=2, masked="", proposals=0, in_place=False),
        # one chat user, vocabulary of the 8B shape, everything on: latency of a long row
        dict(name="logits_single_128k", op="logits", requests=1, rows=1, vocab=128256, history=1500,
             penalties=True, bias=20, masked="most", proposals=0, in_place=False),
        # an ordinary decode step of a full batch; an odd vocabulary leaves rows unaligned
        dict(name="logits_decode_odd", op="logits", requests=203, rows=1, vocab=32003, history=900,
             penalties=True, bias=5, masked="", proposals=0, in_place=False),
        # the verify pass of the default workload: 256 requests, 4 proposals each
        dict(name="logits_verify_32k", op="logits", requests=256, rows=5, vocab=32000, history=1280,
             penalties=True, bias=0, masked="", proposals=4, in_place=False),
        # grammar-constrained decoding: masks alone, written into the logits in place
        dict(name="logits_grammar_in_place", op="logits", requests=256, rows=1, vocab=128256, history=0,
             penalties=False, bias=0, masked="most", proposals=0, in_place=True),
        # the verify pass of the 8B shape with every control on: the largest
        dict(name="logits_verify_128k", op="logits", requests=256, rows=6, vocab=128256, history=1500,
             penalties=True, bias=10, masked="half", proposals=5, in_place=False),
        # one decoding request with one adapter on the output projection: launch latency
        dict(name="lora_single_o", op="lora", requests=1, tokens=1, adapters=1, none=0, ranks="16", k=2048, n=2048,
             kind="plain", dtype="bfloat16", out="float32"),
        # the float32 character-level model, small odd ranks, a ragged batch
        dict(name="lora_char_f32", op="lora", requests=7, tokens=61, adapters=3, none=1, ranks="4,5,12", k=128, n=704,
             kind="swiglu", dtype="float32", out="float32"),
        # a decode step of the default workload: 256 requests over 64 adapters, a quarter without one, fused q|k|v
        dict(name="lora_decode_qkv", op="lora", requests=256, tokens=256, adapters=64, none=16, ranks="8,16,32,64",
             k=2048, n=2560, kind="qkv", dtype="bfloat16", out="bfloat16"),
        # the verify pass of the default workload through gate/up, with the SwiGLU
        dict(name="lora_verify_gate_up", op="lora", requests=256, tokens=1280, adapters=32, none=4, ranks="16,32", k=2048,
             n=11264, kind="swiglu", dtype="bfloat16", out="bfloat16"),
        # the 8B verify pass through the down projection, an adapter for every request: the weights are the traffic
        dict(name="lora_verify_8b_down", op="lora", requests=256, tokens=1536, adapters=256, none=0, ranks="16", k=14336,
             n=4096, kind="plain", dtype="bfloat16", out="float32"),
        # a prefill of long prompts through the 8B gate/up with large ranks: the largest
        dict(name="lora_prefill_8b_gate_up", op="lora", requests=5, tokens=8192, adapters=4, none=0, ranks="64,128",
             k=4096, n=28672, kind="swiglu", dtype="bfloat16", out="bfloat16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    if rng.random() < 0.5:
        vocab = _log_int(rng, 65, 131072)
        rows = rng.choice([1, 1, 2, 4, 5, 6, 9])
        requests = min(_log_int(rng, 1, 320), max(1, 256 * 6 * 128256 // (rows * vocab)))
        penalties = rng.random() < 0.8
        masked = rng.choice(["", "half", "most"])
        in_place = not penalties and masked != ""
        bias = rng.choice([0, 1, 7, 40]) if penalties else 0 if in_place else 7
        return dict(op="logits", requests=requests, rows=rows, vocab=vocab,
                    history=_log_int(rng, 1, 4096) if penalties else 0, penalties=penalties, bias=bias, masked=masked,
                    proposals=rows - 1 if penalties else 0, in_place=in_place)
    f32 = rng.random() < 0.15
    kind = rng.choice(["plain", "qkv", "swiglu"])
    if f32:  # the small models: any width
        k = _log_int(rng, 32, 512)
        n = 16 * _log_int(rng, 3, 64) if kind != "plain" else _log_int(rng, 32, 700)
        tokens = _log_int(rng, 1, 400)
    else:
        k = 64 * _log_int(rng, 2, 224)
        n = 128 * _log_int(rng, 1, 200)
        tokens = min(_log_int(rng, 1, 8192), max(1, 8192 * 28672 // n))
    if kind == "qkv":
        n = max(n // 96 * 96, 96)
    case = dict(op="lora", requests=0, tokens=tokens, adapters=_log_int(rng, 1, 96), none=rng.choice([0, 0, 1, 9]),
                ranks=rng.choice(["8", "16", "64", "8,16,32,64", "4,20,128", "5,7"]), k=k, n=n, kind=kind,
                dtype="float32" if f32 else "bfloat16", out="float32" if f32 or kind == "plain" else "bfloat16")
    # every token against every adapter, as the plain form has it, costs at most what the largest case does
    dense = int(_ranks(case).sum()) * (len(_slice_columns(case)) * k + n)
    case["tokens"] = min(tokens, max(1, 8192 * 384 * (2 * 4096 + 28672) // dense))
    case["requests"] = min(case["tokens"], _log_int(rng, 1, 256))
    return case


# --------------------------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _words(vocab):
    return (vocab + 31) // 32


def _pack_bits(flags):
    """(n, V) truth values as (n, ceil(V / 32)) int32 words, token v at bit v % 32 of word v / 32."""
    n, vocab = flags.shape
    full = torch.zeros((n, _words(vocab) * 32), dtype=torch.int64, device=flags.device)
    full[:, :vocab] = flags
    words = (full.view(n, -1, 32) << torch.arange(32, device=flags.device)).sum(-1)
    return torch.where(words >= 1 << 31, words - (1 << 32), words).to(torch.int32)


def _prepare_logits(case, seed):
    g = _generator(seed)
    B, R, V = case["requests"], case["rows"], case["vocab"]
    dev = "cuda"
    s = {"op": "logits", "rows": R, "in_place": case["in_place"],
         "logits": torch.randn((B * R, V), generator=g, device=dev) * 3.0,
         "counts": None, "seen": None, "slots": None, "penalties": None, "bias_start": None, "bias_ids": None,
         "bias_values": None, "masks": None, "mask_rows": None, "proposals": None}
    if case["penalties"]:
        slots = torch.randperm(B + 3, generator=g, device=dev)[:B].to(torch.int32)
        H = case["history"]
        # text repeats itself: token ids crowd towards the low end of the vocabulary
        said = (torch.rand((B + 3, H), generator=g, device=dev) ** 3 * V).long().clamp(max=V - 1)
        generated = torch.arange(H, device=dev) >= H // 3  # the first third is the prompt
        counts = torch.zeros((B + 3, V), dtype=torch.int32, device=dev)
        counts.scatter_add_(1, said, generated.to(torch.int32).expand(B + 3, H).contiguous())
        seen = torch.zeros((B + 3, V), dtype=torch.bool, device=dev).scatter_(1, said, True)
        s["counts"], s["seen"], s["slots"] = counts, _pack_bits(seen), slots
        p = torch.rand((B, 3), generator=g, device=dev)
        s["penalties"] = torch.stack([1.0 + 0.5 * p[:, 0], 0.8 * p[:, 1], 0.4 * p[:, 2]], 1).contiguous()
        if case["proposals"]:
            u = torch.rand((case["proposals"], B), generator=g, device=dev)
            s["proposals"] = (u ** 3 * V).to(torch.int32).clamp(max=V - 1)
    if case["bias"]:
        n = min(case["bias"], V)
        ids = torch.rand((B, V), generator=g, device=dev).topk(n, dim=1).indices.sort(dim=1).values
        s["bias_ids"] = ids.to(torch.int32).reshape(-1).contiguous()
        s["bias_values"] = torch.randn(B * n, generator=g, device=dev) * 4.0
        s["bias_start"] = torch.arange(B + 1, dtype=torch.int32, device=dev) * n
    if case["masked"]:
        # a third as many grammar states as rows; every fifth row is free
        n = max(1, B * R // 3)
        share = 0.5 if case["masked"] == "half" else 0.02
        allowed = torch.rand((n, V), generator=g, device=dev) < share
        allowed[:, 0] = True
        s["masks"] = _pack_bits(allowed)
        rows = torch.randint(0, n, (B * R,), generator=g, device=dev, dtype=torch.int32)
        if B * R > 1:
            rows[::5] = -1
        s["mask_rows"] = rows
    return s


def _adapter_of_requests(case):
    """Adapter id (-1: none) of each request: every adapter is in use when there are enough requests."""
    n = case["adapters"] + case["none"]
    i = np.arange(case["requests"]) * 7 + 3 if n % 7 else np.arange(case["requests"]) * 5 + 3
    a = i % n
    return np.where(a < case["adapters"], a, -1)


def _tokens_of_requests(case):
    """Ragged token counts, at least one each, that sum to ``tokens``."""
    w = np.arange(case["requests"]) % 3 + 1.0
    if case["tokens"] % case["requests"] == 0 and case["tokens"] < 8 * case["requests"]:
        w[:] = 1.0  # a verify pass: the same few rows for every request
    lens = 1 + np.floor((case["tokens"] - case["requests"]) * w / w.sum()).astype(np.int64)
    lens[-1] += case["tokens"] - lens.sum()
    return lens


def _ranks(case):
    r = [int(x) for x in case["ranks"].split(",")]
    return np.array([r[i % len(r)] for i in range(case["adapters"])], dtype=np.int64)


def _slice_columns(case):
    n = case["n"]
    if case["kind"] == "qkv":
        return [n // 3 * 2, n // 6, n - n // 3 * 2 - n // 6]
    return [n // 2, n // 2] if case["kind"] == "swiglu" else [n]


def _prepare_lora(case, seed):
    g = _generator(seed)
    dev = "cuda"
    dt = getattr(torch, case["dtype"])
    T, K, N = case["tokens"], case["k"], case["n"]
    ranks = _ranks(case)
    R, ns = int(ranks.sum()), len(_slice_columns(case))
    offsets = np.cumsum(ranks) - ranks
    of_token = np.repeat(_adapter_of_requests(case), _tokens_of_requests(case))
    order = np.argsort(of_token, kind="stable")
    # the batch's plan: tiles of up to 64 tokens of one adapter, as positions in `order`
    ids, first = np.unique(of_token[order], return_index=True)
    lens = np.diff(np.append(first, T))
    n = -(-lens // 64)
    start = np.repeat(first, n) + 64 * (np.arange(n.sum()) - np.repeat(np.cumsum(n) - n, n))
    count = np.minimum(64, np.repeat(first + lens, n) - start)
    tiles = np.stack([start, count, np.repeat(ids, n), start * 0], 1)
    i32 = lambda v: torch.from_numpy(np.ascontiguousarray(v).astype(np.int32)).to(dev)  # noqa: E731
    alpha = torch.rand(case["adapters"], generator=g, device=dev) + 0.5
    return {
        "op": "lora", "kind": case["kind"], "out": getattr(torch, case["out"]), "slices": _slice_columns(case),
        "x": torch.randn((T, K), generator=g, device=dev).to(dt),
        "a": (torch.randn((ns * R, K), generator=g, device=dev) * K ** -0.5).to(dt),
        "b": (torch.randn((R, N), generator=g, device=dev) * 0.1).to(dt),
        "base": torch.randn((T, N), generator=g, device=dev),
        "scales": alpha, "ranks": i32(ranks), "offsets": i32(offsets),
        "max_rank": int(ranks.max()), "of_token": i32(of_token), "order": i32(order), "tiles": i32(tiles),
    }


def prepare(case, seed):
    return _prepare_logits(case, seed) if case["op"] == "logits" else _prepare_lora(case, seed)


# ------------------------------------------------------------------------------------------------ run


def _unpack_bits(words, vocab):
    bits = (words.unsqueeze(-1) >> torch.arange(32, dtype=torch.int32, device=words.device)) & 1
    return bits.reshape(words.shape[0], -1)[:, :vocab].bool()


def _plain_logits(s):
    x = s["logits"]
    rows, V = x.shape
    R = s["rows"]
    B = rows // R
    y = x.view(B, R, V)
    if s["penalties"] is not None:
        slots = s["slots"].long()
        count = s["counts"][slots].unsqueeze(1)
        seen = _unpack_bits(s["seen"][slots], V).unsqueeze(1)
        if s["proposals"] is not None:
            G = s["proposals"].shape[0]
            ids = s["proposals"].t().long().unsqueeze(1).expand(B, R, G)
            before = torch.arange(G, device=x.device) < torch.arange(R, device=x.device).unsqueeze(1)
            more = torch.zeros((B, R, V), dtype=torch.int32, device=x.device)
            more.scatter_add_(2, ids, before.to(torch.int32).expand(B, R, G))
            count = count + more
            seen = seen | (more > 0)
        rep, pres, freq = (s["penalties"][:, k].view(B, 1, 1) for k in range(3))
        y = torch.where(seen, torch.where(y > 0, y / rep, y * rep), y)
        y = y - freq * count - pres * (count > 0)
    if s["bias_ids"] is not None:
        n = s["bias_ids"].numel() // B
        bias = torch.zeros((B, V), device=x.device)
        bias.scatter_(1, s["bias_ids"].view(B, n).long(), s["bias_values"].view(B, n))
        y = y + bias.unsqueeze(1)
    if s["masks"] is not None:
        free = (s["mask_rows"] < 0).unsqueeze(1)
        allowed = _unpack_bits(s["masks"], V)[s["mask_rows"].clamp(min=0).long()]
        y = torch.where((allowed | free).view(B, R, V), y, NEG_INF)
    y = y.reshape(rows, V)
    return x.copy_(y) if s["in_place"] else y


def _plain_lora(s):
    T, N = s["base"].shape
    ranks, ns = s["ranks"].long(), len(s["slices"])
    R = s["b"].shape[0]
    of_col = torch.repeat_interleave(torch.arange(ranks.numel(), device=ranks.device), ranks, output_size=R)
    inside = torch.arange(R, device=ranks.device) - s["offsets"].long()[of_col]
    at = ns * s["offsets"].long()[of_col] + inside
    mine = s["of_token"].unsqueeze(1) == of_col
    weight = torch.where(mine, s["scales"][of_col], 0.0)
    low = s["x"].float() @ s["a"].float().t()
    low = [low[:, at + j * ranks[of_col]] * weight for j in range(ns)]
    b = s["b"].float()
    if s["kind"] == "swiglu":
        b = b.view(R, N // 16, 2, 8)
        base = s["base"].view(T, N // 16, 2, 8)
        gate = base[:, :, 0].reshape(T, -1) + low[0] @ b[:, :, 0].reshape(R, -1)
        up = base[:, :, 1].reshape(T, -1) + low[1] @ b[:, :, 1].reshape(R, -1)
        return (gate / (1.0 + torch.exp(-gate)) * up).to(s["out"])
    parts = [w @ c for w, c in zip(low, torch.split(b, s["slices"], 1))]
    return (s["base"] + torch.cat(parts, 1)).to(s["out"])


def _own_logits(s):
    from microserve_b200.logits import LogitControls, TokenCounts, apply_logit_controls

    counts = None if s["counts"] is None else TokenCounts(s["counts"], s["seen"])
    controls = LogitControls(slots=s["slots"], penalties=s["penalties"], bias_start=s["bias_start"],
                             bias_ids=s["bias_ids"], bias_values=s["bias_values"], masks=s["masks"],
                             mask_rows=s["mask_rows"])
    return apply_logit_controls(s["logits"], controls, counts, rows_per_request=s["rows"],
                                proposals=s["proposals"], out=s["logits"] if s["in_place"] else None)


def _own_lora(s):
    from microserve_b200.lora import LoraPlan, LoraProjection, lora_add

    proj = LoraProjection(a=s["a"], b=s["b"], offsets=s["offsets"], ranks=s["ranks"], scales=s["scales"],
                          max_rank=s["max_rank"], slices=s["slices"], interleaved=s["kind"] == "swiglu")
    plan = LoraPlan(order=s["order"], tiles=s["tiles"])
    return lora_add(s["x"], s["base"], proj, plan, swiglu=s["kind"] == "swiglu", out_dtype=s["out"])


def run(state):
    if state["op"] == "logits":
        return _own_logits(state) if own else _plain_logits(state)
    return _own_lora(state) if own else _plain_lora(state)


# ----------------------------------------------------------------------------------------------- work


def work(case):
    if case["op"] == "logits":
        B, rows, V = case["requests"], case["requests"] * case["rows"], case["vocab"]
        words = 4 * _words(V)
        masked = rows - -(-rows // 5) if rows > 1 else rows
        share = {"": 0.0, "half": 0.5, "most": 0.98}[case["masked"]]
        if case["in_place"]:  # the mask words, and a write for each token they forbid
            states = min(masked, max(1, rows // 3))
            return {"bytes": states * words + masked * V * share * 4, "flops": 0}
        total = rows * V * 8 + B * case["bias"] * 8
        if case["masked"]:
            total += min(masked, max(1, rows // 3)) * words
        if case["penalties"]:
            # ids are V * u^3: the expected number of distinct ones among `history` draws
            edge = (np.arange(V + 1) / V) ** (1 / 3)
            distinct = float((1 - (1 - np.diff(edge)) ** case["history"]).sum())
            total += B * (words + 4 * distinct + 12)
        return {"bytes": total, "flops": 0}
    T, K, N = case["tokens"], case["k"], case["n"]
    ns = len(_slice_columns(case))
    wide = 4 if case["dtype"] == "float32" else 2
    ranks, of_request, lens = _ranks(case), _adapter_of_requests(case), _tokens_of_requests(case)
    used = ranks[np.unique(of_request[of_request >= 0])].sum()
    served = of_request >= 0
    out = T * (N // 2 if case["kind"] == "swiglu" else N) * (4 if case["out"] == "float32" else 2)
    total = lens[served].sum() * K * wide + used * (ns * K + N) * wide + T * N * 4 + out + T * 4
    flops = 2 * (ranks[of_request[served]] * lens[served]).sum() * (ns * K + N)
    return {"bytes": float(total), "flops": float(flops)}


# ---------------------------------------------------------------------------------------------- exact


def exact(case, seed):
    def of_logits(s):
        V, R = case["vocab"], case["rows"]
        out = torch.empty(s["logits"].shape, dtype=torch.float64, device="cuda")
        bit = torch.arange(V, device="cuda")
        for r in range(out.shape[0]):
            b, i = divmod(r, R)
            y = s["logits"][r].double()
            if s["penalties"] is not None:
                slot = int(s["slots"][b])
                rep, pres, freq = s["penalties"][b].tolist()
                said = s["counts"][slot].double()
                seen = (s["seen"][slot][bit // 32] >> (bit % 32)) & 1
                if s["proposals"] is not None:
                    for v in s["proposals"][:i, b].tolist():
                        said[v] += 1
                        seen[v] = 1
                y = torch.where(seen == 1, torch.maximum(y, y * 0) / rep + torch.minimum(y, y * 0) * rep, y)
                y = y - said * freq - torch.sign(said) * pres
            if s["bias_ids"] is not None:
                lo, hi = s["bias_start"][b : b + 2].tolist()
                y[s["bias_ids"][lo:hi].long()] += s["bias_values"][lo:hi].double()
            if s["masks"] is not None and int(s["mask_rows"][r]) >= 0:
                word = s["masks"][int(s["mask_rows"][r])][bit // 32]
                y[((word >> (bit % 32)) & 1) == 0] = NEG_INF
            out[r] = y
        return out

    def of_lora(s):
        ranks, offsets, ns = _ranks(case), np.cumsum(_ranks(case)) - _ranks(case), len(s["slices"])
        N = case["n"]
        col = np.arange(N)
        of_col = (col // 8 % 2) if case["kind"] == "swiglu" else np.repeat(np.arange(ns), s["slices"])
        at = [torch.from_numpy(np.flatnonzero(of_col == j)).cuda() for j in range(ns)]
        y = s["base"].double()
        of_token = s["of_token"].long()
        for a in range(case["adapters"]):
            t = torch.nonzero(of_token == a).flatten()
            if t.numel() == 0:
                continue
            r, o = int(ranks[a]), int(offsets[a])
            x = s["x"][t].double()
            b = s["b"][o : o + r].double()
            for j in range(ns):
                low = x @ s["a"][ns * o + j * r : ns * o + (j + 1) * r].double().t()
                y[t.unsqueeze(1), at[j]] += s["scales"][a].double() * (low @ b[:, at[j]])
        if case["kind"] != "swiglu":
            return y
        gate, up = y[:, at[0]], y[:, at[1]]
        return gate * torch.sigmoid(gate) * up

    s = prepare(case, seed)
    return of_logits(s) if case["op"] == "logits" else of_lora(s)

"""Per-request logit controls (ms_apply_logit_controls) and the token counts they read, against
the 64-bit restatement."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import philox
from oracle.controls import control_row
from oracle.sampling import near_boundary, sample_row

pytestmark = pytest.mark.gpu

DEV = "cuda"


class Case:
    """Random controls of B requests x R rows, on the host and on the device."""

    def __init__(self, B: int, R: int, V: int, *, seed: int, penalties: bool = True, bias: int = 3,
                 masks: bool = True, gamma: int = 0, first: int = 0, spread: float = 3.0) -> None:
        from microserve_b200.logits import LogitControls, TokenCounts, pack_masks

        rng = np.random.default_rng(seed)
        self.B, self.R, self.V, self.first = B, R, V, first
        self.x = (rng.standard_normal((B * R, V)) * spread).astype(np.float32)
        n_slots = B + 2
        self.counts = np.zeros((n_slots, V), np.int32)
        self.seen = np.zeros((n_slots, V), bool)
        for s in range(n_slots):
            said = (rng.random(V // 2 + 3) ** 2 * V).astype(int)
            np.add.at(self.counts[s], said, 1)
            self.seen[s, said] = True
            self.seen[s, rng.integers(0, V, 5)] = True  # prompt only
        self.slots = rng.permutation(n_slots)[:B].astype(np.int32)
        if B > 2:
            self.slots[1] = -1  # a request without penalties
        self.pen = np.stack([rng.uniform(0.6, 1.9, B), rng.uniform(-0.5, 1.0, B),
                             rng.uniform(-0.2, 0.7, B)], 1).astype(np.float32)
        self.props = rng.integers(0, V, (gamma, B)).astype(np.int32)
        if gamma > 1:
            self.props[1] = self.props[0]  # the same token twice in a round
        self.bias = [{int(v): float(np.float32(rng.standard_normal() * 5))
                      for v in np.unique(rng.integers(0, V, bias))} if b % 3 else {} for b in range(B)]
        if gamma and bias:
            self.bias[0] = {int(self.props[0, 0]): 1.5}
        self.allowed = rng.random((B + 1, V)) < 0.3
        self.allowed[B] = False  # allows nothing
        self.mask_rows = rng.integers(-1, B, B * R).astype(np.int32)
        if B * R > 1:
            self.mask_rows[-1] = B
        self.penalties, self.masks, self.biased = penalties, masks, bias > 0
        t = lambda a: torch.from_numpy(np.ascontiguousarray(a)).to(DEV)  # noqa: E731
        self.tc = TokenCounts(t(self.counts), t(pack_masks(self.seen)))
        ids = [sorted(d) for d in self.bias]
        start = np.cumsum([0] + [len(i) for i in ids]).astype(np.int32)
        flat = np.array([v for i in ids for v in i], np.int32)
        vals = np.array([d[v] for d, i in zip(self.bias, ids) for v in i], np.float32)
        self.controls = LogitControls(
            slots=t(self.slots) if penalties else None, penalties=t(self.pen) if penalties else None,
            bias_start=t(start) if bias else None, bias_ids=t(flat) if bias else None,
            bias_values=t(vals) if bias else None, masks=t(pack_masks(self.allowed)) if masks else None,
            mask_rows=t(self.mask_rows) if masks else None)
        self.dprops = t(self.props) if gamma else None

    def want(self) -> tuple[np.ndarray, np.ndarray]:
        ys, mags = [], []
        for row in range(self.B * self.R):
            b, i = divmod(row, self.R)
            on = self.penalties and self.slots[b] >= 0
            slot = max(int(self.slots[b]), 0)
            said = self.props[: self.first + i, b].tolist() if on and len(self.props) else []
            m = self.allowed[self.mask_rows[row]] if self.masks and self.mask_rows[row] >= 0 else None
            y, mag = control_row(self.x[row], self.counts[slot], self.seen[slot], said,
                                 tuple(self.pen[b]) if on else None,
                                 self.bias[b] if self.biased else {}, m)
            ys.append(y)
            mags.append(mag)
        return np.stack(ys), np.stack(mags)

    def run(self, logits: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        from microserve_b200.logits import apply_logit_controls

        return apply_logit_controls(logits, self.controls, self.tc, rows_per_request=self.R,
                                    proposals=self.dprops, first_proposal=self.first, out=out)


def assert_controlled(got: np.ndarray, want: np.ndarray, mag: np.ndarray) -> None:
    """Five float32 operations, each off by at most 2^-24 of a magnitude no larger than the
    sum of those that enter: 5 * 2^-24 * mag.  Non-finite values have to be the same."""
    fin = np.isfinite(want)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    rest = ~fin & ~np.isnan(want)
    assert np.array_equal(got[rest], want[rest])
    assert (np.abs(got[fin] - want[fin]) <= 5 * 2.0 ** -24 * mag[fin]).all()


CASES = [
    dict(B=1, R=1, V=65, bias=0, masks=False), dict(B=3, R=1, V=65), dict(B=1, R=1, V=1, bias=1),
    dict(B=2, R=4, V=33, gamma=3), dict(B=5, R=1, V=4095, gamma=4, first=2),
    dict(B=4, R=5, V=4096, gamma=4), dict(B=3, R=3, V=4100, gamma=6, first=4),
    dict(B=7, R=2, V=8191, gamma=1), dict(B=2, R=6, V=32003, gamma=5, bias=300),
    dict(B=6, R=1, V=32000, penalties=False), dict(B=3, R=1, V=128256, penalties=False, bias=0),
    dict(B=2, R=3, V=128256, gamma=2, bias=40), dict(B=300, R=1, V=97),
    dict(B=1, R=65, V=40, gamma=64),
]


@pytest.mark.parametrize("kw", CASES, ids=lambda k: "-".join(f"{a}{b}" for a, b in k.items()))
def test_controls_match_the_restatement(kw: dict) -> None:
    from microserve_b200 import _lib

    c = Case(**kw, seed=kw["V"] + kw["B"])
    want, mag = c.want()
    x = torch.from_numpy(c.x).to(DEV)
    got = c.run(x)
    assert_controlled(got.cpu().numpy(), want, mag)
    assert np.array_equal(x.cpu().numpy(), c.x)  # the input is only read
    again = x.clone()
    assert c.run(again, out=again) is again
    assert torch.equal(again, got)  # in place: the same bits
    assert _lib.device_error() == 0


@pytest.mark.parametrize("stride,shift", [(4104, 0), (4103, 0), (4104, 1)])
def test_strided_rows_leave_their_padding_alone(stride: int, shift: int) -> None:
    c = Case(4, 2, 4100, seed=stride + shift, gamma=1)
    want, mag = c.want()
    pad = torch.full((8 * stride + 8,), 7.0, device=DEV)
    view = pad[shift : shift + 8 * stride].view(8, stride)[:, :4100]
    view.copy_(torch.from_numpy(c.x))
    dst = torch.full((8 * stride + 8,), 7.0, device=DEV)
    out = dst[shift : shift + 8 * stride].view(8, stride)[:, :4100]
    c.run(view, out=out)
    assert_controlled(out.cpu().numpy(), want, mag)
    c.run(view, out=view)
    assert torch.equal(view, out)
    for buf in (pad, dst):
        rest = buf.clone()
        rest[shift : shift + 8 * stride].view(8, stride)[:, :4100] = 7.0
        assert (rest == 7.0).all()


def test_infinite_and_nan_logits() -> None:
    """Masked places become -inf whatever was there; elsewhere NaN and infinities
    go through the formula."""
    c = Case(4, 1, 4096, seed=5, bias=0)
    rng = np.random.default_rng(1)
    for bad in (np.inf, -np.inf, np.nan, np.finfo(np.float32).min, np.finfo(np.float32).max):
        c.x[rng.integers(0, 4, 60), rng.integers(0, 4096, 60)] = bad
    c.pen[:, 0] = 1.25  # min * 1.25 overflows to -inf in float32
    c.controls.penalties.copy_(torch.from_numpy(c.pen))
    with np.errstate(over="ignore", invalid="ignore"):
        want, mag = c.want()
        want = np.where(np.abs(want) > np.finfo(np.float32).max, np.sign(want) * np.inf, want)
    x = torch.from_numpy(c.x).to(DEV)
    got = c.run(x)
    assert_controlled(got.cpu().numpy(), want, mag)
    assert torch.equal(torch.nan_to_num(c.run(x, out=x), 3.0), torch.nan_to_num(got, 3.0))


def test_masked_rows_are_drawn_from_their_allowed_tokens() -> None:
    """Controls, then ms_sample: the oracle's draw on the controlled row; a row whose mask leaves
    one token draws it at any setting."""
    from microserve_b200 import _lib
    from microserve_b200.config import SamplingConfig
    from microserve_b200.logits import LogitControls, apply_logit_controls, pack_masks
    from microserve_b200.sampling import make_params, params_to_device

    for V in (65, 5000, 32000, 128256):
        rng = np.random.default_rng(V)
        rows = 10
        x = (rng.standard_normal((rows, V)) * 2).astype(np.float32)
        allowed = rng.random((rows, V)) < 0.02
        allowed[:, V // 2] = True
        allowed[0] = False
        allowed[0, V - 1] = True
        ctl = LogitControls(masks=torch.from_numpy(pack_masks(allowed)).to(DEV),
                            mask_rows=torch.arange(rows, dtype=torch.int32, device=DEV))
        y = apply_logit_controls(torch.from_numpy(x).to(DEV), ctl)
        host = np.where(allowed, x, np.float32(-np.inf))
        assert np.array_equal(y.cpu().numpy(), host)
        for t, k, p in [(0.8, None, None), (1.0, None, 0.9), (1.0, 3, None), (0.0, None, None)]:
            params = params_to_device(make_params([SamplingConfig(t, k, p)] * rows, range(rows),
                                                  [7] * rows), torch.device(DEV))
            tok = torch.empty(rows, dtype=torch.int32, device=DEV)
            _lib.call("ms_sample", y.data_ptr(), V, rows, V, params.data_ptr(), None, 0,
                      tok.data_ptr(), None, None, None, None, _lib.stream_ptr())
            got = tok.cpu().numpy()
            assert allowed[np.arange(rows), got].all()
            assert got[0] == V - 1
            for r in range(rows):
                u = float(philox.uniform(r, 7, 0))
                want, row = sample_row(host[r], t, k, p, u)
                assert got[r] == want or near_boundary(row, u)


def test_counts_follow_prompts_draws_and_accepted_rounds() -> None:
    from microserve_b200 import _lib
    from microserve_b200.logits import TokenCounts, pack_masks

    V, S = 131, 5
    rng = np.random.default_rng(3)
    tc = TokenCounts.empty(S, V, DEV)
    counts, seen = np.zeros((S, V), np.int32), np.zeros((S, V), bool)
    t = lambda a, d=np.int32: torch.from_numpy(np.asarray(a, d)).to(DEV)  # noqa: E731

    def same() -> None:
        assert np.array_equal(tc.counts.cpu().numpy(), counts)
        assert np.array_equal(tc.seen.cpu().numpy(), pack_masks(seen))

    # ragged histories with a prompt part; a slot twice; a sequence that does not count
    slots, lens, prompt = [4, 0, 4, -1, 2], [700, 1, 300, 50, 0], [100, 1, 0, 0, 0]
    toks = [rng.integers(0, V, n) for n in lens]
    for s, x, p in zip(slots, toks, prompt):
        if s >= 0:
            np.add.at(counts[s], x[p:], 1)
            seen[s, x] = True
    start = np.cumsum([0] + lens[:-1])
    tc.append(t(slots), t(np.concatenate(toks)), t(lens), row_start=t(start, np.int64), max_len=700,
              n_prompt=t(prompt))
    same()
    # one drawn token each
    drawn = rng.integers(0, V, (3, 1))
    tc.append(t([1, 2, 1]), t(drawn))
    for s, x in zip([1, 2, 1], drawn):
        np.add.at(counts[s], x, 1)
        seen[s, x] = True
    same()
    # a speculative round's emitted tokens: the accepted prefix and one more
    out, nacc = rng.integers(0, V, (3, 5)), [0, 4, 2]
    tc.append(t([0, 3, 1]), t(out), t(nacc), len_add=1)
    for s, x, n in zip([0, 3, 1], out, nacc):
        np.add.at(counts[s], x[: n + 1], 1)
        seen[s, x[: n + 1]] = True
    same()
    tc.reset(t([4, -1, 1]))
    counts[[4, 1]] = 0
    seen[[4, 1]] = False
    same()
    assert _lib.device_error() == 0
    # bad metadata: reported, skipped, the rest counted
    tc.append(t([0, 9]), t([[1, V, -1], [1, 1, 1]]))
    counts[0, 1] += 1
    seen[0, 1] = True
    same()
    assert _lib.device_error() != 0
    tc.reset(t([7]))
    same()
    assert _lib.device_error() != 0


def test_bad_metadata_sets_the_error_word_and_is_skipped() -> None:
    from microserve_b200 import _lib

    def check(change, kept) -> None:
        c = Case(3, 2, 4100, seed=11, gamma=1)
        change(c)
        got = c.run(torch.from_numpy(c.x).to(DEV)).cpu().numpy()
        assert _lib.device_error() != 0
        kept(c)
        want, mag = c.want()
        assert_controlled(got, want, mag)

    def slot(c):
        c.controls.slots[0] = 99

    def no_slot(c):
        c.slots[0] = -1

    def mask(c):
        c.controls.mask_rows[2] = 4

    def no_mask(c):
        c.mask_rows[2] = -1

    def prop(c):
        c.dprops[0, 2] = 4100

    def no_prop(c):
        c.x = c.x  # request 2's only proposal is invalid: as if its row 1 saw none

    check(slot, no_slot)
    check(mask, no_mask)
    c = Case(3, 2, 4100, seed=11, gamma=1, bias=0)
    c.dprops[0, 2] = 4100
    got = c.run(torch.from_numpy(c.x).to(DEV)).cpu().numpy()
    assert _lib.device_error() != 0
    y, mag = control_row(c.x[5], c.counts[c.slots[2]], c.seen[c.slots[2]], [], tuple(c.pen[2]), {},
                         c.allowed[c.mask_rows[5]] if c.mask_rows[5] >= 0 else None)
    assert_controlled(got[5], y, mag)
    # biases: out of the vocabulary, out of order, the same id twice: the entry is dropped
    for ids in ([5, 4100], [-3, 5], [9, 5], [5, 5]):
        c = Case(1, 1, 4100, seed=12, penalties=False, masks=False)
        c.controls.bias_start = torch.tensor([0, 2], dtype=torch.int32, device=DEV)
        c.controls.bias_ids = torch.tensor(ids, dtype=torch.int32, device=DEV)
        c.controls.bias_values = torch.tensor([2.0, 3.0], device=DEV)
        good = {i: v for k, (i, v) in enumerate(zip(ids, [2.0, 3.0]))
                if 0 <= i < 4100 and (k == 0 or ids[k - 1] < i)}
        got = c.run(torch.from_numpy(c.x).to(DEV)).cpu().numpy()
        assert _lib.device_error() != 0
        want, mag = control_row(c.x[0], c.counts[0], c.seen[0], [], None, good, None)
        assert_controlled(got[0], want, mag)


def test_proposals_not_drawn_yet_are_not_read() -> None:
    """A draft pass hands over the round's whole buffer; what no row sees may hold anything."""
    from microserve_b200 import _lib

    c = Case(3, 2, 4100, seed=13, gamma=4, first=1)
    c.dprops[2:] = -12345
    got = c.run(torch.from_numpy(c.x).to(DEV)).cpu().numpy()
    want, mag = c.want()
    assert_controlled(got, want, mag)
    assert _lib.device_error() == 0


def test_replayed_graph_and_other_stream_read_current_values() -> None:
    c = Case(3, 3, 5001, seed=21, gamma=2)
    x = torch.from_numpy(c.x).to(DEV)
    out = torch.empty_like(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.run(x, out=out)
    torch.cuda.current_stream().wait_stream(side)
    first = out.clone()
    want, mag = c.want()
    assert_controlled(first.cpu().numpy(), want, mag)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.run(x, out=out)
        c.tc.append(c.controls.slots, c.dprops[0].view(3, 1))
    c.x += 1.0
    x.copy_(torch.from_numpy(c.x))
    for _ in range(2):  # the second replay sees the first one's counts
        want, mag = c.want()
        graph.replay()
        assert_controlled(out.cpu().numpy(), want, mag)
        for b in range(3):
            if c.slots[b] >= 0:
                c.counts[c.slots[b], c.props[0, b]] += 1
                c.seen[c.slots[b], c.props[0, b]] = True


def test_refusals() -> None:
    from dataclasses import replace

    from microserve_b200.logits import LogitControls, TokenCounts, apply_logit_controls

    c = Case(2, 2, 64, seed=1, gamma=1)
    x = torch.from_numpy(c.x).to(DEV)

    def refused(logits=x, ctl=c.controls, counts=c.tc, **kw) -> None:
        with pytest.raises(ValueError):
            apply_logit_controls(logits, ctl, counts, **{"rows_per_request": 2, **kw})

    refused(x.double())
    refused(x.bfloat16())
    refused(x[0])
    refused(x.t())
    refused(rows_per_request=3)
    refused(rows_per_request=0)
    refused(counts=None)
    refused(counts=TokenCounts.empty(3, 65, DEV))
    refused(ctl=replace(c.controls, slots=None))
    refused(ctl=replace(c.controls, penalties=None))
    refused(ctl=replace(c.controls, slots=c.controls.slots.long()))
    refused(ctl=replace(c.controls, slots=c.controls.slots.cpu()))
    refused(ctl=replace(c.controls, penalties=c.controls.penalties[:1]))
    refused(ctl=replace(c.controls, bias_values=None))
    refused(ctl=replace(c.controls, bias_start=c.controls.bias_start[:-1].contiguous()))
    refused(ctl=replace(c.controls, masks=None))
    refused(ctl=replace(c.controls, masks=c.controls.masks[:, :1]))
    refused(ctl=replace(c.controls, mask_rows=c.controls.mask_rows[:3]))
    refused(proposals=c.dprops, first_proposal=1)  # row 1 would see two of one
    refused(proposals=c.dprops, first_proposal=-1)
    refused(proposals=torch.zeros((65, 2), dtype=torch.int32, device=DEV))
    refused(proposals=c.dprops[:, :1])
    refused(out=x[:1])
    refused(out=torch.empty_like(x, dtype=torch.float64))
    from microserve_b200._lib import MicroserveError

    buf = torch.zeros(4 * 64 + 4, device=DEV)  # overlapping, not in place
    with pytest.raises(MicroserveError, match="overlap"):
        apply_logit_controls(buf[:256].view(4, 64), LogitControls(), out=buf[4:].view(4, 64))
    empty = torch.empty((0, 64), device=DEV)
    assert apply_logit_controls(empty, LogitControls()).shape == (0, 64)
    same = apply_logit_controls(x, LogitControls())  # nothing set: a copy
    assert torch.equal(same, x) and same.data_ptr() != x.data_ptr()

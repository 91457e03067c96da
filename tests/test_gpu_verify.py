"""Verification of drafted tokens against the float64 oracle, which follows the
rule one child after the other with p normalised anew each time.

Tolerances.  Whole numbers are equal.  A log-probability is one rounding to fp32
of a sum taken in 64 bits of exponentials with errors of 2^-22 each (their own and
that of their exponent's last bits): 2^-24 |lp| + 2^-22, and for fp32 logits as much
again for x - max, 2^-24 (|lp| + 40) (the rows here span less than 40).
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd.sample import verify_drafts
from oracle import tree as otree
from tests.util import to_np64

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


def _cu(lens):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32)


def _tree(n, kids):
    return [-1][:n] + [(i - 1) // kids for i in range(1, n)]


class Case:
    def __init__(self, sizes, kids, vocab, dtype, mode, seed=0, temp=0.8, noise=0.7, shuffle=True):
        g = torch.Generator().manual_seed(seed)
        self.cu = _cu(sizes)
        total = sum(sizes)
        parents = []
        for n in sizes:
            if shuffle and kids > 1:  # any earlier node as the parent
                parents += [-1][:n] + [int(torch.randint(max(0, i - 3), i, (1,), generator=g))
                                       for i in range(1, n)]
            else:
                parents += _tree(n, kids)
        self.parents = torch.tensor(parents, dtype=torch.int32)
        x = torch.randn(total, vocab, generator=g) * (1 + 3 * torch.rand(total, 1, generator=g))
        self.logits = x.to(dtype)
        self.draft = None
        self.temp = 0.0 if mode == "greedy" else temp
        if mode == "drawn":
            self.draft = (x + noise * torch.randn(total, vocab, generator=g)).to(dtype)
        self.u = torch.rand(total, generator=g)
        self.tokens = torch.zeros(total, dtype=torch.int64)
        for f, n in zip(self.cu.tolist(), sizes):
            for i in range(1, n):
                at = f + parents[f + i]
                row = (self.draft if mode == "drawn" else self.logits)[at].double()
                t = temp if mode == "drawn" else 0.7
                self.tokens[f + i] = torch.multinomial(torch.softmax(row / t, -1), 1, generator=g)

    def call(self, **kw):
        args = dict(draft_logits=None if self.draft is None else self.draft.to(DEV),
                    temperature=self.temp)
        args.update(kw)
        logits = args.pop("logits", None)
        return verify_drafts(self.logits.to(DEV) if logits is None else logits,
                             self.tokens.to(DEV), self.parents.to(DEV), self.cu.to(DEV),
                             self.u.to(DEV), **args)

    def oracle(self, td=None):
        return otree.verify(to_np64(self.logits), None if self.draft is None else
                            to_np64(self.draft), self.tokens.numpy(), self.parents.numpy(),
                            self.cu.numpy(), self.u.double().numpy(), self.temp, td)

    def check(self, r, td=None):
        want = self.oracle(td)
        assert r.counts.tolist() == want["counts"]
        assert r.last.tolist() == want["last"]
        assert r.next_tokens.tolist() == want["next"]
        assert r.accepted.cpu().numpy().tolist() == want["accepted"].tolist()
        lp, got = want["logprobs"], to_np64(r.logprobs)
        assert np.array_equal(np.isnan(lp), np.isnan(got))
        ok = np.isfinite(lp)
        assert np.array_equal(lp[~ok & ~np.isnan(lp)], got[~ok & ~np.isnan(lp)])
        tol = 2.0 ** -24 * np.abs(lp[ok]) + 2.0 ** -22
        if self.logits.dtype == F32:
            tol = tol + 2.0 ** -24 * (np.abs(lp[ok]) + 40)
        assert (np.abs(got[ok] - lp[ok]) <= tol).all()
        return want


MODES = pytest.mark.parametrize("mode", ["drawn", "certain", "greedy"])


@MODES
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("sizes,kids,vocab", [
    ([1], 1, 1), ([2], 1, 2), ([5], 1, 37), ([1, 1, 4], 2, 2047), ([9, 0, 3], 2, 2048),
    ([6], 1, 2049), ([17, 30], 3, 8192), ([12], 4, 8193), ([40, 3, 1], 5, 10007),
    ([7, 7], 2, 20011), ([5, 8], 3, 151936),
])
def test_matches_the_oracle(mode, dtype, sizes, kids, vocab):
    c = Case(sizes, kids, vocab, dtype, mode, seed=vocab + len(sizes))
    c.check(c.call())


@MODES
def test_many_requests(mode):
    g = torch.Generator().manual_seed(1)
    sizes = torch.randint(0, 12, (300,), generator=g).tolist()
    c = Case(sizes, 3, 101, F32, mode, seed=2)
    want = c.check(c.call())
    assert max(want["counts"]) >= 2 and min(want["counts"]) == 0


@MODES
@pytest.mark.parametrize("kids", [1, 255])
def test_the_most_nodes(mode, kids):
    """A chain of 256 and 255 children of one node."""
    c = Case([256, 3, 256], kids, 53, F32, mode, seed=3, noise=0.1, shuffle=False)
    if kids == 1 and mode != "drawn":  # (long accepted chains)
        for i in range(1, len(c.tokens)):
            if c.parents[i] >= 0:
                f = max(x for x in c.cu.tolist() if x <= i)
                c.tokens[i] = c.logits[f + int(c.parents[i])].argmax()
    want = c.check(c.call())
    if kids == 1 and mode == "greedy":
        assert want["counts"] == [255, 2, 255]


def test_late_children_behind_many_rejected_ones():
    """Every child but a late one has a number that rejects wherever the rule
    allows: sums of third and later children."""
    for kids in (3, 4, 7):
        for seed in range(6):
            c = Case([1 + kids + 2 * kids] * 3, kids, 9001, BF16, "drawn", seed=seed, noise=1.5,
                     shuffle=False)
            c.u[1:] = 0.999 + 0.001 * c.u[1:]
            late = (c.parents >= 0) & (torch.arange(len(c.u)) % kids == 0)
            c.u[late] = 0.2
            c.check(c.call())


@pytest.mark.parametrize("td", [0.3, 1.0, 1.7])
def test_a_draft_temperature_of_its_own(td):
    c = Case([13, 6], 2, 3001, BF16, "drawn", seed=4)
    c.check(c.call(draft_temperature=td), td)


@pytest.mark.parametrize("temp", [1e-4, 0.35, 1.0, 30.0, 1e4])
@pytest.mark.parametrize("mode", ["drawn", "certain"])
def test_temperatures(temp, mode):
    c = Case([13, 6, 1], 2, 3001, F32, mode, seed=5, temp=max(temp, 0.3))
    c.temp = float(np.float32(temp))
    c.check(c.call())


def test_drafts_from_the_target_s_own_distribution_are_all_accepted():
    c = Case([9, 5], 2, 4099, BF16, "drawn", seed=6, shuffle=False)
    c.draft = c.logits.clone()
    c.u = c.u * 0 + (1 - 2.0 ** -24)  # the largest number below 1
    r = c.call()
    c.check(r)
    # the first child of every node on the path
    assert r.counts.tolist() == [3, 2]


def test_the_added_token_where_no_mass_is_left():
    """p removed to nothing by certain drafts: drawn from p as it was."""
    c = Case([3, 3], 2, 7, F32, "certain", seed=7, shuffle=False)
    c.logits[:] = float("-inf")
    c.logits[:, 2], c.logits[:, 5] = 0.0, -1.0
    c.tokens[[1, 2, 4, 5]] = torch.tensor([2, 5, 5, 2])
    c.u[:] = 1.0  # (not below 1: nothing is accepted)
    r = c.call()
    assert r.counts.tolist() == [0, 0] and r.next_tokens.tolist() == [5, 5]
    c.u[0], c.u[3] = 0.1, 0.9
    assert c.call().next_tokens.tolist() == [2, 5]


def test_numbers_at_and_outside_the_borders():
    c = Case([1] * 6, 1, 5000, BF16, "certain", seed=8)
    c.logits[:, 0] = c.logits[:, 4999] = float("-inf")  # the first and last id are impossible
    c.u = torch.tensor([0.0, 1 - 2.0 ** -24, 1.0, 7.0, float("nan"), -1.0])
    assert c.call().next_tokens.tolist() == [1, *c.oracle()["next"][1:2], 4998, 4998, 4998, 1]


@MODES
def test_excluded_ids(mode):
    """-inf and the type's lowest value, whole segments of them among them."""
    for dtype in (BF16, F32):
        c = Case([6, 4], 2, 30011, dtype, mode, seed=9)
        low = torch.finfo(dtype).min
        c.logits[:, 8000:17000] = float("-inf")
        c.logits[:, 100:9000] = low
        c.logits[1::2, :100] = float("-inf")
        if c.draft is not None:
            c.draft[:, 8000:20000] = float("-inf")
            c.draft[:, 20000:21000] = low
        c.check(c.call())


@MODES
@pytest.mark.parametrize("value", [float("nan"), float("inf"), "all -inf"])
@pytest.mark.parametrize("node", [0, 1, 3])
def test_rows_without_a_finite_maximum(mode, value, node):
    for vocab in (50, 20011):
        c = Case([4, 3], 1, vocab, F32, mode, seed=10, noise=0.0)
        if mode != "drawn":
            for f, n in ((0, 4), (4, 3)):
                for i in range(1, n):
                    c.tokens[f + i] = c.logits[f + i - 1].argmax()
        c.u[1:4] = 0.0  # (accepted as far as the rows allow)
        row = c.logits[node]
        if isinstance(value, str):
            row[:] = float("-inf")
        else:
            row[vocab // 2] = value
        r = c.call()
        c.check(r)
        assert r.last.tolist()[0] == node and r.next_tokens.tolist()[0] == -1
        assert r.next_tokens.tolist()[1] >= 0


@pytest.mark.parametrize("value", [float("nan"), float("inf")])
def test_draft_rows_without_a_finite_maximum(value):
    c = Case([5, 5], 2, 9001, BF16, "drawn", seed=11, noise=0.0, shuffle=False)
    c.draft[0, 17] = value
    r = c.call()
    c.check(r)
    assert r.counts.tolist()[0] == 0 and r.counts.tolist()[1] > 0


@MODES
def test_tokens_and_parents_out_of_range(mode):
    c = Case([12, 6], 2, 301, F32, mode, seed=12, noise=0.2)
    c.tokens[2], c.tokens[3], c.tokens[13] = -1, 301, 2 ** 40
    c.tokens[0] = -5  # (node 0's token is not looked at)
    c.parents[5], c.parents[7], c.parents[9] = -1, 7, 300  # padding, themselves, a later one
    c.parents[0] = 4                                       # (nor is its parent)
    r = c.call()
    c.check(r)
    assert r.logprobs[[2, 3, 5, 7, 9, 13]].isnan().all()


@pytest.mark.parametrize("mode", ["drawn", "certain"])
def test_the_same_child_several_times(mode):
    c = Case([9] * 8, 8, 40, F32, mode, seed=13, shuffle=False)
    for f in range(0, 72, 9):
        c.tokens[f + 1 : f + 9] = c.tokens[f + 1 : f + 5].repeat(2)
    c.check(c.call())


def test_greedy_takes_the_lowest_of_equal_ids():
    c = Case([3, 3], 2, 20000, BF16, "greedy", seed=14, shuffle=False)
    c.logits[:, [77, 9000, 19999]] = 30.0
    c.tokens[[1, 2, 4, 5]] = torch.tensor([9000, 77, 19999, 9000])
    r = c.call()
    c.check(r)
    assert r.last.tolist() == [2, 0] and r.next_tokens.tolist() == [77, 77]
    zero = Case([1], 1, 64, F32, "greedy")
    zero.logits[:] = -0.0
    zero.logits[0, 9] = 0.0
    assert zero.call().next_tokens.tolist() == [0]


@MODES
def test_nodes_behind_the_last_request(mode):
    """A padded batch: nodes of no request are not accepted, NaN, and change nothing."""
    c = Case([5, 7, 4], 2, 500, F32, mode, seed=15)
    want = c.oracle()
    c.cu = c.cu[:3]
    r = c.call()
    assert r.counts.tolist() == want["counts"][:2] and r.next_tokens.tolist() == want["next"][:2]
    assert not r.accepted[12:].any() and r.logprobs[12:].isnan().all()


@MODES
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_strided_and_unaligned_rows(mode, dtype):
    c = Case([6, 3], 2, 8195, dtype, mode, seed=16)
    room = torch.zeros(9, 8300, dtype=dtype, device=DEV)
    room[:, 3:8198] = c.logits.to(DEV)
    kw = {}
    if c.draft is not None:
        wide = torch.zeros(9, 9001, dtype=dtype, device=DEV)
        wide[:, 1:8196] = c.draft.to(DEV)
        kw["draft_logits"] = wide[:, 1:8196]
    c.check(c.call(logits=room[:, 3:8198], **kw))


def test_one_row_for_all_nodes():
    c = Case([4, 4], 1, 700, F32, "certain", seed=17)
    c.logits[:] = c.logits[0]
    r = c.call(logits=c.logits[:1].to(DEV).expand(8, -1))
    c.check(r)


@MODES
def test_replayed_from_a_graph(mode):
    c = Case([16, 9, 4], 3, 20011, BF16, mode, seed=18)
    logits, draft = c.logits.to(DEV), None if c.draft is None else c.draft.to(DEV)
    u, tok, par, cu = (x.to(DEV) for x in (c.u, c.tokens, c.parents, c.cu))
    run = lambda: verify_drafts(logits, tok, par, cu, u, draft_logits=draft, temperature=c.temp)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = run()
    g = torch.Generator().manual_seed(0)
    for _ in range(3):
        u.copy_(torch.rand(u.shape, generator=g))
        logits.copy_(logits.flip(1))
        graph.replay()
        eager = run()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


def test_two_streams_at_once():
    cs = [Case([16, 9, 4], 3, 151936, BF16, "drawn", seed=s) for s in (19, 20)]
    wants = [c.call() for c in cs]
    on = [(c.logits.to(DEV), c.tokens.to(DEV), c.parents.to(DEV), c.cu.to(DEV), c.u.to(DEV),
           c.draft.to(DEV)) for c in cs]
    streams = [torch.cuda.Stream() for _ in cs]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for i, (s, a) in enumerate(zip(streams, on)):
            with torch.cuda.stream(s):
                outs.append((i, verify_drafts(*a[:5], draft_logits=a[5], temperature=0.8)))
    torch.cuda.synchronize()
    for i, r in outs:
        for a, b in zip(r, wants[i]):
            assert torch.equal(a.nan_to_num(7.0), b.nan_to_num(7.0))


@pytest.mark.parametrize("mode", ["drawn", "certain"])
@pytest.mark.parametrize("kids", [1, 3])
def test_the_first_token_is_distributed_as_the_target_s(mode, kids):
    """40,000 requests with drafts of their own over 6 ids: the first token that
    comes out (an accepted child of node 0 or the added one) has the target's
    frequencies, each within 5 standard deviations."""
    b, vocab = 40000, 6
    g = torch.Generator().manual_seed(21)
    p_log = torch.tensor([0.3, 1.2, -0.4, 0.9, -2.0, 0.0])
    q_log = torch.tensor([1.0, 0.1, 0.2, -1.0, 0.7, 0.0])
    n = 1 + kids
    draws = torch.multinomial(torch.softmax(q_log, -1).expand(b, -1), kids, replacement=True,
                              generator=g)
    if mode == "certain":
        draws = torch.arange(kids).expand(b, -1) * 2 % vocab
    tokens = torch.cat((torch.zeros(b, 1, dtype=torch.int64), draws), 1).reshape(-1)
    r = verify_drafts(p_log.to(DEV).expand(b * n, -1), tokens.to(DEV),
                      torch.tensor([-1] + [0] * kids, dtype=torch.int32).repeat(b).to(DEV),
                      _cu([n] * b).to(DEV), torch.rand(b * n, generator=g).to(DEV),
                      draft_logits=(q_log.to(DEV).expand(b * n, -1) if mode == "drawn" else None))
    last = r.last.long().cpu()
    first = torch.where(last > 0, tokens.view(b, n).gather(1, last[:, None])[:, 0],
                        r.next_tokens.cpu())
    p = torch.softmax(p_log.double(), -1)
    freq = torch.bincount(first, minlength=vocab).double() / b
    assert ((freq - p).abs() <= 5 * (p * (1 - p) / b).sqrt()).all(), (freq, p)
    assert 0.05 < (last > 0).double().mean() < 1


@MODES
@pytest.mark.parametrize("vocab", [5003, 40009])
def test_rows_past_32_bits(mode, vocab):
    c = Case([4, 2], 1, vocab, BF16, mode, seed=vocab)
    step = 700_000_000  # the last row is 3.5e9 elements behind the first
    far = lambda x: torch.empty(5 * step + vocab, dtype=x.dtype, device=DEV).as_strided(
        (6, vocab), (step, 1)).copy_(x)
    kw = {} if c.draft is None else {"draft_logits": far(c.draft)}
    c.check(c.call(logits=far(c.logits), **kw))

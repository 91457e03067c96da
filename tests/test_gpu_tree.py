"""Attention of trees of drafted tokens, over the bf16 and the 8-bit cache, against
the float64 oracle.

Tolerances.  With w the weights of a row (sum 1) and A = sum w_t |v_t|, an output
o = sum w_t v_t differs from the oracle on the same cache by at most
  2^-8 |o|     its rounding to bf16
  2^-8 A       each weight's rounding to bf16
  2 (D 2^-24 S + 2^-18) A   the weights' relative error (in the numerator and in
               the sum) from fp32 scores, S the largest scale * sum |q_d k_d|, and
               from the exponentials
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd import paged
from oracle import kv8 as okv8
from oracle import tree as otree
from tests.util import to_np64

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cu(lens):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32)


def _random_parents(g, n):
    return [-1][:n] + [int(torch.randint(i, (1,), generator=g)) for i in range(1, n)]


class Case:
    """A batch of trees over one layer's cache of `bits`."""

    def __init__(self, nodes, cached, hq, hkv, d, bits, seed=0, spread=0.5, extra=7):
        g = torch.Generator().manual_seed(seed)
        self.bits, self.hq, self.hkv, self.d = bits, hq, hkv, d
        kv = [n + c for n, c in zip(nodes, cached)]
        self.cu_q, self.cu_k = _cu(nodes), _cu(kv)
        self.pages = sum(kv) + extra
        self.indices = torch.randperm(self.pages, generator=g)[: sum(kv)].to(torch.int32)
        self.q = torch.randn(sum(nodes), hq, d, generator=g).to(torch.bfloat16)
        rows = [torch.randn(self.pages, hkv, d, generator=g)
                * torch.randn(self.pages, hkv, 1, generator=g).mul(spread).exp() for _ in range(2)]
        self.k, self.v = (x.to(torch.bfloat16) for x in rows)
        self.parents = [_random_parents(g, n) for n in nodes]
        self.seen = [s for p in self.parents for s in otree.ancestors(p)]
        self.words = max(1, -(-max(nodes, default=1) // 64))

    def masks(self):
        return torch.from_numpy(otree.mask_words(self.seen, self.words))

    def cache(self):
        """(device tensors of the cache, its K and V in float64)"""
        if self.bits == 16:
            return ((self.k.to(DEV), self.v.to(DEV)), to_np64(self.k), to_np64(self.v))
        (k, ks), (v, vs) = (okv8.quantize_rows(to_np64(x)) for x in (self.k, self.v))
        scales = np.stack((ks.T, vs.T), -1)
        dev = [torch.from_numpy(x).float().to(torch.float8_e4m3fn).contiguous().to(DEV)
               for x in (k, v)]
        dev.append(torch.from_numpy(scales).to(torch.bfloat16).contiguous().to(DEV))
        return tuple(dev), okv8.values(k, scales, 0), okv8.values(v, scales, 1)

    def plan(self):
        return paged.plan("tree", self.cu_q, self.cu_k, self.hq, self.hkv, self.d,
                          kv_bits=self.bits)

    def call(self, cache, q=None, plan=None, **kw):
        f = paged.tree_attention if self.bits == 16 else paged.tree_attention8
        return f(plan or self.plan(), self.q.to(DEV) if q is None else q, *cache,
                 self.indices.to(DEV), self.cu_q.to(DEV), self.cu_k.to(DEV), self.masks().to(DEV),
                 **kw)

    def oracle(self, k, v):
        """(outputs, tolerance)"""
        args = (self.indices.numpy(), self.cu_q.numpy(), self.cu_k.numpy(), self.seen)
        q, scale = to_np64(self.q), self.d ** -0.5
        want = otree.tree_attention(q, k, v, *args, scale)
        a = otree.tree_attention(q, k, np.abs(v), *args, scale)
        kf = np.where(np.isfinite(k), np.abs(k), 0.0)
        s = np.abs(q).max() * kf.sum(-1).max() * scale
        return want, 2.0 ** -8 * np.abs(want) + a * (
            2.0 ** -8 + 2 * (self.d * 2.0 ** -24 * s + 2.0 ** -18)) + 1e-30

    def check(self, out, k, v):
        want, tol = self.oracle(k, v)
        got = to_np64(out)
        bad = np.isfinite(want)
        assert np.array_equal(np.isnan(got), np.isnan(want))
        assert np.array_equal(got[~bad & ~np.isnan(want)], want[~bad & ~np.isnan(want)])
        worst = np.where(bad, np.abs(np.where(bad, got, 0) - np.where(bad, want, 0))
                         - np.where(bad, tol, 0), 0)
        assert worst.max(initial=0) <= 0, (
            f"{worst.max()} over the tolerance at {np.unravel_index(worst.argmax(), worst.shape)}")


BITS = pytest.mark.parametrize("bits", [16, 8])


@BITS
@pytest.mark.parametrize("nodes,cached,hq,hkv,d", [
    ([1], [0], 8, 2, 96),               # one token, nothing cached
    ([1], [33], 12, 4, 64),
    ([8], [24], 8, 2, 96),
    ([17], [300], 16, 8, 128),
    ([5, 1, 31, 12], [0, 200, 63, 64], 12, 4, 64),
    ([64], [31], 32, 8, 128),           # a part of a sub-tile before the nodes
    ([65, 2], [1, 700], 8, 8, 64),      # two mask words
    ([33, 40], [129, 5], 8, 1, 96),     # eight heads a kv-head, several tiles
    ([256], [97], 8, 4, 64),            # the most nodes
    ([200, 7], [0, 1000], 16, 8, 128),
    ([3, 0, 2], [40, 9, 0], 6, 1, 128),  # a request without nodes
])
def test_matches_the_oracle(bits, nodes, cached, hq, hkv, d):
    c = Case(nodes, cached, hq, hkv, d, bits, seed=sum(nodes) + d)
    cache, k, v = c.cache()
    c.check(c.call(cache), k, v)


@BITS
@pytest.mark.parametrize("nodes,cached,hq,hkv,d", [
    ([6], [4093], 16, 8, 128), ([17], [2500], 32, 8, 128), ([40], [3001], 12, 4, 64),
    ([100, 9], [1500, 2200], 8, 2, 96), ([4, 4, 4, 3, 4, 4, 4, 4], [1800] * 8, 16, 8, 128),
])
def test_long_caches(bits, nodes, cached, hq, hkv, d):
    c = Case(nodes, cached, hq, hkv, d, bits, seed=len(nodes) + d)
    cache, k, v = c.cache()
    c.check(c.call(cache), k, v)


@BITS
@pytest.mark.parametrize("cached", [0, 19, 1300])
def test_any_mask(bits, cached):
    """Masks of no tree: nodes that see later ones, all, none (zeros where
    nothing is cached), and bits past the request's nodes."""
    nodes = [70, 9]
    c = Case(nodes, [cached, cached], 8, 2, 96, bits, seed=5)
    g = torch.Generator().manual_seed(1)
    c.seen = [set(torch.randperm(128, generator=g)[: int(torch.randint(90, (1,), generator=g))]
                  .tolist()) for _ in range(sum(nodes))]
    c.seen[0] = c.seen[71] = set()
    c.seen[3] = {69}
    c.seen[4] = set(range(128))
    c.seen[75] = {9, 64, 127}  # none of them a node of that request
    cache, k, v = c.cache()
    out = c.call(cache)
    c.check(out, k, v)
    if cached == 0:
        assert (out[[0, 71, 75]] == 0).all()


@BITS
def test_a_chain_is_the_causal_prefill(bits):
    nodes, cached = [20, 7], [50, 333]
    c = Case(nodes, cached, 16, 8, 128, bits, seed=9)
    c.seen = [set(range(i + 1)) for n in nodes for i in range(n)]
    cache, k, v = c.cache()
    p = paged.plan("prefill", c.cu_q, c.cu_k, 16, 8, 128, kv_bits=bits)
    f = paged.prefill if bits == 16 else paged.prefill8
    want = f(p, c.q.to(DEV), *cache, c.indices.to(DEV), c.cu_q.to(DEV), c.cu_k.to(DEV))
    # (both are within one tolerance of the oracle)
    _, tol = c.oracle(k, v)
    assert (np.abs(to_np64(c.call(cache)) - to_np64(want)) <= 2 * tol + 2.0 ** -8 * np.abs(
        to_np64(want))).all()


@pytest.mark.parametrize("value", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("which", ["k", "v"])
@pytest.mark.parametrize("cached", [0, 70, 2000])
def test_unseen_values_do_not_reach_an_output(value, which, cached):
    """One node's K or V row holds a value that is not finite: the nodes that
    see it get what the formula gives, the others what they had."""
    c = Case([40], [cached], 8, 2, 96, 16, seed=3)
    at = 11
    page = int(c.indices[cached + at])
    clean = c.call(c.cache()[0])
    x = c.k if which == "k" else c.v
    x[page, 0, 5] = value
    x[page, 1, 90] = value
    cache, k, v = c.cache()
    out = c.call(cache)
    sees = torch.tensor([at in s for s in c.seen])
    assert sees.any() and not sees.all()
    assert torch.equal(out[~sees.to(DEV)], clean[~sees.to(DEV)])
    if which == "v":
        c.check(out, k, v)
        assert not out[sees.to(DEV)][:, :, [5, 90]].isfinite().all()
    else:  # (an infinite score: the formula's own result is NaN or without that node)
        hit = out[sees.to(DEV)]
        if value != value:
            assert hit.isnan().all()


def test_infinities_of_both_signs_and_nan_in_one_tile():
    c = Case([64], [0], 4, 1, 64, 16, seed=8)
    pages = c.indices.long()
    c.v[pages[3], 0, 0] = float("inf")
    c.v[pages[9], 0, 0] = float("-inf")
    c.v[pages[20], 0, 1] = float("nan")
    c.v[pages[20], 0, 2] = float("inf")
    c.seen = [set() for _ in range(64)]
    c.seen[0], c.seen[1], c.seen[2] = {3, 5}, {9, 5}, {3, 9}
    c.seen[3], c.seen[4], c.seen[5] = {20}, {63}, {3, 9, 20, 40}
    cache, k, v = c.cache()
    out = c.call(cache)
    c.check(out, k, v)
    assert (out[0, :, 0] == float("inf")).all() and (out[1, :, 0] == float("-inf")).all()
    assert out[2, :, 0].isnan().all() and out[4].isfinite().all()
    assert out[3, :, 1].isnan().all() and (out[3, :, 2] == float("inf")).all()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("cached", [0, 1500])
def test_a_nan_token_of_the_8_bit_cache(which, cached):
    """A node stored with a NaN (K or V): NaN for the nodes that see it, no other."""
    c = Case([30], [cached], 8, 2, 96, 8, seed=4)
    clean = c.call(c.cache()[0])
    cache, _, _ = c.cache()
    page = int(c.indices[cached + 6])
    cache[2][1, page, which] = float("nan")
    out = c.call(cache)
    sees = torch.tensor([6 in s for s in c.seen]).to(DEV)
    assert out[sees][:, 4:].isnan().all()
    assert torch.equal(out[~sees], clean[~sees]) and torch.equal(out[:, :4], clean[:, :4])


@BITS
def test_pages_outside_the_pool_are_rows_of_zeros(bits):
    c = Case([9, 4], [50, 200], 8, 2, 96, bits, seed=6)
    c.indices[[3, 55, 80]] = torch.tensor([-1, c.pages, 2 ** 31 - 1], dtype=torch.int32)
    cache, k, v = c.cache()
    c.check(c.call(cache), k, v)


@BITS
def test_rows_of_a_fused_projection_and_a_given_output(bits):
    c = Case([13], [77], 16, 8, 128, bits, seed=2)
    wide = torch.zeros(13, 32 * 128, dtype=torch.bfloat16, device=DEV)
    q = wide[:, : 16 * 128].view(13, 16, 128)
    q.copy_(c.q)
    cache, k, v = c.cache()
    room = torch.full((20, 16, 128), 3.0, dtype=torch.bfloat16, device=DEV)
    out = c.call(cache, q=q, out=room[:13])
    assert out.data_ptr() == room.data_ptr() and (room[13:] == 3).all()
    c.check(out, k, v)
    assert torch.equal(out, c.call(cache))


@BITS
@pytest.mark.parametrize("planned", [([40, 40], [2000, 100]), ([64, 64], [64, 64])])
def test_lengths_other_than_planned(bits, planned):
    """The plan's lengths are those of a step's largest trees; the device's are
    smaller trees behind shorter and longer caches."""
    c = Case([3, 38], [1400, 700], 12, 4, 64, bits, seed=7)
    cache, k, v = c.cache()
    p = paged.plan("tree", _cu(planned[0]), _cu([n + m for n, m in zip(*planned)]), 12, 4, 64,
                   kv_bits=bits)
    n = sum(planned[0])
    pad = lambda x, m: torch.cat((x, torch.zeros(m, *x.shape[1:], dtype=x.dtype)))
    q = pad(c.q, n - 41).to(DEV)
    masks = pad(c.masks(), n - 41).to(DEV)
    idx = pad(c.indices, max(0, p.total_kv - len(c.indices))).to(DEV)
    room = torch.full_like(q, 5.0)
    f = paged.tree_attention if bits == 16 else paged.tree_attention8
    out = f(p, q, *cache, idx, c.cu_q.to(DEV), c.cu_k.to(DEV), masks, out=room)
    assert (out[41:] == 5).all()
    c.check(out[:41], k, v)


@BITS
def test_the_scale_is_the_caller_s(bits):
    c = Case([5], [20], 8, 2, 96, bits, seed=1)
    cache, k, v = c.cache()
    args = (c.indices.numpy(), c.cu_q.numpy(), c.cu_k.numpy(), c.seen)
    want = otree.tree_attention(to_np64(c.q), k, v, *args, 0.3)
    a = otree.tree_attention(to_np64(c.q), k, np.abs(v), *args, 0.3)
    s = np.abs(to_np64(c.q)).max() * np.abs(k).sum(-1).max() * 0.3
    tol = 2.0 ** -8 * np.abs(want) + a * (2.0 ** -8 + 2 * (96 * 2.0 ** -24 * s + 2.0 ** -18))
    assert (np.abs(to_np64(c.call(cache, sm_scale=0.3)) - want) <= tol).all()


@BITS
def test_replayed_from_a_graph_on_another_stream(bits):
    """A captured call, replayed with eager work of the program between the
    replays and other contents of the same buffers."""
    c = Case([17, 6], [1600, 900], 16, 8, 128, bits, seed=12)
    cache, _, _ = c.cache()
    p = c.plan()
    q = c.q.to(DEV)
    idx, cu_q, cu_k, masks = (x.to(DEV) for x in (c.indices, c.cu_q, c.cu_k, c.masks()))
    out = torch.empty_like(q)
    f = paged.tree_attention if bits == 16 else paged.tree_attention8
    run = lambda o: f(p, q, *cache, idx, cu_q, cu_k, masks, out=o)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        run(out)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        run(out)
    g = torch.Generator().manual_seed(0)
    for _ in range(3):
        q.copy_(torch.randn(q.shape, generator=g))
        out.zero_()
        graph.replay()
        eager = run(torch.empty_like(q))
        torch.cuda.synchronize()
        assert torch.equal(out, eager)


@BITS
def test_two_calls_of_one_plan_on_two_streams(bits):
    c = Case([12], [3000], 16, 8, 128, bits, seed=13)
    cache, k, v = c.cache()
    p = c.plan()
    want = c.call(cache, plan=p)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    outs = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                outs.append(c.call(cache, plan=p))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


# -- masks -----------------------------------------------------------------------

@pytest.mark.parametrize("sizes", [[1], [7, 1, 30], [64, 65], [256], [0, 3, 0], [130, 256, 2]])
def test_masks_and_depths_of_random_trees(sizes):
    g = torch.Generator().manual_seed(sum(sizes))
    parents = [_random_parents(g, n) for n in sizes if n]
    flat = torch.tensor(sum(parents, []), dtype=torch.int32)
    top = max(sizes)
    masks, depths = paged.tree_masks(flat.to(DEV), _cu(sizes).to(DEV), top)
    seen = [s for p in parents for s in otree.ancestors(p)]
    assert masks.shape == (sum(sizes), -(-top // 64))
    assert (masks.cpu().numpy() == otree.mask_words(seen, masks.shape[1])).all()
    assert depths.tolist() == [len(s) - 1 for s in seen]


def test_masks_of_chains_and_of_nodes_without_an_earlier_parent():
    n = 256
    chain = torch.arange(-1, n - 1, dtype=torch.int32)
    odd = chain.clone()
    odd[5], odd[70], odd[200] = 5, 255, -7  # themselves, a later one, none
    both = torch.cat((chain, odd)).to(DEV)
    masks, depths = paged.tree_masks(both, _cu([n, n]).to(DEV), n)
    seen = otree.ancestors(chain.tolist()) + otree.ancestors(odd.tolist())
    assert (masks.cpu().numpy() == otree.mask_words(seen, 4)).all()
    assert depths.tolist() == [len(s) - 1 for s in seen]


def test_masks_past_the_most_nodes_and_past_the_words():
    chain = torch.arange(-1, 299, dtype=torch.int32)
    masks, depths = paged.tree_masks(chain.to(DEV), _cu([300]).to(DEV), 128)
    seen = otree.ancestors(chain.tolist())[:256] + [set()] * 44
    assert (masks.cpu().numpy() == otree.mask_words(seen, 2)).all()
    assert depths.tolist() == [*range(256), *([0] * 44)]


def test_masks_leave_rows_past_the_last_request():
    flat = torch.full((10,), -1, dtype=torch.int32, device=DEV)
    masks, depths = paged.tree_masks(flat, _cu([4, 50]).to(DEV), 64)  # (cu past the nodes)
    assert masks[:4].flatten().tolist() == [1, 2, 4, 8]
    assert masks[4:].flatten().tolist() == [1, 2, 4, 8, 16, 32]
    assert (depths == 0).all()


@BITS
@pytest.mark.parametrize("parts", [False, True])
@pytest.mark.parametrize("nodes,cached,hq,hkv,d", [
    ([6, 1], [3100, 2600], 8, 2, 96), ([16], [4030], 8, 4, 64), ([17, 9], [0, 3900], 16, 8, 128),
    ([31], [2500], 16, 8, 128), ([9], [247], 8, 8, 128), ([9], [279], 8, 8, 128),
])
def test_few_rows_with_long_parts(bits, parts, nodes, cached, hq, hkv, d):
    """At most 64 rows and more than eight sub-tiles a part, which its wavefronts share:
    without a workspace, and where the device's lengths are six times the planned."""
    c = Case(nodes, cached, hq, hkv, d, bits, seed=sum(cached) + d)
    short = _cu([n + x // 6 for n, x in zip(nodes, cached)])
    plan = paged.plan("tree", c.cu_q, short if parts else c.cu_k, hq, hkv, d, kv_bits=bits,
                      **({} if parts else {"workspace_bytes": 0}))
    if not parts:
        assert plan.num_parts == 1
    plan.total_kv = int(c.cu_k[-1])  # (what the indices are checked for)
    cache, k, v = c.cache()
    c.check(c.call(cache, plan=plan), k, v)


@BITS
def test_values_nobody_sees_in_a_shared_part(bits):
    c = Case([12, 3], [610, 290], 8, 4, 64, bits, seed=77)
    g = torch.Generator().manual_seed(3)
    c.seen = [sorted({i} | set(torch.randint(12, (2,), generator=g).tolist())) for i in range(12)]
    c.seen = [[j for j in s if j != 5] for s in c.seen] + [[0], [], [0, 2]]
    if bits == 16:
        c.v[c.indices[610 + 5].long()] = float("nan")  # node 5 is seen by none
        c.v[c.indices[-2].long()] = float("-inf")      # nor is node 1 of the second
    plan = paged.plan("tree", c.cu_q, c.cu_k, 8, 4, 64, kv_bits=bits, workspace_bytes=0)
    cache, k, v = c.cache()
    out = c.call(cache, plan=plan)
    if bits == 16:
        k, v = k.copy(), np.where(np.isfinite(v), v, 0.0)
    c.check(out, k, v)
    assert torch.isfinite(out).all()


@BITS
def test_pages_at_the_end_of_the_largest_pool(bits):
    """Rows next to 4 GiB into a layer's cache: offsets past 31 bits."""
    c = Case([9, 5], [300, 40], 16, 8, 128, bits, seed=5)
    small, k, v = c.cache()
    pages = (2_097_000 if bits == 16 else 4_194_000)
    assert pages * 8 * 128 * (2 if bits == 16 else 1) > 0.999 * 2 ** 32
    at = pages - c.pages
    cache = []
    for t in small[:2]:
        big = torch.empty((pages, *t.shape[1:]), dtype=t.dtype, device=DEV)
        big[at:] = t
        cache.append(big)
    if bits == 8:
        scales = torch.empty((8, pages, 2), dtype=torch.bfloat16, device=DEV)
        scales[:, at:] = small[2]
        cache.append(scales)
    c.indices += at
    out = c.call(cache)
    c.indices -= at
    c.check(out, k, v)

"""The 8-bit KV cache: quantising append, decode and prefill attention, against
the float64 oracle.

Tolerances.  The append is exact: codes and scales are compared bit for bit.
An attention output o = sum w_t v_t (A = sum w_t |v_t|) differs from the oracle
on the same codes by at most
  2^-8 |o|     the output's rounding to bf16
  2^-8 A       each weight's rounding to bf16 (twice in the prefill, whose row
               sum is taken of the rounded weights)
  2^-11 A      the decode's fp16 partial states
  2 D 2^-24 S  A  relative error of the weights from fp32 scores, with S the
               largest scale * sum |q_d k_d|, and 2^-18 A for the exponentials
and K and V enter the products exactly.
"""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd import _lib, paged
from aios_amd.kernel import store_cache, store_cache8
from aios_amd.layers import HipOps
from oracle import kv8 as okv8
from tests.util import to_np64

pytestmark = pytest.mark.gpu
DEV = "cuda"
FP8 = torch.float8_e4m3fn


def _rows(g, *shape, spread=1.0):
    x = torch.randn(*shape, generator=g)
    return (x * torch.randn(*shape[:-1], 1, generator=g).mul(spread).exp()).to(torch.bfloat16)


def _pool(g, pages, hkv, d):
    """A filled cache: k8, v8, scales on the GPU and its values in float64."""
    k, ks = okv8.quantize_rows(to_np64(_rows(g, pages, hkv, d, spread=0.3)))
    v, vs = okv8.quantize_rows(to_np64(_rows(g, pages, hkv, d)))
    scales = np.stack((ks.T, vs.T), -1)
    dev = [torch.from_numpy(x).float().to(FP8).contiguous().to(DEV) for x in (k, v)]
    return (*dev, torch.from_numpy(scales).to(torch.bfloat16).contiguous().to(DEV))


def _values(k8, v8, scales):
    s = to_np64(scales)
    return (okv8.values(to_np64(k8.float()), s, 0), okv8.values(to_np64(v8.float()), s, 1))


def _cu(lens):
    return torch.tensor([0, *lens]).cumsum(0).to(torch.int32)


def _oracle(q, k, v, indices, cu_q, cu_k, weights=1):
    """(outputs, tolerance) of every query row."""
    q, idx = to_np64(q), indices.cpu().numpy()
    hq, d = q.shape[1:]
    hkv = k.shape[1]
    g = hq // hkv
    out, tol = np.zeros(q.shape), np.zeros(q.shape)
    for r in range(len(cu_q) - 1):
        pages = idx[int(cu_k[r]):int(cu_k[r + 1])]
        ok = (pages >= 0) & (pages < k.shape[0])
        n, t = len(pages), int(cu_q[r + 1] - cu_q[r])
        if n == 0 or t == 0:
            continue
        kr = np.where(ok[:, None, None], k[np.where(ok, pages, 0)], 0.0)
        vr = np.where(ok[:, None, None], v[np.where(ok, pages, 0)], 0.0)
        seen = np.arange(n)[None, :] <= (n - t + np.arange(t))[:, None]
        for h in range(hq):
            qh, kh, vh = q[int(cu_q[r]):int(cu_q[r + 1]), h], kr[:, h // g], vr[:, h // g]
            s = np.where(seen, qh @ kh.T * d ** -0.5, -np.inf)
            w = np.exp(s - s.max(-1, keepdims=True))
            w /= w.sum(-1, keepdims=True)
            o, a = w @ vh, w @ np.abs(vh)
            big = float((np.abs(qh) @ np.abs(kh).T).max()) * d ** -0.5
            rel = weights * 2.0 ** -8 + 2.0 ** -11 + 2 * d * 2.0 ** -24 * big + 2.0 ** -18
            out[int(cu_q[r]):int(cu_q[r + 1]), h] = o
            tol[int(cu_q[r]):int(cu_q[r + 1]), h] = 2.0 ** -8 * np.abs(o) + rel * a
    return out, tol


def _near(out, want, tol):
    got = to_np64(out)
    assert np.isfinite(got).all()
    worst = np.abs(got - want) - tol
    assert (worst <= 0).all(), f"{worst.max()} over the tolerance at {np.unravel_index(worst.argmax(), worst.shape)}"


# -- append ------------------------------------------------------------------

def _bits(t):
    return t.cpu().contiguous().view(torch.uint8 if t.element_size() == 1 else torch.int16)


@pytest.mark.parametrize("tokens,hkv,d", [(1, 1, 64), (5, 2, 96), (8, 2, 96), (7, 8, 128),
                                          (300, 4, 64), (1000, 8, 128)])
def test_append_is_exact(tokens, hkv, d):
    g = torch.Generator().manual_seed(tokens + d)
    pages = tokens + 9
    k8, v8, scales = _pool(g, pages, hkv, d)
    was = [x.clone() for x in (k8, v8, scales)]
    k = _rows(g, tokens, hkv, d, spread=3.0)
    qkv = _rows(g, tokens, 4 * hkv, d, spread=3.0)
    v = qkv[:, 3 * hkv:]  # a strided view, as the model's
    loc = torch.randperm(pages, generator=g)[:tokens].to(torch.int32)
    if tokens > 4:
        loc[1], loc[3] = -1, pages  # not written
    store_cache8(k8, v8, scales, loc.to(DEV), k.to(DEV), qkv.to(DEV)[:, 3 * hkv:])
    for w, (cache, old, x) in enumerate(((k8, was[0], k), (v8, was[1], v))):
        codes, s = okv8.quantize_rows(to_np64(x))
        live = ((loc >= 0) & (loc < pages)).nonzero()[:, 0]
        want, ws = old.cpu().float(), was[2][:, :, w].cpu().clone()
        want[loc[live].long()] = torch.from_numpy(codes).float()[live]
        ws[:, loc[live].long()] = torch.from_numpy(s.T).to(torch.bfloat16)[:, live]
        assert torch.equal(_bits(cache), _bits(want.to(FP8)))
        assert torch.equal(_bits(scales[:, :, w]), _bits(ws))


def test_append_with_64_bit_indices():
    """Indices past 32 bits are outside the pool, not somewhere in it."""
    g = torch.Generator().manual_seed(2)
    k8, v8, scales = _pool(g, 8, 2, 64)
    want = [x.clone() for x in (k8, v8, scales)]
    k, v = _rows(g, 4, 2, 64).to(DEV), _rows(g, 4, 2, 64).to(DEV)
    loc = torch.tensor([2 ** 32 + 3, 5, -2 ** 32 + 1, -1], device=DEV)
    store_cache8(k8, v8, scales, loc, k, v)
    store_cache8(*want, torch.tensor([-1, 5, 8, -1], dtype=torch.int32, device=DEV), k, v)
    assert all(torch.equal(_bits(a), _bits(b)) for a, b in zip((k8, v8, scales), want))


@pytest.mark.parametrize("d", [64, 96, 128])
def test_append_extreme_rows(d):
    """Zero rows, subnormals, the type's largest values, borders of the scale
    (448 2^e and the next value above), NaN and infinities."""
    base = torch.linspace(-1, 1, d)
    top = torch.finfo(torch.bfloat16).max
    rows = [base * 0, base * 2.0 ** -126, base * 2.0 ** -133, base * top, base * 1e-30,
            torch.where(base > 0.9, 448.0, 0.25), torch.where(base > 0.9, 450.0, 0.25),
            torch.where(base > 0.9, 2.0 ** -7 * 448, 2.0 ** -16),
            torch.where(base > 0.99, float("nan"), base), torch.where(base > 0.99, float("inf"), base),
            torch.where(base < 0, float("-inf"), float("nan")), -base]
    x = torch.stack(rows)[:, None].to(torch.bfloat16)
    n = len(rows)
    k8 = torch.zeros(n, 1, d).to(FP8).to(DEV)
    v8, scales = k8.clone(), torch.zeros(1, n, 2, dtype=torch.bfloat16, device=DEV)
    loc = torch.arange(n, dtype=torch.int32, device=DEV)
    store_cache8(k8, v8, scales, loc, x.to(DEV), x.flip(0).to(DEV))
    for w, (cache, rows_in) in enumerate(((k8, x), (v8, x.flip(0)))):
        codes, s = okv8.quantize_rows(to_np64(rows_in))
        # (a zero code's sign is the sign of its value: compared as values)
        np.testing.assert_array_equal(to_np64(cache.float()), codes)
        np.testing.assert_array_equal(to_np64(scales[0, :, w]), s[:, 0])


@pytest.mark.parametrize("tokens,hq,hkv,d", [(1, 8, 2, 96), (7, 12, 4, 64), (33, 16, 8, 128),
                                             (700, 32, 8, 128), (260, 8, 8, 64)])
def test_rope_append_equals_its_two_calls(tokens, hq, hkv, d):
    g = torch.Generator().manual_seed(tokens)
    qkv = _rows(g, tokens, hq + 2 * hkv, d).view(tokens, -1).to(DEV)
    qw, kw = (torch.rand(d, generator=g).to(torch.bfloat16).to(DEV) for _ in range(2))
    ang = torch.rand(800, d, generator=g) * 6
    cos, sin = ang.cos().to(DEV), ang.sin().to(DEV)
    pos = torch.randint(-3, 900, (tokens,), generator=g).to(torch.int32).to(DEV)
    pages = tokens + 5
    loc = torch.randperm(pages, generator=g)[:tokens].to(torch.int32)
    if tokens > 1:
        loc[0] = -1
    loc = loc.to(DEV)
    a, b = _pool(g, pages, hkv, d), None
    b = [x.clone() for x in a]
    q1, k1 = HipOps.qk_norm_rope(qkv, qw, kw, cos, sin, pos, hq, hkv, d, 1e-6)
    store_cache8(*a, loc, k1, qkv[:, (hq + hkv) * d:].view(tokens, hkv, d))
    q2 = HipOps.qk_norm_rope_append8(qkv, qw, kw, cos, sin, pos, hq, 1e-6, *b, loc)
    assert torch.equal(_bits(q1), _bits(q2))
    for x, y in zip(a, b):
        assert torch.equal(_bits(x), _bits(y))


# -- decode ------------------------------------------------------------------

def _decode_case(seed, hq, hkv, d, prefix, own, scattered=True, spare=11):
    g = torch.Generator().manual_seed(seed)
    b = len(own)
    total = prefix + sum(own)
    pages = total + spare
    ids = (torch.randperm(pages, generator=g) if scattered else torch.arange(pages))[:total]
    tails = ids[prefix:].split(list(own))
    indices = torch.cat([torch.cat((ids[:prefix], t)) for t in tails]).to(torch.int32)
    cu_k = _cu([prefix + n for n in own])
    q = (torch.randn(b, hq, d, generator=g) * 2).to(torch.bfloat16)
    return g, _pool(g, pages, hkv, d), q, indices, cu_k


def _run_decode(cache, q, indices, cu_k, hkv, prefix, **kw):
    b, hq, d = q.shape
    p = paged.plan("decode", torch.arange(b + 1, dtype=torch.int32), cu_k, hq, hkv, d,
                   shared_prefix_len=prefix, kv_bits=8, **kw)
    ws = torch.empty(p.ws_bytes, dtype=torch.uint8, device=DEV).fill_(255) if p.ws_bytes else None
    return p, ws, paged.decode8(p, q.to(DEV), *cache, indices.to(DEV), cu_k.to(DEV), workspace=ws)


DECODES = [
    # hq, hkv, d, prefix, own lengths, plan overrides
    (8, 2, 96, 24, [3, 1, 16, 7], {}),
    (8, 2, 96, 24, [3, 1, 16, 7], {"prefix_chunk_len": 32}),
    (12, 4, 64, 300, [1, 33, 64, 130, 2], {}),
    (16, 8, 128, 257, [1] * 9, {}),
    (32, 8, 128, 1000, [17, 5, 90, 1, 40, 64], {}),
    (32, 8, 128, 513, [3] * 40, {}),                       # two groups of 128 query rows
    (16, 8, 128, 0, [1], {}),
    (8, 1, 64, 0, [31, 32, 33, 1], {}),                    # group 8
    (8, 8, 128, 0, [65, 127, 128, 129], {}),               # group 1
    (6, 2, 96, 0, [700, 3], {}),                           # group 3
    (6, 1, 128, 0, [257, 256], {}),                        # group 6
    (12, 4, 64, 0, [2000, 1999, 5], {}),
    (32, 8, 128, 0, [4001], {}),
    (16, 8, 128, 0, [500, 20], {"suffix_split_len": 37}),  # items that end inside a sub-tile
    (8, 2, 96, 330, [260, 3], {"prefix_chunk_len": 96, "suffix_split_len": 50}),
]


@pytest.mark.parametrize("hq,hkv,d,prefix,own,kw", DECODES)
def test_decode_matches_oracle(hq, hkv, d, prefix, own, kw):
    g, cache, q, indices, cu_k = _decode_case(hq + d + prefix, hq, hkv, d, prefix, own)
    _, _, out = _run_decode(cache, q, indices, cu_k, hkv, prefix, **kw)
    want, tol = _oracle(q, *_values(*cache), indices, np.arange(len(own) + 1), cu_k)
    _near(out, want, tol)


@pytest.mark.parametrize("hq,hkv,d,prefix,own,kw", DECODES)
def test_append_decode_equals_its_two_calls(hq, hkv, d, prefix, own, kw):
    g, cache, q, indices, cu_k = _decode_case(7 + hq + d, hq, hkv, d, prefix, own)
    b = len(own)
    k = _rows(g, b, hkv, d).to(DEV)
    v = _rows(g, b, 3 * hkv, d).to(DEV)[:, hkv:2 * hkv]
    loc = indices[(cu_k[1:] - 1).long()].to(DEV)
    fused = [x.clone() for x in cache]
    store_cache8(*cache, loc, k, v)
    p, ws, want = _run_decode(cache, q, indices, cu_k, hkv, prefix, **kw)
    out = paged.append_decode8(p, q.to(DEV), k, v, loc, *fused, indices.to(DEV), cu_k.to(DEV),
                               workspace=ws)
    for x, y in zip(cache, fused):
        assert torch.equal(_bits(x), _bits(y))
    assert torch.equal(_bits(out), _bits(want))


@pytest.mark.parametrize("hq,hkv,d,prefix,own", [
    (8, 2, 96, 24, [3, 1, 16, 7]), (12, 4, 64, 300, [1, 33, 64, 130, 2]),
    (32, 8, 128, 1000, [17, 5, 90, 1, 40, 64]), (16, 8, 128, 0, [700, 20]), (8, 8, 64, 0, [9, 1])])
def test_append_decode_rope(hq, hkv, d, prefix, own):
    """Against qk_norm_rope's own rows: a head's sum of squares is taken in
    another order, which may move a normalised element by one bf16 step
    (2^-7), so the scores move by at most 2^-7 of sum |q k| and the codes of
    the new token by one step (2^-3 of a value)."""
    g, cache, q, indices, cu_k = _decode_case(hq + d, hq, hkv, d, prefix, own)
    b = len(own)
    qkv = _rows(g, b, hq + 2 * hkv, d, spread=0.2).view(b, -1).to(DEV)
    qw, kw = (torch.rand(d, generator=g).add(0.5).to(torch.bfloat16).to(DEV) for _ in range(2))
    ang = torch.rand(64, d // 2, generator=g).repeat(1, 2) * 6
    cos, sin = ang.cos().to(DEV), ang.sin().to(DEV)
    pos = torch.randint(0, 64, (b,), generator=g).to(torch.int32).to(DEV)
    q1, k1 = HipOps.qk_norm_rope(qkv, qw, kw, cos, sin, pos, hq, hkv, d, 1e-6)
    v = qkv[:, (hq + hkv) * d:].view(b, hkv, d)
    loc = indices[(cu_k[1:] - 1).long()].to(DEV)
    fused = [x.clone() for x in cache]
    store_cache8(*cache, loc, k1, v)
    p, ws, _ = _run_decode(cache, q1.cpu(), indices, cu_k, hkv, prefix)
    out = paged.append_decode_rope8(
        p, qkv[:, :hq * d].view(b, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(b, hkv, d), v, loc,
        *fused, indices.to(DEV), cu_k.to(DEV), qw, kw, cos.to(torch.bfloat16),
        sin.to(torch.bfloat16), pos, 1e-6, workspace=ws)
    assert torch.equal(_bits(cache[1]), _bits(fused[1]))
    same = (cache[0].view(torch.uint8) == fused[0].view(torch.uint8)).float().mean().item()
    assert same > 0.999
    assert torch.equal(_bits(cache[2]), _bits(fused[2]))
    want, tol = _oracle(q1.cpu(), *_values(*fused), indices, np.arange(b + 1), cu_k)
    bound = np.abs(to_np64(q1)).max() * np.abs(_values(*fused)[0]).max() * d ** 0.5
    got = to_np64(out)
    assert np.isfinite(got).all()
    # (a moved query element acts on all weights: relative 2^-7 |q k| at most)
    extra = 2 * 2.0 ** -7 * min(bound, 8.0) * (tol * 2 ** 8)
    assert (np.abs(got - want) <= tol + extra).all()


# -- prefill -----------------------------------------------------------------

PREFILLS = [
    # hq, hkv, d, (new, cached) of each request
    (8, 2, 96, [(32, 0)]), (12, 4, 64, [(64, 0)]), (16, 8, 128, [(1, 0)]),
    (16, 8, 128, [(2, 128)]), (8, 2, 96, [(1, 76)]), (8, 8, 64, [(5, 0)]),
    (8, 2, 96, [(3, 0), (1, 8), (40, 0), (17, 33), (0, 0), (0, 5)]),
    (32, 8, 128, [(100, 31), (33, 0)]),
    (8, 1, 64, [(17, 100)]), (6, 2, 96, [(45, 3)]), (6, 1, 128, [(23, 300)]),
    (32, 8, 128, [(6, 1501)]), (12, 4, 64, [(6, 1000), (1, 700)]), (16, 8, 128, [(17, 900)]),
    (32, 8, 128, [(100, 1700)]), (8, 2, 96, [(700, 0)]), (16, 8, 128, [(600, 65)]),
    # few rows, parts of several steps: one row tile and two, ragged ends
    (32, 8, 128, [(8 - i % 3, 1900 - 77 * i) for i in range(16)]),
    (12, 4, 64, [(15, 3000), (21, 1203), (1, 64)]),
    (8, 2, 96, [(10, 2500 - 131 * i) for i in range(9)]),
    (16, 8, 128, [(9, 600 - i) for i in range(40)]),
]


def _prefill_case(seed, hq, hkv, d, lens):
    g = torch.Generator().manual_seed(seed)
    new, kv = [a for a, _ in lens], [a + c for a, c in lens]
    pages = sum(kv) + 13
    indices = torch.randperm(pages, generator=g)[:sum(kv)].to(torch.int32)
    q = (torch.randn(sum(new), hq, d, generator=g) * 2).to(torch.bfloat16)
    return g, _pool(g, pages, hkv, d), q, indices, _cu(new), _cu(kv)


def _run_prefill(cache, q, indices, cu_q, cu_k, hkv, **kw):
    p = paged.plan("prefill", cu_q, cu_k, q.shape[1], hkv, q.shape[2], kv_bits=8, **kw)
    return p, paged.prefill8(p, q.to(DEV), *cache, indices.to(DEV), cu_q.to(DEV), cu_k.to(DEV))


@pytest.mark.parametrize("hq,hkv,d,lens", PREFILLS)
def test_prefill_matches_oracle(hq, hkv, d, lens):
    g, cache, q, indices, cu_q, cu_k = _prefill_case(hq + d, hq, hkv, d, lens)
    _, out = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    want, tol = _oracle(q, *_values(*cache), indices, cu_q, cu_k, weights=2)
    _near(out, want, tol)
    # and without room for partial states
    p, whole = _run_prefill(cache, q, indices, cu_q, cu_k, hkv, workspace_bytes=0)
    assert p.num_parts <= 1 and p.ws_bytes == 0
    _near(whole, want, tol)


@pytest.mark.parametrize("hq,hkv,d,lens", [
    (8, 8, 64, [(700 - 9 * i, 310 + 40 * i) for i in range(19)]),   # tiles of 256 tokens
    (12, 2, 96, [(330 - 7 * i, 700) for i in range(28)]),           # of 42
    (32, 8, 128, [(250 - i, 760 + i) for i in range(14)])])          # of 64
def test_prefill_in_wide_tiles(hq, hkv, d, lens):
    """Batches whose tiles hold 256 MFMA rows, the requests' ends inside them:
    a sample of the rows against the oracle, every row against batches of one
    request (whose tiles are the narrow ones)."""
    g, cache, q, indices, cu_q, cu_k = _prefill_case(hq + d, hq, hkv, d, lens)
    _, out = _run_prefill(cache, q, indices, cu_q, cu_k, hkv, workspace_bytes=0)
    for r in range(len(lens)):
        qs, ks = slice(int(cu_q[r]), int(cu_q[r + 1])), slice(int(cu_k[r]), int(cu_k[r + 1]))
        one = (_cu([lens[r][0]]), _cu([sum(lens[r])]))
        _, alone = _run_prefill(cache, q[qs], indices[ks], *one, hkv, workspace_bytes=0)
        assert torch.equal(out[qs], alone)
        if r in (0, len(lens) - 1):
            _near(alone, *_oracle(q[qs], *_values(*cache), indices[ks], *one, weights=2))


@pytest.mark.parametrize("prefix", [0, 320])
def test_lengths_on_the_device(prefix):
    """A plan built for the longest rows serves shorter ones (a captured step's
    lengths come from cu_k on the device), down to a row with no position."""
    hq, hkv, d = 16, 8, 128
    longest = [prefix + 700] * 3
    own = [700, 1, 40] if prefix else [700, 1, 0]
    g, cache, q, indices, cu_k = _decode_case(8, hq, hkv, d, prefix, own)
    p = paged.plan("decode", torch.arange(4, dtype=torch.int32), _cu(longest), hq, hkv, d,
                   shared_prefix_len=prefix, kv_bits=8)
    ws = torch.empty(p.ws_bytes, dtype=torch.uint8, device=DEV).fill_(255)
    idx = torch.cat((indices, torch.full((sum(longest) - len(indices),), -1, dtype=torch.int32)))
    out = paged.decode8(p, q.to(DEV), *cache, idx.to(DEV), cu_k.to(DEV), workspace=ws)
    want, tol = _oracle(q, *_values(*cache), indices, np.arange(4), cu_k)
    _near(out, want, tol)
    if not prefix:
        assert (out[2] == 0).all()
    cu_q = _cu([2, 1, 3])
    qp = (torch.randn(6, hq, d, generator=g) * 2).to(torch.bfloat16)
    kv = [prefix + max(3, n) for n in own]
    pp = paged.plan("prefill", cu_q, _cu([2000] * 3), hq, hkv, d, kv_bits=8)
    cu = _cu(kv)
    idx = torch.randint(0, cache[0].shape[0], (6000,), generator=g).to(torch.int32)
    out = paged.prefill8(pp, qp.to(DEV), *cache, idx.to(DEV), cu_q.to(DEV), cu.to(DEV))
    _near(out, *_oracle(qp, *_values(*cache), idx[:int(cu[-1])], cu_q, cu, weights=2))


# -- both --------------------------------------------------------------------

def test_pages_outside_the_pool_read_zeros():
    hq, hkv, d = 16, 8, 128
    g, cache, q, indices, cu_k = _decode_case(3, hq, hkv, d, 300, [40, 3])
    pages = cache[0].shape[0]
    indices[5], indices[100], indices[310] = -1, pages, 2 ** 30
    indices[340 + 5], indices[340 + 100] = -1, pages  # (the shared prefix, row 1)
    values = _values(*cache)
    for prefix in (300, 0):
        _, _, out = _run_decode(cache, q, indices, cu_k, hkv, prefix,
                                **({"prefix_chunk_len": 64} if prefix else {}))
        _near(out, *_oracle(q, *values, indices, np.arange(3), cu_k))
    cu_q = _cu([7, 1])
    q = (torch.randn(8, hq, d, generator=g)).to(torch.bfloat16)
    _, out = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    _near(out, *_oracle(q, *values, indices, cu_q, cu_k, weights=2))


@pytest.mark.parametrize("which", [0, 1])
def test_a_nan_token_reaches_only_the_rows_that_attend_to_it(which):
    """The token at position 40 of the second request holds a NaN (K or V): its
    earlier queries and the other request are as without it."""
    hq, hkv, d = 8, 2, 64
    g, cache, q, indices, cu_q, cu_k = _prefill_case(5, hq, hkv, d, [(70, 10), (60, 0)])
    _, clean = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    x = [torch.randn(1, hkv, d, generator=g).to(torch.bfloat16) for _ in range(2)]
    x[which][0, 1, 3] = float("nan")
    x[which][0, 1, 5] = float("inf")
    loc = indices[80 + 40:80 + 41].to(DEV)
    store_cache8(*cache, loc, x[0].to(DEV), x[1].to(DEV))
    _, out = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    assert torch.equal(_bits(out[:70 + 40]), _bits(clean[:70 + 40]))
    assert out[110:, 4:].isnan().all() and out[110:, :4].isfinite().all()
    # a decode over both requests' pages
    qd = q[:2]
    for prefix in (0, 0):
        _, _, dec = _run_decode(cache, qd, indices, cu_k, hkv, prefix)
        assert dec[0].isfinite().all()
        assert dec[1, 4:].isnan().all() and dec[1, :4].isfinite().all()


def test_last_pages_of_a_pool_beyond_2_gib():
    """Rows whose byte offsets need the 32nd bit, with records behind 2^24."""
    hq, hkv, d, pages = 16, 8, 128, 4_100_000  # 4.2e9 bytes of K codes
    g, small, q, indices, cu_q, cu_k = _prefill_case(9, hq, hkv, d, [(9, 141)])
    big = [torch.zeros(pages, hkv, d, dtype=torch.uint8, device=DEV).view(FP8) for _ in range(2)]
    scales = torch.zeros(hkv, pages, 2, dtype=torch.bfloat16, device=DEV)
    at = (indices.long() + pages - small[0].shape[0]).to(DEV)
    for b, s in zip(big, small):
        b.view(torch.uint8)[at] = s.view(torch.uint8)[indices.long().to(DEV)]
    scales[:, at] = small[2][:, indices.long().to(DEV)]
    far = at.to(torch.int32).cpu()
    _, want = _run_prefill(small, q, indices, cu_q, cu_k, hkv)
    _, out = _run_prefill((*big, scales), q, far, cu_q, cu_k, hkv)
    assert torch.equal(_bits(out), _bits(want))
    one = _cu([150])
    k, v = _rows(g, 1, hkv, d).to(DEV), _rows(g, 1, hkv, d).to(DEV)
    outs = []
    for cache, idx in ((small, indices), ((*big, scales), far)):
        p, ws, _ = _run_decode(cache, q[:1], idx, one, hkv, 0)
        outs.append(paged.append_decode8(p, q[:1].to(DEV), k, v, idx[-1:].to(DEV), *cache,
                                         idx.to(DEV), one.to(DEV), workspace=ws))
    assert torch.equal(_bits(outs[0]), _bits(outs[1]))
    assert torch.equal(_bits(big[0][at[-1]]), _bits(small[0][indices[-1].long()]))


def test_rows_behind_the_batch_are_left_alone():
    """A prefill and a decode write their own output rows only, and the pages
    of no other token."""
    hq, hkv, d = 12, 4, 64
    g, cache, q, indices, cu_q, cu_k = _prefill_case(2, hq, hkv, d, [(19, 3), (2, 400)])
    p = paged.plan("prefill", cu_q, cu_k, hq, hkv, d, kv_bits=8)
    buf = torch.full((q.shape[0] + 4, hq, d), 7.0, dtype=torch.bfloat16, device=DEV)
    was = [x.clone() for x in cache]
    paged.prefill8(p, q.to(DEV), *cache, indices.to(DEV), cu_q.to(DEV), cu_k.to(DEV),
                   out=buf[:q.shape[0]])
    assert (buf[q.shape[0]:] == 7).all()
    b = 2
    p, ws, _ = _run_decode(cache, q[:b], indices, cu_k, hkv, 0)
    paged.decode8(p, q[:b].to(DEV), *cache, indices.to(DEV), cu_k.to(DEV), workspace=ws,
                  out=buf[:b])
    assert (buf[q.shape[0]:] == 7).all()
    for x, y in zip(cache, was):
        assert torch.equal(_bits(x), _bits(y))


def test_a_captured_step_replays():
    """An appending decode and an extension in one graph, replayed on new
    inputs between eager calls, equal the eager results."""
    hq, hkv, d, prefix, own = 32, 8, 128, 513, [70, 64, 3]
    g, cache, q, indices, cu_k = _decode_case(4, hq, hkv, d, prefix, own)
    b = len(own)
    p = paged.plan("decode", torch.arange(b + 1, dtype=torch.int32), cu_k, hq, hkv, d,
                   shared_prefix_len=prefix, kv_bits=8)
    cu_q = _cu([1] * b)
    pp = paged.plan("prefill", cu_q, cu_k, hq, hkv, d, kv_bits=8)
    ws = torch.empty(p.ws_bytes, dtype=torch.uint8, device=DEV)
    qd, idx, cuk, cuq = q.to(DEV), indices.to(DEV), cu_k.to(DEV), cu_q.to(DEV)
    k, v = _rows(g, b, hkv, d).to(DEV), _rows(g, b, hkv, d).to(DEV)
    loc = indices[(cu_k[1:] - 1).long()].to(DEV)

    def step():
        a = paged.append_decode8(p, qd, k, v, loc, *cache, idx, cuk, workspace=ws)
        return a, paged.prefill8(pp, qd, *cache, idx, cuq, cuk)

    step()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = step()
    for i in range(4):
        qd.copy_((torch.randn(q.shape, generator=g) * 2).to(torch.bfloat16))
        k.copy_(_rows(g, b, hkv, d))
        graph.replay()
        got = [x.clone() for x in outs]
        want = step()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(_bits(x), _bits(y))


def test_calls_on_two_streams():
    hq, hkv, d = 16, 8, 128
    cases = []
    for seed in (1, 2):
        g, cache, q, indices, cu_q, cu_k = _prefill_case(seed, hq, hkv, d, [(300, 500)])
        cases.append((cache, q.to(DEV), indices.to(DEV), cu_q.to(DEV), cu_k.to(DEV),
                      paged.plan("prefill", cu_q, cu_k, hq, hkv, d, kv_bits=8)))
    run = lambda c: paged.prefill8(c[5], c[1], *c[0], *c[2:5])  # noqa: E731
    want = [run(c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        outs = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                outs.append(run(c))
        torch.cuda.synchronize()
        for x, y in zip(outs, want):
            assert torch.equal(_bits(x), _bits(y))


def test_a_cache_of_exact_values_gives_the_bf16_caches_outputs():
    """Rows of values that e4m3 holds: both caches' attention of one batch
    agree within both sides' weight roundings and the output's."""
    hq, hkv, d = 16, 8, 128
    g, cache, q, indices, cu_q, cu_k = _prefill_case(6, hq, hkv, d, [(130, 70), (4, 500)])
    kv, vv = _values(*cache)
    kb, vb = (torch.from_numpy(x).to(torch.bfloat16).to(DEV) for x in (kv, vv))
    p = paged.plan("prefill", cu_q, cu_k, hq, hkv, d)
    want16 = paged.prefill(p, q.to(DEV), kb, vb, indices.to(DEV), cu_q.to(DEV), cu_k.to(DEV))
    _, out = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    want, tol = _oracle(q, kv, vv, indices, cu_q, cu_k, weights=2)
    assert (np.abs(to_np64(out) - to_np64(want16)) <= 2 * tol).all()

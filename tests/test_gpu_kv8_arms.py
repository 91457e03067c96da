"""Attention over the 8-bit cache in the forms that long rows, long shared
prefixes and many parts take, and NaN tokens in each of them; bounds as in
tests/test_gpu_kv8.py.  Every case asserts from its plan that it takes the form
it is there for."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd import paged
from aios_amd.kernel import store_cache8
from aios_amd.layers import HipOps
from tests.test_gpu_kv8 import (DEV, _bits, _decode_case, _near, _oracle, _prefill_case, _rows,
                                _run_decode, _run_prefill, _values)

pytestmark = pytest.mark.gpu

# -- decode -------------------------------------------------------------------

# hq, hkv, d, prefix, own lengths, plan overrides, what the plan has to be
CHUNKS = [  # of the shared prefix, above 128 positions
    (32, 8, 128, 1000, [17, 5, 90, 1], {"prefix_chunk_len": 160}, 160),   # the last one 40
    (8, 2, 96, 577, [3, 40, 16, 7], {"prefix_chunk_len": 192}, 192),      # the last one 1
    (12, 4, 64, 600, [1, 33, 64, 130, 2, 9], {"prefix_chunk_len": 1000}, 608),
    (16, 8, 128, 513, [3] * 70, {"prefix_chunk_len": 256}, 256),          # two groups of 128 rows
    (8, 8, 64, 777, [9] * 17, {"prefix_chunk_len": 320}, 320),            # group 1
    (8, 1, 64, 400, [5, 300], {"prefix_chunk_len": 200, "suffix_split_len": 128}, 224),  # group 8
    (32, 8, 128, 2112, [2] * 40, {}, 192),                                # as planned
]
MANY = [  # more parts than the combine asks for at once
    (32, 8, 128, 0, [4096, 1, 2000], {"suffix_split_len": 64}, 64),
    (8, 2, 96, 0, [3100, 3100], {"suffix_split_len": 50}, 62),
    (8, 1, 128, 0, [4063], {"suffix_split_len": 64}, 64),     # group 8
    (6, 1, 128, 0, [1500], {"suffix_split_len": 32}, 47),                 # group 6
    (8, 2, 96, 1500, [260, 700, 1, 5], {"prefix_chunk_len": 32, "suffix_split_len": 48}, 62),
    (12, 4, 64, 1500, [600, 33, 2, 1, 8, 640], {"prefix_chunk_len": 32, "suffix_split_len": 40}, 63),
]
GROUPS = [  # states of groups 1, 6 and 8
    (8, 8, 128, 0, [700, 20, 129], {"suffix_split_len": 64}, 11),
    (8, 8, 96, 300, [7] * 16, {"prefix_chunk_len": 64}, 9),
    (6, 1, 64, 0, [700, 20, 129], {"suffix_split_len": 64}, 11),
    (12, 2, 96, 300, [40, 1, 9], {"prefix_chunk_len": 64}, 9),
    (8, 1, 128, 0, [700, 20, 129], {"suffix_split_len": 64}, 11),
    (16, 2, 96, 300, [40, 200], {"prefix_chunk_len": 64, "suffix_split_len": 64}, 9),
    (16, 2, 64, 333, [7, 70], {"prefix_chunk_len": 96}, 8),
]
DECODES = CHUNKS + MANY + GROUPS


def _expect(p, case):
    if case in CHUNKS:
        assert p.prefix_len and p.prefix_chunk_len == case[6] > 128
    else:
        assert p.num_parts == case[6]


@pytest.mark.parametrize("case", DECODES)
def test_decode(case):
    hq, hkv, d, prefix, own, kw, _ = case
    g, cache, q, indices, cu_k = _decode_case(hq + d + prefix + len(own), hq, hkv, d, prefix, own)
    p, _, out = _run_decode(cache, q, indices, cu_k, hkv, prefix, **kw)
    _expect(p, case)
    _near(out, *_oracle(q, *_values(*cache), indices, np.arange(len(own) + 1), cu_k))


@pytest.mark.parametrize("case", DECODES)
def test_append_decode_equals_its_two_calls(case):
    hq, hkv, d, prefix, own, kw, _ = case
    g, cache, q, indices, cu_k = _decode_case(3 + hq + d, hq, hkv, d, prefix, own)
    b = len(own)
    k, v = _rows(g, b, hkv, d).to(DEV), _rows(g, b, 2 * hkv, d).to(DEV)[:, hkv:]
    loc = indices[(cu_k[1:] - 1).long()].to(DEV)
    fused = [x.clone() for x in cache]
    store_cache8(*cache, loc, k, v)
    p, ws, want = _run_decode(cache, q, indices, cu_k, hkv, prefix, **kw)
    ws.fill_(255)
    out = paged.append_decode8(p, q.to(DEV), k, v, loc, *fused, indices.to(DEV), cu_k.to(DEV),
                               workspace=ws)
    for x, y in zip(cache, fused):
        assert torch.equal(_bits(x), _bits(y))
    assert torch.equal(_bits(out), _bits(want))


@pytest.mark.parametrize("case", DECODES)
def test_append_decode_rope_equals_its_two_calls(case):
    """The launch takes a head's sum of squares in another order than
    qk_norm_rope.  Projections that are small whole numbers have a sum that is
    exact in any order, so outputs and stored rows are equal bit for bit."""
    hq, hkv, d, prefix, own, kw, _ = case
    g, cache, q, indices, cu_k = _decode_case(hq + d, hq, hkv, d, prefix, own)
    b = len(own)
    qkv = torch.randint(-8, 9, (b, (hq + 2 * hkv) * d), generator=g).to(torch.bfloat16).to(DEV)
    qw, kw_ = (torch.rand(d, generator=g).add(0.5).to(torch.bfloat16).to(DEV) for _ in range(2))
    ang = torch.rand(64, d // 2, generator=g).repeat(1, 2) * 6
    cos, sin = ang.cos().to(DEV), ang.sin().to(DEV)
    pos = torch.randint(0, 64, (b,), generator=g).to(torch.int32).to(DEV)
    q1, k1 = HipOps.qk_norm_rope(qkv, qw, kw_, cos, sin, pos, hq, hkv, d, 1e-6)
    v = qkv[:, (hq + hkv) * d:].view(b, hkv, d)
    loc = indices[(cu_k[1:] - 1).long()].to(DEV)
    fused = [x.clone() for x in cache]
    store_cache8(*cache, loc, k1, v)
    p, ws, want = _run_decode(cache, q1.cpu(), indices, cu_k, hkv, prefix, **kw)
    _expect(p, case)
    ws.fill_(255)
    out = paged.append_decode_rope8(
        p, qkv[:, :hq * d].view(b, hq, d), qkv[:, hq * d:(hq + hkv) * d].view(b, hkv, d), v, loc,
        *fused, indices.to(DEV), cu_k.to(DEV), qw, kw_, cos.to(torch.bfloat16),
        sin.to(torch.bfloat16), pos, 1e-6, workspace=ws)
    for x, y in zip(cache, fused):
        assert torch.equal(_bits(x), _bits(y))
    assert torch.equal(_bits(out), _bits(want))


# -- prefill ------------------------------------------------------------------

PARTS = [  # few rows in more than 32 parts
    (12, 4, 64, [(6, 12000)]),
    (16, 4, 128, [(3, 15001)]),
    (8, 2, 96, [(5, 20000), (1, 3000)]),
    (8, 1, 64, [(7, 9000)]),
]


@pytest.mark.parametrize("hq,hkv,d,lens", PARTS)
def test_prefill_in_many_parts(hq, hkv, d, lens):
    g, cache, q, indices, cu_q, cu_k = _prefill_case(hq + d, hq, hkv, d, lens)
    p, out = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    assert p.num_parts > 32
    _near(out, *_oracle(q, *_values(*cache), indices, cu_q, cu_k, weights=2))


# -- NaN tokens ----------------------------------------------------------------

def _poison(cache, page, head, which):
    """A NaN scale, as a row with a NaN or an infinity has it."""
    cache = [x.clone() for x in cache]
    cache[2][head, page, which] = float("nan")
    return cache


def _only(out, clean, hit, group, head):
    """Rows ``hit`` are NaN in the heads of kv-head ``head``; all else as it was."""
    heads = slice(head * group, (head + 1) * group)
    assert out[hit][:, heads].isnan().all()
    rest = out.clone()
    rest[:, heads] = torch.where(hit[:, None, None], clean[:, heads], rest[:, heads])
    assert torch.equal(_bits(rest), _bits(clean))


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("case,at", [
    (CHUNKS[0], 170), (CHUNKS[0], 999), (CHUNKS[1], 576), (CHUNKS[2], 5),  # long chunks
    ((16, 8, 128, 300, [40, 3, 9, 1, 1, 1, 1, 1], {"prefix_chunk_len": 64}, 6), 100),  # short ones
    (GROUPS[5], 299), (MANY[4], 1499)])
def test_a_nan_in_the_shared_prefix(case, at, which):
    hq, hkv, d, prefix, own, kw, _ = case
    g, cache, q, indices, cu_k = _decode_case(hq, hq, hkv, d, prefix, own)
    p, _, clean = _run_decode(cache, q, indices, cu_k, hkv, prefix, **kw)
    assert p.prefix_len == prefix
    _, _, out = _run_decode(_poison(cache, int(indices[at]), hkv - 1, which), q, indices, cu_k, hkv,
                            prefix, **kw)
    _only(out, clean, torch.ones(len(own), dtype=torch.bool, device=DEV), hq // hkv, hkv - 1)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("case,row,at", [
    (MANY[0], 0, 4095), (MANY[0], 2, 63), (MANY[1], 1, 3000), (GROUPS[0], 0, 64), (GROUPS[2], 2, 128),
    (GROUPS[4], 0, 650), (MANY[5], 5, 600), (CHUNKS[0], 2, 89)])
def test_a_nan_in_a_rows_own_positions(case, row, at, which):
    hq, hkv, d, prefix, own, kw, _ = case
    g, cache, q, indices, cu_k = _decode_case(hq, hq, hkv, d, prefix, own)
    p, _, clean = _run_decode(cache, q, indices, cu_k, hkv, prefix, **kw)
    assert p.num_parts > 1
    page = int(indices[int(cu_k[row]) + prefix + at])
    _, _, out = _run_decode(_poison(cache, page, 0, which), q, indices, cu_k, hkv, prefix, **kw)
    _only(out, clean, torch.arange(len(own), device=DEV) == row, hq // hkv, 0)


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("hq,hkv,d,lens,at", [
    (32, 8, 128, [(6, 1501), (3, 40)], 700),      # few rows, in parts: a cached token,
    (32, 8, 128, [(6, 1501), (3, 40)], 1504),     # a new one
    (12, 4, 64, [(6, 12000)], 11999), (12, 4, 64, [(6, 12000)], 12003),
    (32, 8, 128, [(100, 1700)], 900), (32, 8, 128, [(100, 1700)], 1750)])
def test_a_nan_in_a_split_prefill(hq, hkv, d, lens, at, which):
    g, cache, q, indices, cu_q, cu_k = _prefill_case(hq + d, hq, hkv, d, lens)
    p, clean = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    assert p.num_parts > 1
    _, out = _run_prefill(_poison(cache, int(indices[at]), 1, which), q, indices, cu_q, cu_k, hkv)
    new, cached = lens[0]
    row = torch.arange(len(q), device=DEV)
    _only(out, clean, (row < new) & (cached + row >= at), hq // hkv, 1)

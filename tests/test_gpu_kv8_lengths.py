"""Decode over the 8-bit cache where the rows' lengths on the device are not
the plan's: a row may have outgrown its planned length, past the batch's longest
one, while the split of long rows was planned for fewer parts than that takes.
Bounds as in tests/test_gpu_kv8.py; the workspace starts as NaN, so a state
that is read without having been written shows."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd import paged
from aios_amd.kernel import store_cache8
from tests.test_gpu_kv8 import (DEV, _bits, _cu, _decode_case, _near, _oracle, _pool, _rows,
                                _values)

pytestmark = pytest.mark.gpu

CASES = [
    # hq, hkv, d, prefix, own lengths planned, own lengths on the device, plan overrides
    (16, 8, 128, 0, [700, 128, 300], [700, 129, 300], {"suffix_split_len": 128}),
    (16, 8, 128, 0, [700, 128, 300], [300, 900, 2000], {"suffix_split_len": 128}),
    (8, 2, 96, 0, [3000, 5], [5, 3000], {}),
    (32, 8, 128, 0, [4001, 1, 1], [4001, 4001, 4001], {}),
    (8, 8, 64, 0, [900, 130, 1], [4, 3000, 700], {"suffix_split_len": 96}),
    (8, 2, 96, 330, [260, 3, 40, 1], [3, 400, 300, 65], {"prefix_chunk_len": 96, "suffix_split_len": 50}),
    # rows planned with nothing behind the shared prefix
    (12, 4, 64, 300, [200, 0, 0, 0, 0, 0], [1, 150, 90, 33, 7, 64],
     {"prefix_chunk_len": 96, "suffix_split_len": 150}),
    # more rows than a wavefront has lanes
    (12, 4, 64, 0, [600] + [100] * 69, [300] * 70, {"suffix_split_len": 128}),
    (8, 8, 64, 0, [600] + [1] * 130, [1] * 65 + [200] * 65 + [900], {"suffix_split_len": 128}),
]


def _case(hq, hkv, d, prefix, planned, own, kw):
    g, cache, q, indices, cu_k = _decode_case(hq + d + sum(own), hq, hkv, d, prefix, own)
    b = len(own)
    p = paged.plan("decode", torch.arange(b + 1, dtype=torch.int32),
                   _cu([prefix + n for n in planned]), hq, hkv, d, shared_prefix_len=prefix,
                   kv_bits=8, **kw)
    assert p.num_parts > 1 and p.suffix_parts_per_item == 0  # (split)
    ws = torch.empty(p.ws_bytes, dtype=torch.uint8, device=DEV).fill_(255)
    # (the plan's number of page ids at least; the ones behind the rows are not read)
    idx = torch.cat((indices, torch.full((max(0, p.total_kv - len(indices)),), -1, dtype=torch.int32)))
    return g, cache, q, indices, cu_k, p, ws, idx.to(DEV)


@pytest.mark.parametrize("hq,hkv,d,prefix,planned,own,kw", CASES)
def test_rows_longer_than_planned(hq, hkv, d, prefix, planned, own, kw):
    g, cache, q, indices, cu_k, p, ws, idx = _case(hq, hkv, d, prefix, planned, own, kw)
    out = paged.decode8(p, q.to(DEV), *cache, idx, cu_k.to(DEV), workspace=ws)
    want, tol = _oracle(q, *_values(*cache), indices, np.arange(len(own) + 1), cu_k)
    _near(out, want, tol)


@pytest.mark.parametrize("hq,hkv,d,prefix,planned,own,kw",
                         [c for c in CASES if min(c[4]) > 0])
def test_appends_to_rows_longer_than_planned(hq, hkv, d, prefix, planned, own, kw):
    g, cache, q, indices, cu_k, p, ws, idx = _case(hq, hkv, d, prefix, planned, own, kw)
    b = len(own)
    k, v = _rows(g, b, hkv, d).to(DEV), _rows(g, b, hkv, d).to(DEV)
    loc = indices[(cu_k[1:] - 1).long()].to(DEV)
    fused = [x.clone() for x in cache]
    store_cache8(*cache, loc, k, v)
    want = paged.decode8(p, q.to(DEV), *cache, idx, cu_k.to(DEV), workspace=ws)
    ws.fill_(255)
    out = paged.append_decode8(p, q.to(DEV), k, v, loc, *fused, idx, cu_k.to(DEV), workspace=ws)
    for x, y in zip(cache, fused):
        assert torch.equal(_bits(x), _bits(y))
    assert torch.equal(_bits(out), _bits(want))
    _near(out, *_oracle(q, *_values(*cache), indices, np.arange(b + 1), cu_k))


def test_a_captured_step_whose_rows_grow():
    """One plan and one graph while every row grows by a token a step, over the
    border of a part and past the planned lengths."""
    hq, hkv, d, steps = 16, 8, 128, 6
    planned, start = [512, 256, 128], [510, 253, 126]
    g, cache, q, _, _ = _decode_case(3, hq, hkv, d, 0, [n + steps for n in start])
    pages = torch.arange(sum(start) + 3 * steps, dtype=torch.int32).split([n + steps for n in start])
    p = paged.plan("decode", torch.arange(4, dtype=torch.int32), _cu(planned), hq, hkv, d, kv_bits=8,
                   suffix_split_len=128)
    ws = torch.empty(p.ws_bytes, dtype=torch.uint8, device=DEV).fill_(255)
    qd, k, v = (torch.zeros(3, n, d, dtype=torch.bfloat16, device=DEV) for n in (hq, hkv, hkv))
    idx = torch.zeros(sum(len(x) for x in pages), dtype=torch.int32, device=DEV)
    cuk, loc = torch.zeros(4, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV)

    def fill(step):
        lens = [n + step for n in start]
        rows = [x[:n] for x, n in zip(pages, lens)]
        cuk.copy_(_cu(lens))
        idx[:sum(lens)].copy_(torch.cat(rows))
        loc.copy_(torch.stack([x[-1] for x in rows]))
        qn = (torch.randn(3, hq, d, generator=g) * 2).to(torch.bfloat16)
        qd.copy_(qn)
        k.copy_(_rows(g, 3, hkv, d))
        v.copy_(_rows(g, 3, hkv, d))
        return qn, torch.cat(rows), _cu(lens)

    fill(0)
    step_fn = lambda: paged.append_decode8(p, qd, k, v, loc, *cache, idx, cuk, workspace=ws)  # noqa: E731
    step_fn()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        out = step_fn()
    for step in range(steps + 1):
        qn, rows, cu = fill(step)
        ws.fill_(255)
        graph.replay()
        _near(out, *_oracle(qn, *_values(*cache), rows, np.arange(4), cu))


@pytest.mark.parametrize("hq,hkv,d,planned,lens", [
    # (new, cached) planned, and on the device
    (32, 8, 128, [(6, 1500), (6, 300)], [(6, 300), (5, 4000)]),    # few rows, in parts
    (8, 2, 96, [(10, 100)] * 3, [(10, 2000), (1, 0), (4, 700)]),   # few rows, planned whole
    (32, 8, 128, [(100, 1700)], [(70, 3000)]),                     # more rows, in parts
    (12, 4, 64, [(90, 10), (90, 0)], [(90, 1100), (50, 0)]),       # a workgroup per tile
])
def test_prefills_longer_than_planned(hq, hkv, d, planned, lens):
    g = torch.Generator().manual_seed(hq + d)
    kv = [a + c for a, c in lens]
    pages = sum(kv) + 13
    cache = _pool(g, pages, hkv, d)
    indices = torch.randperm(pages, generator=g)[:sum(kv)].to(torch.int32)
    cu_q, cu_k = _cu([a for a, _ in lens]), _cu(kv)
    q = (torch.randn(int(cu_q[-1]), hq, d, generator=g) * 2).to(torch.bfloat16)
    p = paged.plan("prefill", _cu([a for a, _ in planned]), _cu([a + c for a, c in planned]), hq, hkv,
                   d, kv_bits=8)
    idx = torch.cat((indices, torch.zeros(max(0, p.total_kv - len(indices)), dtype=torch.int32)))
    rows = torch.zeros(p.total_q, hq, d, dtype=torch.bfloat16)
    rows[:len(q)] = q
    out = paged.prefill8(p, rows.to(DEV), *cache, idx.to(DEV), cu_q.to(DEV), cu_k.to(DEV))
    _near(out[:len(q)], *_oracle(q, *_values(*cache), indices, cu_q, cu_k, weights=2))

"""Prefills over the 8-bit cache in tiles of 256 MFMA rows, by batches whose own
tiles reach the rule; bounds as in tests/test_gpu_kv8.py."""
from __future__ import annotations

import pytest
import torch

from aios_amd import paged
from tests.test_gpu_kv8 import DEV, _cu, _near, _oracle, _prefill_case, _run_prefill, _values

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hq,hkv,d,lens", [
    (12, 2, 96, [(330 - i, 700 - i) for i in range(28)]),                       # group 6: 42 tokens
    (12, 4, 64, [(620 - 3 * i, 450 + i) for i in range(16)]),                   # group 3: 84
    (32, 8, 128, [(1, 0), (2048, 0), (0, 7)] + [(200 + i, 3) for i in range(12)]),
    (16, 2, 64, [(530, 600 + i) for i in range(15)])])                          # group 8: 32
def test_wide_tiles_of_requests_of_different_lengths(hq, hkv, d, lens):
    """Every row as in the narrow tiles, a sample against the oracle."""
    g, cache, q, indices, cu_q, cu_k = _prefill_case(hq + d, hq, hkv, d, lens)
    p, out = _run_prefill(cache, q, indices, cu_q, cu_k, hkv)
    assert p.num_parts == 0 and p.prefill_q_tile * p.group > 128
    for r, (new, cached) in enumerate(lens):
        if new == 0:
            continue
        qs, ks = slice(int(cu_q[r]), int(cu_q[r + 1])), slice(int(cu_k[r]), int(cu_k[r + 1]))
        one = (_cu([new]), _cu([new + cached]))
        pn, alone = _run_prefill(cache, q[qs], indices[ks], *one, hkv, workspace_bytes=0)
        if pn.num_parts == 0:  # (few rows share their sub-tiles: other sums)
            assert pn.prefill_q_tile * pn.group <= 128
            assert torch.equal(out[qs], alone)
        if new < 700 and r % 7 == 0:
            _near(out[qs], *_oracle(q[qs], *_values(*cache), indices[ks], *one, weights=2))


def test_wide_tiles_of_shorter_requests_than_planned():
    hq, hkv, d = 32, 8, 128
    planned, lens = [(4096, 0), (100, 0)], [(100, 900), (700, 0)]
    g, cache, q, indices, cu_q, cu_k = _prefill_case(5, hq, hkv, d, lens)
    p = paged.plan("prefill", _cu([a for a, _ in planned]), _cu([a + c for a, c in planned]), hq, hkv,
                   d, kv_bits=8)
    assert p.prefill_q_tile * p.group > 128
    rows = torch.zeros(p.total_q, hq, d, dtype=torch.bfloat16)
    rows[:len(q)] = q
    idx = torch.cat((indices, torch.full((p.total_kv - len(indices),), -1, dtype=torch.int32)))
    buf = torch.full((p.total_q, hq, d), 7.0, dtype=torch.bfloat16, device=DEV)
    out = paged.prefill8(p, rows.to(DEV), *cache, idx.to(DEV), cu_q.to(DEV), cu_k.to(DEV), out=buf)
    _near(out[:len(q)], *_oracle(q, *_values(*cache), indices, cu_q, cu_k, weights=2))
    assert (out[len(q):] == 7).all()

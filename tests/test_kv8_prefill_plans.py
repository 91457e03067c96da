"""Which prefills over the 8-bit cache take tiles of 256 MFMA rows, by the plan
(no GPU: 256 units)."""
from __future__ import annotations

import pytest
import torch

from aios_amd import paged


def _plan(lens, hq=32, hkv=8, d=128, **kw):
    cu = [torch.tensor([0, *x]).cumsum(0) for x in ([a for a, _ in lens], [a + c for a, c in lens])]
    return paged.plan("prefill", *cu, hq, hkv, d, kv_bits=8, **kw)


@pytest.mark.parametrize("lens,kw,wide", [
    ([(4096, 0)], {}, True),
    ([(3500, 0)], {}, True),                              # 440 workgroups
    ([(2048, 0)], {}, False),                             # 256
    # the requests' own tiles count, not the longest one's for each
    ([(2048, 0)] + [(40, 0)] * 3, {}, False),             # 280
    ([(2048, 0)] + [(100, 0)] * 7, {}, False),            # 368
    ([(1000, 200)] + [(20, 500)] * 15, {}, False),        # 248
    ([(2048, 0)] + [(200, 0)] * 12, {}, True),            # 640
    ([(0, 50), (4096, 0), (0, 0)], {}, True),
    ([(300, 0)] * 16, {}, False),                         # short ones
    ([(330 - i, 700) for i in range(28)], dict(hq=12, hkv=2, d=96), True),
    ([(330 - 7 * i, 700) for i in range(28)], dict(hq=12, hkv=2, d=96), False)])  # 344
def test_wide_tiles_by_the_requests_own(lens, kw, wide):
    p = _plan(lens, **kw)
    rows = p.prefill_q_tile * p.group
    assert p.num_parts == 0 and p.ws_bytes == 0
    assert (128 < rows <= 256) if wide else (64 < rows <= 128)
    longest = max(a for a, _ in lens)
    assert (p.num_q_tiles - 1) * p.prefill_q_tile < longest <= p.num_q_tiles * p.prefill_q_tile


def test_a_split_prefill_keeps_its_tiles():
    p = _plan([(700, 1800)])
    assert p.num_parts > 1 and p.prefill_q_tile * p.group <= 128

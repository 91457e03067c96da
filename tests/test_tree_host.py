"""Trees of drafted tokens without a GPU: plans, the oracle's masks, and the
refusals of the C ABI and of the Python entry points."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd import _lib, paged
from oracle import tree as otree

INVALID, UNSUPPORTED, OK = _lib.AIOS_ERR_INVALID, _lib.AIOS_ERR_UNSUPPORTED, _lib.AIOS_OK


def _plan(nodes, cached, hq=16, hkv=8, d=128, bits=16, page=1, ws=1 << 30):
    cu_q = np.cumsum([0, *nodes]).astype(np.int32)
    cu_k = np.cumsum([0, *(n + c for n, c in zip(nodes, cached))]).astype(np.int32)
    p = _lib.AttnPlan()
    rc = _lib.lib().aios_attn_plan_tree(cu_q.ctypes.data, cu_k.ctypes.data, len(nodes), hq, hkv, d,
                                        page, bits, ws, p)
    return rc, p


def test_the_oracle_s_masks():
    seen = otree.ancestors([-1, 0, 0, 1, 9, 4])
    assert seen == [{0}, {0, 1}, {0, 2}, {0, 1, 3}, {4}, {4, 5}]
    w = otree.mask_words([{0, 63}, {64, 127, 200}], 2)
    assert w.view(np.uint64).tolist() == [[1 | 1 << 63, 0], [0, 1 | 1 << 63]]


@pytest.mark.parametrize("bits,phase", [(16, _lib.PHASE_TREE), (8, _lib.PHASE_TREE8)])
def test_plans(bits, phase):
    for nodes in ([1], [40], [256, 3], [33] * 7):
        rc, p = _plan(nodes, [100] * len(nodes), bits=bits)
        assert rc == OK and p.phase == phase and p.total_q == sum(nodes)
        # every node has a tile, no tile more than 128 MFMA rows, a part more sub-tiles than 0
        assert p.prefill_q_tile * p.num_q_tiles >= max(nodes)
        assert p.prefill_q_tile * p.group <= 128 and p.prefix_chunk_len >= 32 and p.num_parts >= 1
    assert _plan([], [])[0] == OK and _plan([0, 0], [5, 0])[0] == OK


def test_plan_refusals():
    assert _plan([257], [0])[0] == UNSUPPORTED
    assert _plan([3], [5], bits=4)[0] == INVALID
    assert _plan([3], [5], page=16)[0] == UNSUPPORTED
    assert _plan([3], [5], hq=15)[0] == INVALID
    assert _plan([3], [5], d=80)[0] == UNSUPPORTED
    assert _plan([3], [-1])[0] == INVALID  # fewer positions than nodes
    many = torch.arange((1 << 21) + 1, dtype=torch.int32)  # 2^24 tiles: 2^32 threads
    with pytest.raises(ValueError, match="too many tiles"):
        paged.plan("tree", many, many, 8, 8, 64)
    for kw in ({"shared_prefix_len": 4}, {"prefix_chunk_len": 64}, {"suffix_split_len": 64}):
        with pytest.raises(ValueError, match="takes no shared prefix"):
            paged.plan("tree", [0, 3], [0, 8], 16, 8, 128, **kw)
    with pytest.raises(ValueError, match="257 nodes"):
        paged.plan("tree", [0, 257], [0, 300], 16, 8, 128)


def _call(p, bits=16, q=64, kc=64, idx=64, masks=64, words=1, out=64, pages=100, stride=2048,
          scale=0.1):
    lib = _lib.lib()
    tail = (idx, idx, idx, masks, words, out, None, 0, scale, None)
    if bits == 16:
        return lib.aios_attn_tree(p, q, stride, kc, kc, pages, *tail)
    return lib.aios_attn_tree8(p, q, stride, kc, kc, kc, pages, *tail)


@pytest.mark.parametrize("bits", [16, 8])
def test_c_refusals(bits):
    """(addresses are never followed: every call is refused)"""
    _, p = _plan([70], [10], bits=bits)
    call = lambda **kw: _call(p, bits, **{"words": 2, **kw})
    assert call(stride=2040) == INVALID and call(stride=2052) == INVALID
    for name in ("q", "kc", "idx", "masks", "out"):
        assert call(**{name: None}) == INVALID, name
    assert call(q=8) == INVALID and call(out=72) == INVALID and call(masks=68) == INVALID
    assert call(kc=72) == INVALID
    assert call(words=1) == INVALID and call(words=0) == INVALID and call(words=5) == INVALID
    assert call(pages=-1) == INVALID and call(pages=1 << 24) == UNSUPPORTED
    assert call(pages=(1 << 32) // (1024 * bits // 8)) == UNSUPPORTED
    for scale in (0.0, -1.0, float("inf"), float("nan")):
        assert call(scale=scale) == INVALID
    other = _plan([70], [10], bits=24 - bits)[1]
    assert _call(other, bits, words=2) == INVALID
    assert _call(None, bits, words=2) == INVALID
    empty = _plan([0], [10], bits=bits)[1]
    assert _call(empty, bits, q=None) == OK  # nothing to do


def test_masks_c_refusals():
    f = _lib.lib().aios_tree_masks
    assert f(64, 64, -1, 5, 1, 64, 64, None) == INVALID
    assert f(64, 64, 1, -5, 1, 64, 64, None) == INVALID
    assert f(64, 64, 1, 5, 0, 64, 64, None) == INVALID and f(64, 64, 1, 5, 5, 64, 64, None) == INVALID
    assert f(64, 64, 1, 5, 1, 68, 64, None) == INVALID
    for i in (0, 1, 5, 6):
        args = [64, 64, 1, 5, 1, 64, 64, None]
        args[i] = None
        assert f(*args) == INVALID
    assert f(None, None, 0, 0, 1, None, None, None) == OK


def _tensors(bits, n=3, kv=8, hq=16, hkv=8, d=128):
    q = torch.zeros(n, hq, d, dtype=torch.bfloat16)
    if bits == 16:
        cache = [torch.zeros(10, hkv, d, dtype=torch.bfloat16) for _ in range(2)]
    else:
        cache = [torch.zeros(10, hkv, d).to(torch.float8_e4m3fn) for _ in range(2)]
        cache.append(torch.zeros(hkv, 10, 2, dtype=torch.bfloat16))
    lists = [torch.zeros(kv, dtype=torch.int32), torch.tensor([0, n], dtype=torch.int32),
             torch.tensor([0, kv], dtype=torch.int32)]
    return q, cache, lists, torch.zeros(n, 1, dtype=torch.int64)


@pytest.mark.parametrize("bits", [16, 8])
def test_python_refusals(bits):
    f = paged.tree_attention if bits == 16 else paged.tree_attention8
    plan = paged.plan("tree", [0, 3], [0, 8], 16, 8, 128, kv_bits=bits)
    q, cache, lists, masks = _tensors(bits)
    with pytest.raises(ValueError):  # tensors of the host
        f(plan, q, *cache, *lists, masks)
    for other in (paged.plan("prefill", [0, 3], [0, 8], 16, 8, 128, kv_bits=bits),
                  paged.plan("tree", [0, 3], [0, 8], 16, 8, 128, kv_bits=24 - bits)):
        with pytest.raises(ValueError, match="plan was not built for trees"):
            f(other, q, *cache, *lists, masks)
    with pytest.raises(ValueError):  # a plan for trees is none for the prefill
        paged.prefill(plan, q, *cache[:2], *lists)


def test_masks_python_refusals():
    cu = torch.tensor([0, 3], dtype=torch.int32)
    for n in (0, 257):
        with pytest.raises(ValueError, match="max_nodes"):
            paged.tree_masks(torch.zeros(3, dtype=torch.int32), cu, n)
    with pytest.raises(ValueError, match="parents"):
        paged.tree_masks(torch.zeros(3, dtype=torch.int32), cu, 3)  # of the host

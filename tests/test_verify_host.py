"""Verification of drafted tokens without a GPU: the oracle's rule and the
refusals of the C ABI and of the Python entry point."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd import _lib
from aios_amd.sample import verify_drafts
from oracle import tree as otree

INVALID, UNSUPPORTED, OK = _lib.AIOS_ERR_INVALID, _lib.AIOS_ERR_UNSUPPORTED, _lib.AIOS_OK


@pytest.mark.parametrize("drawn", [True, False])
def test_the_oracle_keeps_the_target_s_distribution(drawn):
    """The probability of every first token, by adding up the rule's branches over
    a grid of the random numbers."""
    p_log, q_log = np.array([0.5, -0.2, 0.1]), np.array([-0.3, 0.6, 0.0])
    p = np.exp(p_log) / np.exp(p_log).sum()
    q = np.exp(q_log) / np.exp(q_log).sum()
    m, got = 60, np.zeros(3)
    grid = (np.arange(m) + 0.5) / m
    logits = np.stack((p_log, p_log))
    for x in range(3):
        for u0 in grid:
            for u1 in grid:
                r = otree.verify(logits, np.stack((q_log, q_log)) if drawn else None,
                                 np.array([0, x]), [-1, 0], [0, 2], np.array([u0, u1]), 1.0)
                first = x if r["counts"][0] else r["next"][0]
                got[first] += (q[x] if drawn else 1 / 3) / m ** 2
    assert np.abs(got - p).max() < 2 / m


def test_the_oracle_s_sums_in_closed_form():
    """p behind j rejected children is max(p - l_j q, 0) / F(l_j)."""
    rng = np.random.default_rng(0)
    p, q = rng.dirichlet(np.ones(9)), rng.dirichlet(np.ones(9))
    now, lam, f = p, 0.0, 1.0
    for _ in range(4):
        now = np.maximum(now - q, 0)
        now = now / now.sum()
        lam += f
        f = np.maximum(p - lam * q, 0).sum()
        assert np.abs(now - np.maximum(p - lam * q, 0) / f).max() < 1e-9


def _call(**kw):
    a = dict(logits=64, stride=100, draft=64, dstride=100, vocab=100, elem=2, tokens=64,
             parents=64, cu=64, batch=2, total=9, u=64, temp=1.0, dtemp=1.0, accepted=64,
             counts=64, last=64, next=64, lp=64, ws=64, ws_bytes=1 << 40, stream=None)
    a.update(kw)
    return _lib.lib().aios_verify_drafts(*a.values())


def test_c_refusals():
    """(addresses are never followed: every call is refused)"""
    for kw in ({"batch": -1}, {"total": -1}, {"vocab": 0}, {"stride": 99}, {"stride": -1},
               {"dstride": 99}, {"dstride": -2}, {"temp": -1.0}, {"temp": 1e-5}, {"temp": 2e4},
               {"temp": float("nan")}, {"temp": float("inf")}, {"dtemp": 0.0},
               {"dtemp": float("nan")}, {"logits": 65}, {"draft": 65}, {"logits": 66, "elem": 4}):
        assert _call(**kw) == INVALID, kw
    for name in ("logits", "tokens", "parents", "cu", "u", "accepted", "counts", "last", "next", "lp"):
        assert _call(**{name: None}) == INVALID, name
    assert _call(elem=1) == UNSUPPORTED and _call(total=(1 << 24) + 1) == UNSUPPORTED
    assert _call(vocab=(1 << 30) + 1, stride=1 << 31, dstride=1 << 31) == UNSUPPORTED
    assert _call(batch=(1 << 31) - 1, vocab=1 << 30, stride=1 << 30, dstride=0) == UNSUPPORTED
    big = dict(vocab=151936, stride=151936, dstride=151936)
    for kw in ({"ws": None}, {"ws": 72}, {"ws_bytes": 100}):
        assert _call(**big, **kw) == _lib.AIOS_ERR_WORKSPACE, kw
    assert _call(batch=0, total=0, logits=None, ws=None) == OK
    assert _call(batch=0) == INVALID  # (nodes that no request owns, and no launch to say so)
    # launches of 2^32 threads and more
    assert _call(total=1 << 24) == UNSUPPORTED
    assert _call(total=1 << 23, draft=None, ws=None) == _lib.AIOS_ERR_WORKSPACE
    assert _call(batch=1 << 23, draft=None) == UNSUPPORTED


def test_workspace_sizes():
    f = _lib.lib().aios_verify_workspace
    assert f(0, 9, 100, 1) == 0 and f(2, -1, 100, 1) == 0 and f(2, 9, 0, 1) == 0
    v = 151936
    assert 0 < f(2, 9, 100, 0) < f(2, 9, 100, 1) < f(2, 9, v, 0) < f(2, 9, v, 1) < f(2, 90, v, 1) < f(4, 90, v, 1)
    need = f(2, 9, v, 1)
    assert _call(vocab=v, stride=v, dstride=v, ws_bytes=need - 1) == _lib.AIOS_ERR_WORKSPACE


def test_python_refusals():
    n, v = 4, 10
    x = torch.zeros(n, v)
    tok, par = torch.zeros(n, dtype=torch.int64), torch.zeros(n, dtype=torch.int32)
    cu, u = torch.tensor([0, n], dtype=torch.int32), torch.zeros(n)
    with pytest.raises(ValueError, match="GPU"):
        verify_drafts(x, tok, par, cu, u)

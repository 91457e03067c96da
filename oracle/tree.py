"""Oracle: attention of trees of drafted tokens, and their verification, in
float64 (test infrastructure only)."""
from __future__ import annotations

import numpy as np


def ancestors(parents) -> list[set[int]]:
    """What each node of one tree sees: itself and the nodes that it continues
    (a parent that is not an earlier node counts as none)."""
    seen: list[set[int]] = []
    for i, p in enumerate(parents):
        seen.append({i} | (seen[p] if 0 <= p < i else set()))
    return seen


def mask_words(seen, words: int) -> np.ndarray:
    """int64 [nodes, words]: bit j % 64 of word j / 64 for every j in a node's set."""
    out = np.zeros((len(seen), words), dtype=np.uint64)
    for i, s in enumerate(seen):
        for j in s:
            if j < 64 * words:
                out[i, j // 64] |= np.uint64(1) << np.uint64(j % 64)
    return out.view(np.int64)


def tree_attention(q, k_cache, v_cache, indices, cu_q, cu_k, seen, sm_scale) -> np.ndarray:
    """q [nodes, Hq, D], caches [pages, Hkv, D] (a page outside them is a row of
    zeros), seen: for every node the set of nodes of its request that it sees.
    A node attends to those and to all positions before the request's nodes;
    nothing else is looked at; without any position the output is 0."""
    pages, hkv, d = k_cache.shape
    group = q.shape[1] // hkv
    out = np.zeros(q.shape, dtype=np.float64)
    for r in range(len(cu_q) - 1):
        q0, q1, k0, k1 = (int(x) for x in (cu_q[r], cu_q[r + 1], cu_k[r], cu_k[r + 1]))
        cached = (k1 - k0) - (q1 - q0)
        idx = np.asarray(indices[k0:k1], dtype=np.int64)
        ok = (idx >= 0) & (idx < pages)
        k = np.where(ok[:, None, None], k_cache[np.where(ok, idx, 0)], 0.0)
        v = np.where(ok[:, None, None], v_cache[np.where(ok, idx, 0)], 0.0)
        for i in range(q1 - q0):
            at = [*range(cached), *(cached + j for j in sorted(seen[q0 + i]) if j < q1 - q0)]
            if not at:
                continue
            kk = np.repeat(k[at], group, axis=1)
            vv = np.repeat(v[at], group, axis=1)
            with np.errstate(invalid="ignore", over="ignore"):
                s = np.einsum("hd,khd->hk", q[q0 + i], kk) * sm_scale
                p = np.exp(s - s.max(-1, keepdims=True))
                out[q0 + i] = np.einsum("hk,khd->hd", p / p.sum(-1, keepdims=True), vv)
    return out

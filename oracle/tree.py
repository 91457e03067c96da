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


def _softmax(x, t):
    with np.errstate(over="ignore"):
        x = x / t
        e = np.exp(x - x.max())
    return e / e.sum()


def _log_softmax(x):
    d = x - x.max()
    return d - np.log(np.exp(d).sum())


def verify(logits, draft, tokens, parents, cu, u, t, td=None) -> dict:
    """The acceptance rule, one request after the other, with p normalised anew
    behind every rejected child.  logits, draft (or None) float64 [nodes, vocab]."""
    n, vocab = logits.shape
    td = t if td is None else td
    out = {"accepted": np.zeros(n, bool), "counts": [], "last": [], "next": [],
           "logprobs": np.full(n, np.nan)}

    def good(row):
        return np.isfinite(row.max()) and not np.isnan(row).any()

    for f, e in zip(cu[:-1], cu[1:]):
        f, size = int(f), min(int(e) - int(f), 256)
        if size <= 0:
            for k, v in (("counts", 0), ("last", -1), ("next", -1)):
                out[k].append(v)
            continue
        par = [int(parents[f + i]) for i in range(size)]
        kids = [[i for i in range(v + 1, size) if par[i] == v] for v in range(size)]
        for v in range(size):
            if kids[v] and good(logits[f + v]):
                lp = _log_softmax(logits[f + v])
                for i in kids[v]:
                    if 0 <= tokens[f + i] < vocab:
                        out["logprobs"][f + i] = lp[tokens[f + i]]
        v, count = 0, 0
        out["accepted"][f] = True
        while True:
            row = logits[f + v]
            if not good(row):
                pick = -1
                break
            step = None
            if t == 0:
                pick = int(np.argmax(row))
                step = next((i for i in kids[v] if tokens[f + i] == pick), None)
            else:
                p = whole = _softmax(row, t)
                usable = draft is None or good(draft[f + v])
                for i in kids[v] if usable else ():
                    x = int(tokens[f + i])
                    q = np.zeros(vocab)
                    if draft is not None:
                        q = _softmax(draft[f + v], td)
                    elif 0 <= x < vocab:
                        q[x] = 1.0
                    if 0 <= x < vocab and u[f + i] * q[x] < p[x]:
                        step = i
                        break
                    p = np.maximum(p - q, 0.0)
                    p = p / p.sum() if p.sum() > 0 else p
                if step is None:
                    p = p if p.sum() > 0 else whole
                    over = np.nonzero(np.cumsum(p) > u[f] * p.sum())[0]
                    pick = int(over[0]) if len(over) else int(np.nonzero(p)[0][-1])
            if step is None:
                break
            v, count = step, count + 1
            out["accepted"][f + v] = True
        if pick >= 0:
            out["logprobs"][f] = _log_softmax(row)[pick]
        for k, x in (("counts", count), ("last", v), ("next", pick)):
            out[k].append(x)
    return out

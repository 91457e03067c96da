"""token_logprobs on rows that are split over workgroups: rows without a finite
maximum, ids outside the vocabulary, excluded segments (the joining launch's own
handling); bounds as in tests/test_gpu_logprobs.py."""
from __future__ import annotations

import numpy as np
import pytest
import torch

from aios_amd import _lib
from aios_amd.sample import token_logprobs
from tests.test_gpu_logprobs import DEV, TOL, _check, _logits, _want

pytestmark = pytest.mark.gpu
VOCABS = pytest.mark.parametrize("vocab", [40001, 151936, 300001])
DTYPES = pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])


def _split(x, top):
    assert _lib.lib().aios_token_logprobs_workspace(*x.shape, top) > 0


@VOCABS
@DTYPES
@pytest.mark.parametrize("top", [0, 3, 20])
def test_rows_without_a_finite_maximum(vocab, dtype, top):
    """One row of each kind, the odd logit in the first, a middle and the last
    segment; the rows beside them are as they would be alone."""
    spots = [5, vocab // 2, vocab - 1]
    inf = float("inf")
    kinds = [("nan", i) for i in spots] + [("inf", i) for i in spots] + [("both", i) for i in spots]
    x, tok = _logits(len(kinds) + 3, vocab, dtype, vocab)
    _split(x, top)
    for r, (kind, i) in enumerate(kinds):
        x[r, i] = inf if kind == "inf" else float("nan")
        if kind == "both":
            x[r, (i + vocab // 3) % vocab] = inf
    x[len(kinds)] = -inf
    bad = len(kinds) + 1
    r = token_logprobs(x, tok, top=top)
    for out in (r.logprobs, r.entropies, r.top_logprobs):
        assert out[:bad].isnan().all() and out[bad:].isfinite().all()
    got, ent, ids, alt = _want(x[bad:], tok[bad:], top)
    for a, b in ((r.logprobs, got), (r.entropies, ent), (r.top_logprobs, alt)):
        np.testing.assert_allclose(a[bad:].double().cpu().numpy(), b, atol=TOL, rtol=TOL)
    np.testing.assert_array_equal(r.top_ids[bad:].cpu().numpy(), ids)
    if top:
        for row, (kind, i) in enumerate(kinds):
            assert r.top_ids[row, 0] == i  # (a NaN before anything, then an infinity)
        assert (r.top_ids[len(kinds)] == torch.arange(top, device=DEV)).all()


@VOCABS
@DTYPES
def test_tokens_outside_the_vocabulary(vocab, dtype):
    x, tok = _logits(5, vocab, dtype, 4)
    _split(x, 2)
    tok[:] = torch.tensor([-1, vocab, 2 ** 40, vocab - 1, 0])
    r = _check(x, tok, 2)
    assert r.logprobs[:3].isnan().all() and r.logprobs[3:].isfinite().all()


@VOCABS
def test_segments_of_excluded_ids(vocab):
    """All but one segment at -inf, the likely ids in the first, a middle and the
    last one; a token of an excluded segment is impossible."""
    x, tok = _logits(4, vocab, torch.float32, 6)
    _split(x, 5)
    low = float("-inf")
    keep = [slice(0, 50), slice(vocab // 2, vocab // 2 + 7), slice(vocab - 5, vocab)]
    for r, k in enumerate(keep):
        row = torch.full((vocab,), low, device=DEV)
        row[k] = x[r, k]
        x[r] = row
        tok[r] = k.start + 1
    tok[3] = 17
    x[3, 17] = low
    r = token_logprobs(x, tok, top=5)
    got, ent, ids, alt = _want(x, tok, 5)
    assert r.logprobs[3] == low
    for a, b in ((r.logprobs[:3], got[:3]), (r.entropies, ent), (r.top_logprobs, alt)):
        np.testing.assert_allclose(a.double().cpu().numpy(), b, atol=TOL, rtol=TOL)
    np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ids)

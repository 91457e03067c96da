"""token_logprobs against float64.

Tolerances, with Z = sum e^(x - m), T = sum e^(x - m) (x - m): an fp32 term has
a relative error of at most 2^-21 (the difference, the product with log2 e and
the exponential), a thread adds up to n / 256 of them in fp32 one batch at a
time (each sum's rounding 2^-24 of itself, at most 64 in a row), and all that
joins threads, wavefronts and segments adds 2^-20 more.  So |d ln Z| <= 2^-18 and
|d T / Z| <= 2^-18 |T / Z| + 2^-18, and a result is rounded to fp32 (2^-24)."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from aios_amd import _lib
from aios_amd.sample import token_logprobs

pytestmark = pytest.mark.gpu
DEV = "cuda"
TOL = 2.0 ** -17


def _want(x, tokens, top):
    """(log probabilities, entropies, ids, their log probabilities) of the rows
    (without a NaN) in float64."""
    x = x.double()
    d = x - x.amax(-1, keepdim=True)
    p = d.exp()
    z = p.sum(-1, keepdim=True)
    lp = d - z.log()
    ent = z[:, 0].log() - (p * torch.where(p > 0, d, 0.0)).sum(-1) / z[:, 0]
    ids = torch.sort(x, dim=-1, descending=True, stable=True).indices[:, :top]
    ok = (tokens >= 0) & (tokens < x.shape[1])
    got = lp.gather(1, torch.where(ok, tokens, 0)[:, None])[:, 0]
    got = torch.where(ok, got, float("nan"))
    return [t.cpu().numpy() for t in (got, ent, ids, lp.gather(1, ids))]


def _check(logits, tokens, top):
    r = token_logprobs(logits, tokens, top=top)
    got, ent, ids, alt = _want(logits, tokens, top)
    assert r.logprobs.dtype == r.entropies.dtype == r.top_logprobs.dtype == torch.float32
    assert r.top_ids.shape == r.top_logprobs.shape == (logits.shape[0], top)
    for name, a, b in (("logprobs", r.logprobs, got), ("entropies", r.entropies, ent),
                       ("top_logprobs", r.top_logprobs, alt)):
        np.testing.assert_allclose(a.double().cpu().numpy(), b, atol=TOL, rtol=TOL, err_msg=name)
    np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ids)
    return r


def _logits(rows, vocab, dtype, seed, spread=3.0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    x = torch.randn(rows, vocab, generator=g, device=DEV)
    x *= torch.rand(rows, 1, generator=g, device=DEV) * spread
    tok = torch.randint(vocab, (rows,), generator=g, device=DEV)
    tok[::3] = x[::3].argmax(-1)
    return x.to(dtype), tok


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("rows,vocab,top", [
    (1, 1, 1), (3, 2, 2), (2, 7, 7), (5, 33, 32), (4, 511, 5), (3, 512, 1), (2, 513, 20),
    (9, 2048, 8), (5, 10007, 8), (24, 16384, 0), (1, 151936, 32), (7, 151936, 5), (3, 131071, 3),
    (600, 6400, 2), (520, 2049, 32), (2, 300001, 6), (2, 1100003, 9), (513, 270001, 3)])
def test_matches_float64(rows, vocab, top, dtype):
    _check(*_logits(rows, vocab, dtype, rows * vocab), top)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_go_to_the_lower_id(dtype):
    vocab = 40001
    x = torch.zeros(4, vocab, dtype=dtype, device=DEV)
    x[1] = (torch.arange(vocab, device=DEV) % 5).to(dtype)
    x[2, 20000:] = 1.0
    x[3] = -torch.zeros(vocab, device=DEV).to(dtype)  # -0 and +0 are equal
    x[3, 1::2] = 0.0
    tok = torch.tensor([0, 4, 39999, 7], device=DEV)
    for rows in (slice(0, 4), slice(0, 1)):  # (split in segments either way)
        r = _check(x[rows], tok[rows], 32)
        assert r.top_ids[0].tolist() == list(range(32))
    big = torch.zeros(600, vocab, dtype=dtype, device=DEV)  # (a workgroup per row)
    r = token_logprobs(big, torch.zeros(600, dtype=torch.long, device=DEV), top=9)
    assert (r.top_ids == torch.arange(9, device=DEV)).all()
    assert torch.allclose(r.entropies, torch.full_like(r.entropies, math.log(vocab)), atol=TOL)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("low", ["inf", "lowest"])
def test_excluded_ids(dtype, low):
    low = float("-inf") if low == "inf" else torch.finfo(dtype).min
    x, tok = _logits(6, 30011, dtype, 5)
    x[0, 5:] = low           # five left
    x[1, :] = low
    x[1, 29000] = 2.0        # one left
    x[2, ::2] = low
    x[3, 8192:] = low        # whole segments without an id
    x[4, :30000] = low
    tok[0], tok[1], tok[2], tok[3] = 7, 29000, 0, 3
    if low == float("-inf"):
        r = token_logprobs(x, tok, top=4)
        assert r.logprobs[0] == low and r.logprobs[2] == low
        assert r.logprobs[1] == 0 and r.entropies[1] == 0
        assert r.top_ids[1].tolist() == [29000, 0, 1, 2]
        assert r.top_logprobs[1].tolist() == [0.0, low, low, low]
        keep = torch.tensor([0, 2, 3, 4, 5], device=DEV)
        got, ent, ids, alt = _want(x[keep], tok[keep], 4)
        np.testing.assert_allclose(r.logprobs[keep].cpu().double().numpy(), got, atol=TOL, rtol=TOL)
        np.testing.assert_allclose(r.entropies[keep].cpu().double().numpy(), ent, atol=TOL, rtol=TOL)
        np.testing.assert_array_equal(r.top_ids[keep].cpu().numpy(), ids)
    else:
        r = token_logprobs(x, tok, top=4)
        assert r.entropies.isfinite().all() and r.entropies[1] == 0
        assert r.top_ids[1].tolist() == [29000, 0, 1, 2]
        got, ent, ids, _ = _want(x, tok, 4)
        np.testing.assert_allclose(r.entropies.cpu().double().numpy(), ent, atol=TOL, rtol=TOL)
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ids)


@pytest.mark.parametrize("rows", [3, 700])
def test_rows_without_a_finite_maximum_and_bad_tokens(rows):
    x, tok = _logits(rows, 9001, torch.float32, 3)
    x[0] = float("-inf")
    x[1, 4000] = float("nan")
    x[2, 8000] = float("inf")
    r = token_logprobs(x, tok, top=3)
    for out in (r.logprobs, r.entropies, r.top_logprobs):
        assert out[:3].isnan().all()
        assert out[3:].isfinite().all()
    assert r.top_ids[0].tolist() == [0, 1, 2]
    assert r.top_ids[1, 0] == 4000 and r.top_ids[2, 0] == 8000
    y, tok = _logits(4, 9001, torch.float32, 4)
    tok[:] = torch.tensor([-1, 9001, 2 ** 40, 9000])
    r = _check(y, tok, 2)
    assert r.logprobs[:3].isnan().all() and r.logprobs[3].isfinite()


def test_strided_and_broadcast_rows():
    x, tok = _logits(5, 3000, torch.bfloat16, 8)
    wide = torch.zeros(5, 3005, dtype=torch.bfloat16, device=DEV)
    wide[:, 3:3003] = x
    want = _check(x, tok, 6)
    r = token_logprobs(wide[:, 3:3003], tok, top=6)
    assert torch.equal(r.logprobs, want.logprobs) and torch.equal(r.top_ids, want.top_ids)
    one = x[:1].expand(5, -1)
    r = token_logprobs(one, tok, top=6)
    _check(one, tok, 6)
    assert (r.entropies == r.entropies[0]).all()
    e = token_logprobs(x[:0], tok[:0], top=6)
    assert e.logprobs.shape == (0,) and e.top_ids.shape == (0, 6)


@pytest.mark.parametrize("rows,vocab", [(1, 1000), (2, 151936), (600, 9000)])
def test_peaked_rows_keep_small_values(rows, vocab):
    """ln Z = ln(1 + z) and T / Z of a row with one likely id are as exact as
    the sum z of its small terms: relative 2^-18 (above), not 2^-24 of 1."""
    x = torch.full((rows, vocab), -20.0, device=DEV)
    x[:, 17] = 0.0
    x[:, 20:900:7] = -23.5
    tok = torch.full((rows,), 17, device=DEV)
    r = token_logprobs(x, tok, top=1)
    n = len(range(20, 900, 7))
    z = n * math.exp(-23.5) + (vocab - 1 - n) * math.exp(-20)
    t = -23.5 * n * math.exp(-23.5) - 20 * (vocab - 1 - n) * math.exp(-20)
    lz = math.log1p(z)
    for got, want in ((r.logprobs, -lz), (r.top_logprobs[:, 0], -lz),
                      (r.entropies, lz - t / (1 + z))):
        assert (got.double() - want).abs().max().item() <= 2.0 ** -18 * abs(want)
    assert (r.top_ids == 17).all()


def test_without_a_workspace_and_in_a_graph():
    x, tok = _logits(3, 151936, torch.bfloat16, 1)
    want = _check(x, tok, 5)
    lib = _lib.lib()
    assert lib.aios_token_logprobs_workspace(3, 151936, 5) > 0
    lp = torch.empty(2, 3, device=DEV)
    ids, alt = torch.empty(3, 5, dtype=torch.long, device=DEV), torch.empty(3, 5, device=DEV)
    rc = lib.aios_token_logprobs(x.data_ptr(), x.stride(0), 3, 151936, 2, tok.data_ptr(), 5,
                                 lp.data_ptr(), lp[1].data_ptr(), ids.data_ptr(), alt.data_ptr(),
                                 None, 0, torch.cuda.current_stream().cuda_stream)
    assert rc == 0
    assert torch.equal(ids, want.top_ids)
    assert (lp[0] - want.logprobs).abs().max() < TOL
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        r = token_logprobs(x, tok, top=5)
    for seed in range(3):
        y, t = _logits(3, 151936, torch.bfloat16, seed + 10)
        x.copy_(y)
        tok.copy_(t)
        graph.replay()
        got = [v.clone() for v in (r.logprobs, r.entropies, r.top_ids, r.top_logprobs)]
        w = token_logprobs(x, tok, top=5)
        for a, b in zip(got, (w.logprobs, w.entropies, w.top_ids, w.top_logprobs)):
            assert torch.equal(a, b)

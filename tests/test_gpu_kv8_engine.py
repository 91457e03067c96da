"""The 8-bit pool behind the attention backend, the CandidateGroup engine over
it, and the scoring of given continuations.

Attention outputs are held to the bounds of tests/test_gpu_kv8.py on the codes
the pool holds.  Whole models are compared with the float32 oracle, whose
attention is given the pool's own K and V values, so that what differs is the
bf16 arithmetic of the trunk and not the rounding to 8 bits: logits within the
0.125 that a bf16 model's are held to, hence log-probs (a difference of a logit
and a logsumexp) and their averages within twice that.
"""
from __future__ import annotations

import math
from dataclasses import replace
from types import SimpleNamespace

import pytest
import torch

from aios_amd.attention import Mi355xAttentionBackend
from aios_amd.config import MINIMIND_ATTNRES_0P214B, MINIMIND_IME_0P1B, QWEN3_0P6B
from aios_amd.core import Batch, Context, Req, SamplingParams, reset_global_ctx, set_global_ctx
from aios_amd.ime import CandidateGroupConfig, CandidateGroupEngine, CandidateGroupRuntime
from aios_amd.kvcache import MHAKVCache8
from aios_amd.qwen3 import init_weights, weights_to
from oracle import kv8 as okv8
from oracle.model import OracleModel, _rms, _rope
from tests.test_gpu_kv8 import _cu, _near, _oracle, _rows, _values
from tests.util import to_np64

pytestmark = pytest.mark.gpu
LOGIT_TOL = 0.125
QWEN3 = replace(QWEN3_0P6B, num_layers=4, vocab_size=8192)
CONFIGS = pytest.mark.parametrize(
    "config", [MINIMIND_IME_0P1B.with_layers(4), QWEN3, MINIMIND_ATTNRES_0P214B],
    ids=["minimind-ime-h64-g3", "qwen3-0.6b-h128-g2", "minimind-attnres"])


def teardown_function(_):
    reset_global_ctx()
    torch.cuda.empty_cache()


class PoolOracle(OracleModel):
    """The oracle reading K and V of positions 0.. from ``self.kv`` (one pair of
    [L, Hkv, D] for each layer) instead of computing them."""

    def _attention(self, lw, x):
        c = self.c
        _, n, _ = x.shape
        hq, hkv, d = c.num_qo_heads, c.num_kv_heads, c.head_dim
        i = next(j for j, w in enumerate(self.w["layers"]) if w is lw)
        q = (x @ lw["qkv"].T)[..., : hq * d].reshape(1, n, hq, d)
        q = _rope(_rms(q, lw["q_norm"], c.rms_norm_eps), torch.arange(n), c.rope_theta)[0]
        k, v = (t[:n].repeat_interleave(hq // hkv, dim=1) for t in self.kv[i])
        s = (q.transpose(0, 1) @ k.permute(1, 2, 0)) * d ** -0.5
        s = s.masked_fill(~torch.ones(n, n, dtype=torch.bool).tril(), float("-inf"))
        o = s.softmax(-1) @ v.transpose(0, 1)
        return o.transpose(0, 1).reshape(1, n, hq * d) @ lw["o"].T


def _pool_kv(rt, row, n):
    """K and V of a page-table row's first n positions, for each layer."""
    pages = rt.page_table[row, :n].long().cpu()
    out = []
    for i in range(rt.config.num_layers):
        k, v = _values(*rt.kv_cache.layer(i))
        out.append((torch.from_numpy(k[pages]).float(), torch.from_numpy(v[pages]).float()))
    return out


def _engine(config, use_graphs, kv_bits=8, seed=3, **kw):
    w = init_weights(config, seed, "cpu")
    rt = CandidateGroupRuntime(config, weights_to(w, "cuda"), "cuda", num_pages=512,
                               kv_bits=kv_bits, **kw)
    return CandidateGroupEngine(rt, use_graphs=use_graphs), w


def _ids(config, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(config.vocab_size, (n,), generator=g).tolist()


def _logits(config, w, rt, row, ids):
    """The oracle's logits after each of ids[0..], on row's pool contents."""
    om = PoolOracle(config, w)
    om.kv = _pool_kv(rt, row, len(ids))
    return om.logits(torch.tensor(ids)[None], 0)[0]


@CONFIGS
@pytest.mark.parametrize("use_graphs", [False, True])
def test_candidate_groups_over_the_8_bit_pool(config, use_graphs):
    eng, w = _engine(config, use_graphs)
    rt = eng.rt
    assert isinstance(rt.kv_cache, MHAKVCache8)
    cfg = CandidateGroupConfig(num_candidates=4, max_new_tokens=6)
    text = _ids(config, 75, 5)
    for n in (70, 75):  # a prefix, then its extension (and in graphs, replays)
        prefix = text[:n]
        res = eng.complete(prefix, cfg)
        assert res.reused_prefix_tokens == (0 if n == 70 else 70)
        assert rt.cache_manager.available_size == rt.num_pages - n
        for r, cand in enumerate(res.raw_candidates):
            ref = _logits(config, w, rt, r, prefix + list(cand.token_ids[:-1]))[n - 1 :]
            got = res.prefix_logits[0].float().cpu()
            assert (got - ref[0]).abs().max().item() <= LOGIT_TOL
            lp = ref.log_softmax(-1).gather(1, torch.tensor(cand.token_ids)[:, None])
            assert abs(lp.mean().item() - cand.average_logprob) <= 2 * LOGIT_TOL
            gap = ref[1:].max(-1).values - ref[1:].gather(1, torch.tensor(cand.token_ids)[1:, None])[:, 0]
            assert gap.max().item() <= 2 * LOGIT_TOL  # greedy, up to both logits' errors


@CONFIGS
def test_scores_over_the_8_bit_pool(config):
    eng, w = _engine(config, False)
    rt = eng.rt
    prefix = _ids(config, 61, 7)
    conts = [_ids(config, n, 20 + n) for n in (1, 9, 2, 1, 33)]
    out = eng.score(prefix, conts, top=5)
    assert rt.cache_manager.available_size == rt.num_pages - len(prefix)
    rows = [i for i, c in enumerate(conts) if len(c) > 1]
    for i, (c, s) in enumerate(zip(conts, out)):
        assert s.token_ids == tuple(c)
        # (rows of the batch are the continuations that feed tokens, in order;
        # a single token needs the prefix alone)
        row = rows.index(i) if i in rows else 0
        ref = _logits(config, w, rt, row, prefix + c[:-1])[len(prefix) - 1 :].log_softmax(-1)
        for t in range(len(c)):
            assert abs(s.logprobs[t] - ref[t, c[t]].item()) <= 2 * LOGIT_TOL
            assert len(s.alternatives[t]) == 5
            for k, (tok, lp) in enumerate(s.alternatives[t]):
                assert abs(lp - ref[t, tok].item()) <= 2 * LOGIT_TOL
                assert abs(lp - ref[t].topk(5).values[k].item()) <= 2 * LOGIT_TOL
            assert s.logprobs[t] <= s.alternatives[t][0][1]
    # the same call again: the prefix is kept, nothing else is
    again = eng.score(prefix, conts, top=5)
    assert again == out
    assert eng.score(prefix, []) == ()
    assert rt.cache_manager.available_size == rt.num_pages - len(prefix)
    # and a completion after it starts from the same prefix
    res = eng.complete(prefix, CandidateGroupConfig(num_candidates=3, max_new_tokens=3))
    assert res.reused_prefix_tokens == len(prefix)


def test_scores_beyond_the_page_tables_rows():
    """More continuations than rows of the page table, bfloat16 pool."""
    config = MINIMIND_IME_0P1B.with_layers(4)
    eng, w = _engine(config, True, kv_bits=16, max_attempts=4)
    prefix = _ids(config, 37, 9)
    conts = [_ids(config, 1 + n % 4, 40 + n) for n in range(11)]
    om = OracleModel(config, w)
    for c, s in zip(conts, eng.score(prefix, conts)):
        ref = om.logits(torch.tensor(prefix + c)[None], len(prefix) - 1)[0].log_softmax(-1)
        want = [ref[t, c[t]].item() for t in range(len(c))]
        assert max(abs(a - b) for a, b in zip(want, s.logprobs)) <= 2 * LOGIT_TOL
        entropy = -(ref.exp() * ref).sum(-1)
        # log p off by at most e: |dH| <= sum p (e^e - 1)(|log p| + e) + p e, and sum p |log p| <= ln V
        e = 2 * LOGIT_TOL
        bound = math.expm1(e) * (math.log(config.vocab_size) + e) + e
        assert max(abs(a - b) for a, b in zip(entropy.tolist(), s.entropies)) <= bound
        assert s.alternatives == ()
        assert abs(s.average_logprob - sum(s.logprobs) / len(c)) < 1e-12
    assert eng.rt.cache_manager.available_size == eng.rt.num_pages - len(prefix)


# -- the backend ------------------------------------------------------------

SHAPE = SimpleNamespace(num_qo_heads=12, num_kv_heads=4, head_dim=64)


class _Wrapped:
    """A pool reached through another object."""

    def __init__(self, pool):
        self._pool = pool

    def __getattr__(self, name):
        return getattr(self._pool, name)


def _backend(pages, rows, length, layers=2):
    be = Mi355xAttentionBackend(SHAPE)
    ctx = Context(page_size=1)
    ctx.kv_cache = MHAKVCache8(SHAPE.num_kv_heads, layers, SHAPE.head_dim, pages, 1,
                               torch.float8_e4m3fn, "cuda")
    ctx.attn_backend = be
    ctx.page_table = torch.zeros((rows, length), dtype=torch.int32, device="cuda")
    set_global_ctx(ctx)
    return be, ctx


def _batch(phase, cached, new):
    reqs = [Req(input_ids=torch.empty(c + n, dtype=torch.long), cached_len=c, output_len=1, uid=r,
                sampling_params=SamplingParams(max_tokens=1), table_idx=r)
            for r, (c, n) in enumerate(zip(cached, new))]
    return Batch(reqs=reqs, phase=phase)


def _forward(be, ctx, pool, batch, g, layer, heads=SHAPE):
    """One forward of random rows, checked: the stored rows bit for bit, the
    outputs on the values the pool holds."""
    new = [r.extend_len for r in batch.reqs]
    t = sum(new)
    q = _rows(g, t, heads.num_qo_heads, heads.head_dim)
    k, v = _rows(g, t, heads.num_kv_heads, heads.head_dim), _rows(g, t, heads.num_kv_heads, heads.head_dim)
    out = be.forward(q.cuda(), k.cuda(), v.cuda(), pool, layer, batch)
    kk, vv = _values(*ctx.kv_cache.layer(layer))
    loc = batch.out_loc.cpu().long()
    for held, x in ((kk, k), (vv, v)):
        codes, s = okv8.quantize_rows(to_np64(x))
        assert (held[loc] == codes * s[..., None]).all()
    lens = [r.device_len for r in batch.reqs]
    idx = torch.cat([ctx.page_table[r, :n] for r, n in enumerate(lens)])
    want, tol = _oracle(q, kk, vv, idx, _cu(new), _cu(lens), weights=2)
    _near(out.view(t, heads.num_qo_heads, heads.head_dim), want, tol)


@pytest.mark.parametrize("wrapped", [False, True])
@pytest.mark.parametrize("fused", [False, True])
def test_backend_over_the_8_bit_pool(fused, wrapped):
    be, ctx = _backend(400, 3, 160)
    pool = _Wrapped(ctx.kv_cache) if wrapped else ctx.kv_cache
    ctx.kv_cache = pool
    g = torch.Generator().manual_seed(11)
    free = torch.randperm(400, generator=g).to(torch.int32).cuda()
    cached, new = [0, 0, 0], [70, 1, 33]
    at = 0
    for step in range(4):
        phase = "prefill" if step in (0, 2) else "decode"
        new = [[70, 1, 33], [1, 1, 1], [5, 17, 2], [1, 1, 1]][step]
        batch = _batch(phase, cached, new)
        loc = free[at : at + sum(new)]
        at += sum(new)
        for r, part in enumerate(loc.split(new)):
            ctx.page_table[r, cached[r] : cached[r] + new[r]] = part
        batch.out_loc = loc
        batch.fused_append = fused and phase == "decode"
        be.prepare_metadata(batch)
        assert batch.attn_metadata.dtype == torch.float8_e4m3fn
        for layer in (1, 0):
            _forward(be, ctx, pool, batch, g, layer)
        cached = [c + n for c, n in zip(cached, new)]


def test_static_plans_of_a_named_cache():
    """kv_bits names the cache where no context does."""
    be, ctx = _backend(64, 2, 64)
    table = ctx.page_table
    ids = torch.arange(2, device="cuda")
    assert be.prepare_static_decode(ids, 64, 0, table).dtype == torch.float8_e4m3fn
    assert be.prepare_static_decode(ids, 64, 0, table, kv_bits=16).dtype == torch.bfloat16
    reset_global_ctx()
    assert be.prepare_static_decode(ids, 64, 0, table).dtype == torch.bfloat16
    assert be.prepare_static_prefill(3, 64, table, kv_bits=8).dtype == torch.float8_e4m3fn
    with pytest.raises(ValueError):
        be.prepare_static_prefill(3, 64, table, kv_bits=4)


def test_a_plan_of_the_other_cache_is_refused():
    be, ctx = _backend(64, 2, 64)
    batch = _batch("prefill", [0], [4])
    batch.out_loc = torch.arange(4, dtype=torch.int32, device="cuda")
    batch.attn_metadata = be.prepare_static_prefill(4, 64, ctx.page_table, kv_bits=16)
    q = torch.zeros(4, 12, 64, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="8-bit"):
        be.forward(q, q[:, :4], q[:, :4], ctx.kv_cache, 0, batch)

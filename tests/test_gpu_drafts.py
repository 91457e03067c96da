"""A model over trees of drafts (append with rotation, tree attention, verification)
and the engine that decodes with them, over both pools.

Logits of every node are held to the float32 oracle on the tokens of its path, with
the bf16 model's 0.125 (over the 8-bit pool on the K and V that the pool holds);
log-probs and their averages to twice that.
"""
from __future__ import annotations

from dataclasses import replace

import pytest
import torch

from aios_amd.config import MINIMIND_ATTNRES_0P214B, MINIMIND_IME_0P1B, QWEN3_0P6B
from aios_amd.core import Batch, Req, SamplingParams, reset_global_ctx
from aios_amd.drafts import DraftTree, PhraseDrafter, draft_tree
from aios_amd.ime import CandidateGroupConfig, CandidateGroupEngine, CandidateGroupRuntime
from aios_amd.qwen3 import init_weights, weights_to
from aios_amd.sample import sample_step, stateless_uniforms
from oracle.model import OracleModel
from tests.test_gpu_kv8 import _values
from tests.test_gpu_kv8_engine import PoolOracle

pytestmark = pytest.mark.gpu
LOGIT_TOL = 0.125
QWEN3 = replace(QWEN3_0P6B, num_layers=3, vocab_size=8192)
IME = MINIMIND_IME_0P1B.with_layers(3)
CONFIGS = pytest.mark.parametrize("config", [IME, QWEN3, MINIMIND_ATTNRES_0P214B],
                                  ids=["minimind-ime-h64-g3", "qwen3-0.6b-h128-g2",
                                       "minimind-attnres"])
BITS = pytest.mark.parametrize("kv_bits", [16, 8])


def teardown_function(_):
    reset_global_ctx()
    torch.cuda.empty_cache()


def _engine(config, kv_bits, seed=3, num_pages=512, use_graphs=True):
    w = init_weights(config, seed, "cpu")
    rt = CandidateGroupRuntime(config, weights_to(w, "cuda"), "cuda", num_pages=num_pages,
                               kv_bits=kv_bits)
    return CandidateGroupEngine(rt, use_graphs), w


def _ids(config, n, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(config.vocab_size, (n,), generator=g).tolist()


def _oracle(config, w, rt, ids, pages):
    """The oracle's logits behind the last of ids, whose K/V rows lie in pages."""
    if rt.kv_cache.dtype == torch.bfloat16:
        return OracleModel(config, w).logits(torch.tensor(ids)[None], 0)[0, -1]
    om = PoolOracle(config, w)
    om.kv = []
    for i in range(config.num_layers):
        k, v = _values(*rt.kv_cache.layer(i))
        om.kv.append((torch.from_numpy(k[pages]).float(), torch.from_numpy(v[pages]).float()))
    return om.logits(torch.tensor(ids)[None], 0)[0, -1]


def _greedy_up_to_rounding(config, w, prefix, tokens):
    """Every token's logit is within both sides' errors of the oracle's largest (two
    launches' logits differ, so their tokens need not be the same)."""
    n = len(prefix) - 1
    ref = OracleModel(config, w).logits(torch.tensor(prefix + tokens[:-1])[None], 0)[0, n:]
    gap = ref.max(-1).values - ref.gather(1, torch.tensor(tokens)[:, None])[:, 0]
    assert gap.max().item() <= 2 * LOGIT_TOL
    return ref


def _give_logits(rt, table):
    """The forward runs as ever, and then the logits of position p are row p of a table,
    so that no launch's rounding enters."""
    forward = rt.model.forward

    def with_table():
        b = rt.ctx.batch
        rows = forward().shape[0]
        at = b.positions if rows == b.positions.numel() else b.positions[-1:]
        return table[at.long()]

    rt.model.forward = with_table


@CONFIGS
@BITS
def test_a_batch_of_trees_gives_every_path_s_logits(config, kv_bits):
    eng, w = _engine(config, kv_bits)
    rt = eng.rt
    prefixes = [_ids(config, 41, 1), _ids(config, 7, 2)]
    parents = [[-1, 0, 1, 0, 3, 3, -1], [-1, 0, 0]]
    news = [_ids(config, len(p), 5 + i) for i, p in enumerate(parents)]
    held = []
    for r, ids in enumerate(prefixes):  # the prefixes, one after the other
        pages = rt.cache_manager.allocate(len(ids))
        rt.page_table[r, : len(ids)] = pages
        b = Batch(reqs=[Req(input_ids=torch.empty(len(ids), dtype=torch.long), cached_len=0,
                            output_len=1, uid=r, sampling_params=SamplingParams(), table_idx=r)],
                  phase="prefill")
        b.input_ids = torch.tensor(ids, device="cuda")
        b.positions = torch.arange(len(ids), dtype=torch.int32, device="cuda")
        b.out_loc = pages
        with torch.inference_mode():
            rt.model.attn_backend.prepare_metadata(b)
            with rt.ctx.forward_batch(b):
                rt.model.forward()
        held.append(pages)
    own = rt.cache_manager.allocate(10)
    depths, paths = [], []
    for p in parents:
        for i, x in enumerate(p):
            path = [i]
            while p[path[0]] >= 0:
                path.insert(0, p[path[0]])
            paths.append(path)
            depths.append(len(path) - 1)
    cached = [41] * 7 + [7] * 3
    rt.page_table[0, 41:48] = own[:7]
    rt.page_table[1, 7:10] = own[7:]
    b = Batch(reqs=[Req(input_ids=torch.empty(c + len(n), dtype=torch.long), cached_len=c,
                        output_len=1, uid=i, sampling_params=SamplingParams(), table_idx=i)
                    for i, (c, n) in enumerate(zip((41, 7), news))], phase="prefill")
    b.input_ids = torch.tensor(sum(news, []), device="cuda")
    b.positions = torch.tensor([c + d for c, d in zip(cached, depths)], dtype=torch.int32,
                               device="cuda")
    b.out_loc = own
    b.return_all_logits = True
    b.tree_parents = parents
    with torch.inference_mode():
        rt.model.attn_backend.prepare_metadata(b)
        with rt.ctx.forward_batch(b):
            logits = rt.model.forward()
    assert logits.shape[0] == 10
    for row, path in enumerate(paths):
        r = 0 if row < 7 else 1
        base = 0 if r == 0 else 7
        ids = prefixes[r] + [news[r][i] for i in path]
        pages = torch.cat((held[r], own[base + torch.tensor(path, device="cuda")])).long().cpu()
        want = _oracle(config, w, rt, ids, pages)
        assert (logits[row].float().cpu() - want).abs().max() <= LOGIT_TOL


@CONFIGS
@BITS
@pytest.mark.parametrize("use_graphs", [True, False])
def test_greedy_tokens_with_drafts(config, kv_bits, use_graphs):
    eng, w = _engine(config, kv_bits, use_graphs=use_graphs)
    rt = eng.rt
    prefix = _ids(config, 33, 9)
    cfg = CandidateGroupConfig(max_new_tokens=9)
    plain = eng.complete_drafted(prefix, lambda context, room: None, cfg)
    assert rt.cache_manager.available_size == rt.num_pages - len(prefix)
    tokens = list(plain.candidate.token_ids)
    assert len(tokens) == 9 and plain.passes == 8 and plain.drafted == 0
    assert plain.candidate.stop_reason == "max_new_tokens"
    if kv_bits == 16:
        ref = _greedy_up_to_rounding(config, w, prefix, tokens)
        lp = ref.log_softmax(-1).gather(1, torch.tensor(tokens)[:, None]).mean().item()
        assert abs(lp - plain.candidate.average_logprob) <= 2 * LOGIT_TOL
    # an engine whose logits are given, position by position
    eng.reset_prefix_cache()
    table = (4 * torch.randn(42, config.vocab_size, generator=torch.Generator().manual_seed(1))
             ).to("cuda", torch.bfloat16)
    _give_logits(rt, table)
    eng = CandidateGroupEngine(rt, use_graphs)
    plain = eng.complete_drafted(prefix, lambda context, room: None, cfg)
    tokens = list(plain.candidate.token_ids)
    assert tokens == table[32:41].argmax(-1).tolist()
    # the same tokens drafted, with others beside them: fewer passes
    wrong = _ids(config, 8, 77)

    def drafter(context, room):
        at = len(context) - len(prefix)
        assert room == 9 - at
        return draft_tree([wrong[:3], tokens[at : at + 4] + wrong[:2], tokens[at : at + 1] + wrong])

    r = eng.complete_drafted(prefix, drafter, cfg)
    assert list(r.candidate.token_ids) == tokens and r.reused_prefix_tokens == len(prefix)
    assert r.passes == 2 and r.accepted == 6 and r.drafted > 6  # 1 + (4 + 1) + (2 + 1)
    assert abs(r.candidate.average_logprob - plain.candidate.average_logprob) < 1e-5
    assert rt.cache_manager.available_size == rt.num_pages - len(prefix)
    r = eng.complete_drafted(prefix, PhraseDrafter([prefix[-3:] + tokens, wrong]), cfg)
    assert list(r.candidate.token_ids) == tokens and r.passes == 1
    # an end of sequence inside the accepted drafts
    cut = next(i for i in range(1, 9) if tokens[i] not in tokens[:i])
    r = eng.complete_drafted(prefix, drafter, replace(cfg, eos_token_id=tokens[cut]))
    assert list(r.candidate.token_ids) == tokens[:cut] and r.candidate.stop_reason == "eos"
    assert r.passes == (0 if cut == 0 else 1 if cut <= 5 else 2)  # (none behind the end)
    assert rt.cache_manager.available_size == rt.num_pages - len(prefix)


@BITS
@pytest.mark.parametrize("use_graphs", [True, False])
def test_sampled_tokens_do_not_depend_on_the_drafts(kv_bits, use_graphs):
    """Drafts without logits: the candidate's own draws, whatever is drafted (on given
    logits: a draw depends on the order of the probabilities, and random weights leave
    neighbours closer than a bf16 step)."""
    eng, _ = _engine(IME, kv_bits, use_graphs=use_graphs)
    rt = eng.rt
    prefix = _ids(IME, 20, 4)
    cfg = CandidateGroupConfig(max_new_tokens=8, min_new_tokens=3, blocked_token_ids=(5, 9),
                               sampling=SamplingParams(temperature=0.7, top_k=50, top_p=0.9))
    table = 4 * torch.randn(28, IME.vocab_size, generator=torch.Generator().manual_seed(0))
    table[:, [5, 9]] = 30.0  # what the ban keeps out, and would be drawn without it
    table = table.to("cuda", torch.bfloat16)
    _give_logits(rt, table)
    uni = stateless_uniforms([cfg.seed], 8, "cuda")
    ban = torch.tensor(cfg.blocked_ids(), dtype=torch.int32, device="cuda")
    want, lps = [], []
    for t in range(8):
        pick, lp = sample_step(table[19 + t :][:1], cfg.sampling, uni,
                               torch.tensor(t, device="cuda"), ban, 3)
        want.append(int(pick))
        lps.append(float(lp))
    assert not {5, 9} & set(want[:3]) and {5, 9} & set(want[3:])
    for width in (0, 1, 2, 8):
        r = eng.complete_drafted(prefix, lambda context, room: draft_tree(
            [want[len(context) - 20 :][:width], _ids(IME, 3, len(context))]), cfg)
        assert list(r.candidate.token_ids) == want
        assert abs(r.candidate.average_logprob - sum(lps) / 8) < 1e-5
        assert r.passes == {0: 7, 1: 4, 2: 3, 8: 1}[width]
    assert rt.cache_manager.available_size == rt.num_pages - 20


@BITS
def test_drawn_drafts(kv_bits):
    """A drafter with a distribution of its own: the log-probs are the model's, all
    pages come back, and a draft drawn from the model's own logits is accepted."""
    eng, w = _engine(QWEN3, kv_bits)
    rt = eng.rt
    prefix = _ids(QWEN3, 18, 6)
    cfg = CandidateGroupConfig(max_new_tokens=7, sampling=SamplingParams(temperature=0.9))
    g = torch.Generator(device="cuda").manual_seed(0)

    def drafter(context, room):
        rows = torch.randn(5, 8192, generator=g, device="cuda").to(torch.bfloat16)
        t = torch.multinomial(torch.softmax(rows[:3].float() / 0.9, -1), 2, replacement=True,
                              generator=g)
        # two behind the context, two behind the first of them
        return DraftTree([int(t[0, 0]), int(t[0, 1]), int(t[1, 0]), int(t[1, 1])], [-1, -1, 0, 0],
                         rows)

    r = eng.complete_drafted(prefix, drafter, cfg)
    assert len(r.candidate.token_ids) == 7 and rt.cache_manager.available_size == rt.num_pages - 18
    ids = list(r.candidate.token_ids)
    ref = OracleModel(QWEN3, w).logits(torch.tensor(prefix + ids[:-1])[None], 0)[0, 17:]
    lp = ref.log_softmax(-1).gather(1, torch.tensor(ids)[:, None]).mean().item()
    if kv_bits == 16:
        assert abs(lp - r.candidate.average_logprob) <= 2 * LOGIT_TOL
    with pytest.raises(ValueError, match="without top_k"):
        eng.complete_drafted(prefix, drafter, replace(cfg, sampling=SamplingParams(0.9, top_k=5)))
    assert rt.cache_manager.available_size == rt.num_pages - 18


def test_a_drafter_that_fails_leaves_no_pages_behind():
    eng, _ = _engine(IME, 16)
    prefix = _ids(IME, 12, 8)

    def drafter(context, room):
        if len(context) > 14:
            raise RuntimeError("drafter")
        return None

    with pytest.raises(RuntimeError, match="drafter"):
        eng.complete_drafted(prefix, drafter)
    assert eng.rt.cache_manager.available_size == eng.rt.num_pages - 12
    token = eng.new_generation()

    def cancels(context, room):
        token.cancel()
        return None

    r = eng.complete_drafted(prefix, cancels, cancellation=token)
    assert r.cancelled and len(r.candidate.token_ids) == 2
    assert r.candidate.stop_reason == "cancelled"
    assert eng.rt.cache_manager.available_size == eng.rt.num_pages - 12


@BITS
def test_groups_before_and_behind_a_drafted_completion(kv_bits):
    """The same captured steps give the same candidates; their pages and table rows
    are as they were."""
    eng, _ = _engine(IME, kv_bits)
    prefix = _ids(IME, 24, 12)
    cfg = CandidateGroupConfig(max_new_tokens=6)
    before = eng.complete(prefix, cfg)
    scores = eng.score(prefix, [[1, 2, 3], [4]])
    r = eng.complete_drafted(prefix, PhraseDrafter([prefix[-2:] + [7, 8, 9], [3, 4]]), cfg)
    assert len(r.candidate.token_ids) == 6 and r.reused_prefix_tokens == 24
    behind = eng.complete(prefix, cfg)
    assert [c.token_ids for c in behind.raw_candidates] == [c.token_ids for c in
                                                            before.raw_candidates]
    assert [s.logprobs for s in eng.score(prefix, [[1, 2, 3], [4]])] == [s.logprobs for s in scores]
    assert eng.rt.cache_manager.available_size == eng.rt.num_pages - 24


@CONFIGS
@BITS
def test_a_captured_pass_gives_every_path_s_logits(config, kv_bits):
    """One graph, replayed with trees and lengths of its size and of smaller ones, other
    work between: every node's logits, and no page written but those handed over."""
    eng, w = _engine(config, kv_bits)
    rt = eng.rt
    ids = _ids(config, 90, 31)
    for shift, n in ((0, 8), (37, 8), (5, 6), (0, 5), (37, 7)):
        cached = 40 + shift
        eng.reset_prefix_cache()
        eng.score(ids[:cached], [[1, 2]])  # (fills page-table row 0)
        prefix_pages = eng._prefix_pages
        g = torch.Generator().manual_seed(shift + n)
        parents = [-1] + [int(torch.randint(i, (1,), generator=g)) for i in range(1, n)]
        tokens = _ids(config, n, 50 + n)
        paths = []
        for i in range(n):
            path = [i]
            while parents[path[0]] >= 0:
                path.insert(0, parents[path[0]])
            paths.append(path)
        graph = eng._draft_graph(cached, n)
        assert graph is eng._draft_graph(cached + 1, 8) and graph.nodes == 8
        pages = rt.cache_manager.allocate(8)
        rt.page_table[0, cached : cached + n] = pages[:n]
        pool = rt.kv_cache.k_cache(0) if kv_bits == 16 else rt.kv_cache.layer(0)[0].view(torch.uint8)
        before = pool.clone()
        with torch.inference_mode():
            logits, fed = graph.run(tokens, [cached + len(p) - 1 for p in paths], parents,
                                    cached + n, pages)
        assert fed.tolist() == tokens
        logits = logits.float().cpu()
        other = torch.ones(before.shape[0], dtype=torch.bool, device="cuda")
        other[pages.long()] = False
        assert torch.equal(before[other], pool[other])
        for row, path in enumerate(paths):
            at = torch.cat((prefix_pages, pages[torch.tensor(path, device="cuda")])).long().cpu()
            want = _oracle(config, w, rt, ids[:cached] + [tokens[i] for i in path], at)
            assert (logits[row] - want).abs().max() <= LOGIT_TOL
        rt.cache_manager._free(pages)
    assert len(eng._draft_graphs) == 1


def test_passes_that_no_graph_holds():
    """More nodes than a graph takes, more pages than are left, and a kept number of
    graphs."""
    eng, w = _engine(IME, 16, num_pages=200)
    rt = eng.rt
    assert eng._draft_graph(30, 65) is None and eng._draft_graph(30, 64).nodes == 64
    prefix = _ids(IME, 30, 2)
    cfg = CandidateGroupConfig(max_new_tokens=12)
    tokens = list(eng.complete_drafted(prefix, lambda context, room: None, cfg)
                  .candidate.token_ids)
    wide = [[tokens[0] + 1 + i] for i in range(100)]
    r = eng.complete_drafted(prefix, lambda context, room: draft_tree(
        wide + [tokens[len(context) - 30 :]], 120), cfg)
    assert r.drafted > 100
    _greedy_up_to_rounding(IME, w, prefix, list(r.candidate.token_ids))
    # 12 nodes: a graph would take 16 pages
    graphs = list(eng._draft_graphs)
    held = rt.cache_manager.allocate(rt.cache_manager.available_size - 15)
    r = eng.complete_drafted(prefix, lambda context, room: draft_tree(
        [tokens[len(context) - 30 :]]), cfg)
    assert len(r.candidate.token_ids) == 12 and graphs[0] == list(eng._draft_graphs)[0]
    _greedy_up_to_rounding(IME, w, prefix, list(r.candidate.token_ids))
    rt.cache_manager._free(held)
    assert rt.cache_manager.available_size == rt.num_pages - 30
    for n in (1, 2, 4, 8, 16, 32, 64):
        for cached in (10, 300, 600):
            eng._draft_graph(cached, n)
    assert len(eng._draft_graphs) == eng.MAX_GRAPHS

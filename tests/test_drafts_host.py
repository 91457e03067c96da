"""Drafts without a GPU: trees, the phrase drafter, and what the engine and the
backend refuse or leave out."""
from __future__ import annotations

import threading
from types import SimpleNamespace

import pytest
import torch

from aios_amd.attention.backend import Mi355xAttentionBackend
from aios_amd.core import Batch, Req, SamplingParams, reset_global_ctx, set_global_ctx
from aios_amd.drafts import DraftTree, PhraseDrafter, draft_tree
from aios_amd.ime import CandidateGroupConfig, CandidateGroupEngine
from aios_amd.scheduler import CacheManager


def test_continuations_share_their_beginnings():
    t = draft_tree([[1, 2, 3], [1, 2, 4], [5], [1, 2, 3, 6], []])
    assert list(t.tokens) == [1, 2, 3, 4, 5, 6]
    assert list(t.parents) == [-1, 0, 1, 1, -1, 2]
    assert t.depths() == [1, 2, 3, 3, 1, 4]
    assert list(draft_tree([[1, 2, 3], [4]], 2).tokens) == [1, 2]
    assert list(draft_tree([], 5).tokens) == []


@pytest.mark.parametrize("tokens,parents,match", [
    ([1, 2], [-1], "needs a parent"), ([1], [0], "earlier draft"), ([1], [-2], "earlier draft"),
    ([10], [-1], "vocabulary"), ([-1], [-1], "vocabulary"), ([1] * 256, [-1] * 256, "255 drafts"),
])
def test_trees_are_checked(tokens, parents, match):
    with pytest.raises(ValueError, match=match):
        DraftTree(tokens, parents).validate(10)
    with pytest.raises(ValueError, match="draft logits"):
        DraftTree([1], [-1], torch.zeros(1, 10)).validate(10)
    DraftTree([1], [-1], torch.zeros(2, 10)).validate(10)


def test_phrases_go_on_where_the_context_ends():
    d = PhraseDrafter([[1, 2, 3, 4], [9, 2, 3, 5, 6], [2, 7]])
    t = d([8, 1, 2, 3], 3)  # three tokens of the first phrase match, two of the second
    assert list(t.tokens) == [4, 5, 6] and list(t.parents) == [-1, -1, 1]
    t = d([0, 2], 2)  # one token: every phrase, in their order
    assert list(t.tokens) == [3, 4, 5, 7] and list(t.parents) == [-1, 0, 0, -1]
    assert list(d([4], 5).tokens) == [] and list(d([], 5).tokens) == []
    assert list(PhraseDrafter([[1, 2, 3, 4], [2, 7]], min_match=2)([1, 2], 5).tokens) == [3, 4]
    assert list(PhraseDrafter([[1, 2, 3, 4]], max_drafts=1)([1], 5).tokens) == [2]
    for kw in ({"min_match": 0}, {"min_match": 3, "max_match": 2}, {"max_drafts": 256}):
        with pytest.raises(ValueError):
            PhraseDrafter([], **kw)


def _engine(pages=64, columns=40):
    cache = CacheManager(torch.device("cpu"), pages)
    rt = SimpleNamespace(cache_manager=cache, page_table=torch.zeros(2, columns, dtype=torch.int32),
                         model=SimpleNamespace(w={"embed": torch.zeros(100, 4)}), num_pages=pages,
                         config=SimpleNamespace(max_position_embeddings=columns),
                         max_context=columns, device=torch.device("cpu"))
    e = CandidateGroupEngine.__new__(CandidateGroupEngine)
    e.rt, e._gen_lock, e._run_lock = rt, threading.Lock(), threading.Lock()
    e._active, e._generation_id = None, 0
    return e


def test_drafts_that_cannot_be_checked_are_left_out():
    e = _engine()
    cfg = CandidateGroupConfig()
    tree = DraftTree([1, 2, 3, 4, 5], [-1, 0, 1, -1, 3])
    assert e._trim(tree, 10, 20, cfg) is tree
    assert e._trim(None, 10, 20, cfg).tokens == ()
    t = e._trim(tree, 3, 20, cfg)  # room for two drafts and the added token
    assert list(t.tokens) == [1, 2, 4, 5] and list(t.parents) == [-1, 0, -1, 2]
    assert list(e._trim(tree, 1, 20, cfg).tokens) == []
    t = e._trim(tree, 10, 38, cfg)  # the table's row ends
    assert list(t.tokens) == [1, 2]
    t = _engine(pages=4)._trim(tree, 10, 20, cfg)  # the free pages end
    assert list(t.tokens) == [1, 2, 3] and list(t.parents) == [-1, 0, 1]
    rows = torch.arange(6.0)[:, None].expand(6, 100)
    t = e._trim(DraftTree(tree.tokens, tree.parents, rows), 3, 20,
                CandidateGroupConfig(sampling=SamplingParams(temperature=1.0)))
    assert t.logits[:, 0].tolist() == [0, 1, 2, 4, 5]


@pytest.mark.parametrize("kw", [{"top_k": 5}, {"top_p": 0.9}])
def test_drawn_drafts_need_plain_sampling(kw):
    e = _engine()
    tree = DraftTree([1], [-1], torch.zeros(2, 100))
    with pytest.raises(ValueError, match="without top_k"):
        e._trim(tree, 5, 20, CandidateGroupConfig(sampling=SamplingParams(temperature=1.0, **kw)))
    with pytest.raises(ValueError, match="without top_k"):
        e._trim(tree, 5, 20, CandidateGroupConfig(sampling=SamplingParams(temperature=1.0),
                                                  min_new_tokens=2))
    e._trim(tree, 5, 20, CandidateGroupConfig(sampling=SamplingParams(temperature=1.0)))
    e._trim(tree, 5, 20, CandidateGroupConfig())


def test_engine_refusals():
    e = _engine()
    draft = lambda context, room: None
    with pytest.raises(ValueError, match="no input tokens"):
        e.complete_drafted([], draft)
    with pytest.raises(ValueError, match="vocabulary"):
        e.complete_drafted([100], draft)
    with pytest.raises(ValueError, match="context limit"):
        e.complete_drafted([1] * 30, draft, CandidateGroupConfig(max_new_tokens=11))
    with pytest.raises(ValueError, match="KV budget"):
        _engine(pages=20).complete_drafted([1] * 10, draft, CandidateGroupConfig(max_new_tokens=11))
    with pytest.raises(ValueError, match="max_new_tokens"):
        e.complete_drafted([1], draft, CandidateGroupConfig(max_new_tokens=0))
    token = e.new_generation()
    e.new_generation()
    r = e.complete_drafted([1], draft, cancellation=token)
    assert r.cancelled and r.candidate.token_ids == () and r.passes == 0


def test_backend_refuses_parents_that_are_no_tree():
    be = Mi355xAttentionBackend(SimpleNamespace(num_qo_heads=4, num_kv_heads=2, head_dim=64))
    cu = torch.tensor([0, 3], dtype=torch.int32)
    for parents, match in (([[-1, 0]], "every new token"), ([[-1, 0, 0], [-1]], "every new token"),
                           ([[-1, 1, 0]], "earlier one"), ([[-1, 0, -2]], "earlier one")):
        with pytest.raises(ValueError, match=match):
            be._plan_trees(parents, [3], cu, cu, cu, 16)


def test_backend_refuses_a_decode_batch_of_trees():
    be = Mi355xAttentionBackend(SimpleNamespace(num_qo_heads=4, num_kv_heads=2, head_dim=64))
    ctx = SimpleNamespace(page_table=torch.zeros(1, 8, dtype=torch.int32), kv_cache=None)
    b = Batch(reqs=[Req(input_ids=torch.empty(4, dtype=torch.long), cached_len=3, output_len=1,
                        uid=0, sampling_params=SamplingParams(), table_idx=0)], phase="decode")
    b.tree_parents = [[-1]]
    set_global_ctx(ctx)
    try:
        with pytest.raises(ValueError, match="prefill batch"):
            be.prepare_metadata(b)
    finally:
        reset_global_ctx()

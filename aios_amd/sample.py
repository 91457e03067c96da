"""Stateless candidate sampling on the gfx950 kernels (the interface of
python/aios/engine/sample.py: ``stateless_uniforms`` and
``Sampler.sample_with_logprobs``).

``stateless_uniforms`` computes the SplitMix64 uniforms on the device
(``aios_stateless_uniforms``), keyed by (candidate seed, token step), so a
candidate keeps its stream wherever its row sits in the batch.
``Sampler.sample_with_logprobs`` is one call of ``aios_sample_ws``:
temperature / top-k / top-p on a sampling copy with forbidden ids at -inf,
the token chosen by the candidate's uniform, and the raw log-probability of
the unmodified distribution.  ``sample_step`` is the same launch with the
step index read on the device, for graph-replayed decode loops.
``verify_drafts`` is the acceptance rule of speculative decoding.

Ties in the top-k order go to the lower token id.  Without ``uniforms`` the
uniforms are drawn with ``torch.rand`` (the reference uses
``torch.multinomial`` there; that stream is not reproduced).
"""
from __future__ import annotations

from collections.abc import Sequence
from dataclasses import dataclass
from typing import NamedTuple

import torch

from aios_amd import _lib
from aios_amd.core import SamplingParams

_NO_STEP_LIMIT = 2**31 - 1


def _stream(t: torch.Tensor) -> int:
    return _lib.raw_stream(t)


def stateless_uniforms(candidate_seeds: Sequence[int] | torch.Tensor, steps: int,
                       device: torch.device) -> torch.Tensor:
    """``(rows, steps)`` float32 uniforms, one independent stream per seed."""
    if steps < 1:
        raise ValueError("steps must be positive")
    device = torch.device(device)
    if device.type != "cuda":
        raise ValueError("stateless_uniforms runs on the GPU")
    seeds = torch.as_tensor(candidate_seeds, dtype=torch.int64)
    if seeds.device != device:
        seeds = seeds.to(device)
    seeds = seeds.contiguous()
    out = torch.empty((seeds.numel(), steps), dtype=torch.float32, device=device)
    _lib.check(_lib.lib().aios_stateless_uniforms(seeds.data_ptr(), seeds.numel(), steps,
                                                  out.data_ptr(), _stream(out)),
               "aios_stateless_uniforms")
    return out


def _check_logits(logits: torch.Tensor) -> None:
    if logits.ndim != 2 or logits.stride(1) != 1 or not logits.is_cuda:
        raise ValueError("logits must be a 2-D GPU tensor with contiguous rows")
    if logits.dtype not in (torch.bfloat16, torch.float32):
        raise ValueError("logits must be bfloat16 or float32")


def sample_step(logits: torch.Tensor, params: SamplingParams, uniforms: torch.Tensor,
                step: torch.Tensor, forbidden_ids: torch.Tensor | None = None,
                forbid_before_step: int = _NO_STEP_LIMIT,
                forbidden_by_row: torch.Tensor | None = None,
                out: tuple[torch.Tensor, torch.Tensor] | None = None):
    """Graph-safe launch: row r uses ``uniforms[r, step]`` with ``step`` a
    device int64 scalar; ``forbidden_ids`` (device int32) apply while
    ``step < forbid_before_step``.  Returns (tokens int64 [rows], raw
    log-probs fp32 [rows])."""
    _check_logits(logits)
    rows, vocab = logits.shape
    if uniforms.dtype != torch.float32 or uniforms.ndim != 2 or uniforms.shape[0] != rows \
            or uniforms.stride(1) != 1:
        raise ValueError("uniforms must be float32 [rows, steps] with contiguous rows")
    if step.dtype != torch.int64 or step.numel() != 1:
        raise ValueError("step must be a one-element int64 tensor")
    if forbidden_by_row is not None and (
            forbidden_by_row.dtype != torch.int64 or forbidden_by_row.ndim != 2
            or forbidden_by_row.shape[0] != rows or not forbidden_by_row.is_contiguous()):
        raise ValueError("forbidden_by_row must be contiguous int64 [rows, n]")
    tok, lp = out if out is not None else (
        torch.empty(rows, dtype=torch.int64, device=logits.device),
        torch.empty(rows, dtype=torch.float32, device=logits.device))
    nf = 0 if forbidden_ids is None else forbidden_ids.numel()
    nr = 0 if forbidden_by_row is None else forbidden_by_row.shape[1]
    lib = _lib.lib()
    # (the candidates of long rows: a buffer of this call alone, since calls may
    # overlap on several streams)
    ws_bytes = lib.aios_sample_workspace(rows, vocab, float(params.temperature),
                                         int(params.top_k), float(params.top_p))
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=logits.device) if ws_bytes else None
    _lib.check(lib.aios_sample_ws(
        logits.data_ptr(), logits.stride(0), rows, vocab, logits.element_size(),
        float(params.temperature), int(params.top_k), float(params.top_p),
        uniforms.data_ptr(), uniforms.stride(0), uniforms.shape[1], step.data_ptr(),
        forbidden_ids.data_ptr() if nf else None, nf, int(forbid_before_step),
        forbidden_by_row.data_ptr() if nr else None, nr, tok.data_ptr(), lp.data_ptr(),
        ws.data_ptr() if ws is not None else None, ws_bytes, _stream(logits)), "aios_sample_ws")
    return tok, lp


@dataclass
class Sampler:
    """engine/sample.py:50-160 on the sampling kernel."""

    sampling_params: SamplingParams

    def sample_with_logprobs(
        self,
        logits: torch.Tensor,
        *,
        generator: torch.Generator | None = None,
        uniforms: torch.Tensor | None = None,
        forbidden_token_ids: Sequence[int] = (),
        forbidden_token_ids_by_row: torch.Tensor | None = None,
    ) -> tuple[torch.Tensor, torch.Tensor]:
        """(token ids [rows, 1], raw log-probs [rows, 1]) of 2-D logits."""
        if generator is not None and uniforms is not None:
            raise ValueError("generator and uniforms are mutually exclusive")
        _check_logits(logits)
        rows, vocab = logits.shape
        blocked = sorted({int(t) for t in forbidden_token_ids})
        invalid = [t for t in blocked if t < 0 or t >= vocab]
        if invalid:
            raise ValueError(f"forbidden token ids are outside the vocabulary: {invalid}")
        by_row = None
        if forbidden_token_ids_by_row is not None:
            f = forbidden_token_ids_by_row
            if f.ndim != 2 or f.shape[0] != rows:
                raise ValueError("forbidden_token_ids_by_row must have shape [batch, count]")
            if f.device.type == "cpu" and not bool(((f >= 0) & (f < vocab)).all().item()):
                raise ValueError("row-specific forbidden token ids are outside the vocabulary")
            by_row = f.to(device=logits.device, dtype=torch.int64).contiguous()
            if by_row.shape[1] == 0:
                by_row = None
        p = self.sampling_params
        if p.is_greedy:
            u = torch.full((rows, 1), 0.5, dtype=torch.float32, device=logits.device)
        elif uniforms is None:
            u = torch.rand((rows, 1), generator=generator, device=logits.device)
        else:
            if tuple(uniforms.shape) != (rows,):
                raise ValueError("uniforms must match the sampling batch dimensions: "
                                 f"expected {(rows,)}, got {tuple(uniforms.shape)}")
            u = uniforms.to(device=logits.device, dtype=torch.float32).reshape(rows, 1).contiguous()
        ids = (torch.tensor(blocked, dtype=torch.int32, device=logits.device) if blocked else None)
        step = torch.zeros(1, dtype=torch.int64, device=logits.device)
        tok, lp = sample_step(logits, p, u, step, ids, _NO_STEP_LIMIT, by_row)
        return tok[:, None], lp[:, None]

    def sample(self, logits: torch.Tensor) -> torch.Tensor:
        return self.sample_with_logprobs(logits)[0]


class TokenLogprobs(NamedTuple):
    """:func:`token_logprobs`'s answers for a batch of rows."""

    logprobs: torch.Tensor      # float32 [rows]: ln p of the given tokens
    entropies: torch.Tensor     # float32 [rows], in nats
    top_ids: torch.Tensor       # int64 [rows, top], most likely first
    top_logprobs: torch.Tensor  # float32 [rows, top]


MAX_TOP_LOGPROBS = 32


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, top: int = 0) -> TokenLogprobs:
    """Log probabilities of given tokens (int64 [rows]) under the rows of
    ``logits`` (bfloat16 or float32 [rows, vocab]), each row's entropy and its
    ``top`` most likely ids with their log probabilities (at most 32; equal
    logits by ascending id), in one pass over the logits
    (``aios_token_logprobs``).  A token outside the vocabulary has log
    probability NaN, ids at -inf count as impossible, and a row without a
    finite maximum gives NaN."""
    _check_logits(logits)
    rows, vocab = logits.shape
    if tokens.dtype != torch.int64 or tokens.shape != (rows,) or \
            tokens.get_device() != logits.get_device():
        raise ValueError("tokens must be int64 [rows] on the logits' GPU")
    if not 0 <= top <= min(vocab, MAX_TOP_LOGPROBS):
        raise ValueError(f"top must be within 0..{min(vocab, MAX_TOP_LOGPROBS)}")
    if not tokens.is_contiguous():
        tokens = tokens.contiguous()
    lib, dev = _lib.lib(), logits.device
    # (one allocation for the three: allocations are a good part of a short
    # call's time on the host)
    lp, ent, alt = torch.empty(rows * (2 + top), dtype=torch.float32, device=dev).split_with_sizes(
        (rows, rows, rows * top))
    alt = alt.view(rows, top)
    ids = tokens.new_empty((rows, top))
    # (the states of split rows: a buffer of this call alone, since calls may
    # overlap on several streams)
    ws_bytes = lib.aios_token_logprobs_workspace(rows, vocab, top)
    ws = ids.new_empty((ws_bytes + 7) // 8) if ws_bytes else None
    _lib.check(lib.aios_token_logprobs(
        logits.data_ptr(), logits.stride(0), rows, vocab, logits.element_size(),
        tokens.data_ptr(), top, lp.data_ptr(), ent.data_ptr(), ids.data_ptr(), alt.data_ptr(),
        None if ws is None else ws.data_ptr(), ws_bytes, _lib.current_stream(logits)),
        "aios_token_logprobs")
    return TokenLogprobs(lp, ent, ids, alt)


class VerifiedDrafts(NamedTuple):
    """:func:`verify_drafts`'s answers for a batch of requests with nodes."""

    accepted: torch.Tensor     # bool [nodes]: node 0 of a request and the accepted ones behind it
    counts: torch.Tensor       # int32 [requests]: accepted drafts
    last: torch.Tensor         # int32 [requests]: the last accepted node, counted in the request
    next_tokens: torch.Tensor  # int64 [requests]: the token added behind it
    logprobs: torch.Tensor     # float32 [nodes]: ln p of a node's token; node 0: of the added one


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, parents: torch.Tensor,
                  cu: torch.Tensor, uniforms: torch.Tensor | None = None, *,
                  draft_logits: torch.Tensor | None = None, temperature: float = 1.0,
                  draft_temperature: float | None = None) -> VerifiedDrafts:
    """Which drafted tokens the target accepts, and the token it adds, from
    given random numbers (``aios_verify_drafts``): the tokens that come out are
    distributed as the target's own at ``temperature``.

    Request r's nodes are ``cu[r] .. cu[r + 1]`` (int32 [requests + 1], at most
    256 each): node 0 is decided, node i drafts ``tokens[i]`` (int64 [nodes])
    behind node ``parents[i]`` (int32 [nodes], counted within the request; -1:
    a node that is never accepted).  ``logits`` row i (bfloat16 or float32
    [nodes, vocab]) is the target's behind node i.  ``draft_logits`` row i, of
    the same shape and type, is what the children of node i were drawn from at
    ``draft_temperature`` (default: ``temperature``), one after another in their
    order; without it the drafts count as certain (phrases of a list).
    ``uniforms`` (float32 [nodes], in [0, 1)) decides on each draft, node 0's on
    the added token.

    Children are tried in ascending order, with p = softmax(logits /
    temperature) and q the draft's: x is accepted if u q(x) < p(x), else p
    becomes max(p - q, 0), normalised (certain drafts: p without x).  The added
    token is drawn, in the order of the ids, from what p has become behind the
    last accepted node.  ``temperature`` 0 accepts and adds the most likely
    tokens (the lowest id of equal ones) and reads no uniforms and no draft
    logits.  Log-probs are those of the unscaled logits, as the sampler's."""
    _check_logits(logits)
    n, vocab = logits.shape
    dev = logits.get_device()
    greedy = temperature == 0
    if greedy:
        draft_logits = None
    for t, name, dtype in ((tokens, "tokens", torch.int64), (parents, "parents", torch.int32)):
        if t.dtype is not dtype or t.shape != (n,) or t.get_device() != dev or \
                not t.is_contiguous():
            raise ValueError(f"{name} must be a contiguous {str(dtype)[6:]} [nodes] tensor on the "
                             "logits' GPU")
    if cu.dtype is not torch.int32 or cu.ndim != 1 or cu.numel() < 1 or cu.get_device() != dev or \
            not cu.is_contiguous():
        raise ValueError("cu must be a contiguous int32 [requests + 1] tensor on the logits' GPU")
    if not greedy and (uniforms is None or uniforms.dtype is not torch.float32
                       or uniforms.shape != (n,) or uniforms.get_device() != dev
                       or not uniforms.is_contiguous()):
        raise ValueError("uniforms must be a contiguous float32 [nodes] tensor on the logits' GPU")
    if draft_logits is not None:
        _check_logits(draft_logits)
        if draft_logits.shape != logits.shape or draft_logits.dtype is not logits.dtype or \
                draft_logits.get_device() != dev:
            raise ValueError("draft_logits must be of the logits' shape and type, on their GPU")
    if draft_temperature is None:
        draft_temperature = temperature
    b = cu.numel() - 1
    lib, device = _lib.lib(), logits.device
    accepted = torch.empty(n, dtype=torch.bool, device=device)
    counts, last = torch.empty(2 * b, dtype=torch.int32, device=device).split_with_sizes((b, b))
    nxt = tokens.new_empty(b)
    lp = torch.empty(n, dtype=torch.float32, device=device)
    # (a buffer of this call alone, since calls may overlap on several streams)
    ws_bytes = lib.aios_verify_workspace(b, n, vocab, draft_logits is not None)
    ws = torch.empty(ws_bytes, dtype=torch.uint8, device=device)
    stride = logits.stride(0) if n > 1 else vocab  # (a single row's is not looked at)
    draft, draft_stride = None, 0
    if draft_logits is not None:
        draft = draft_logits.data_ptr()
        draft_stride = draft_logits.stride(0) if n > 1 else vocab
    _lib.check(lib.aios_verify_drafts(
        logits.data_ptr(), stride, draft, draft_stride, vocab, logits.element_size(),
        tokens.data_ptr(), parents.data_ptr(), cu.data_ptr(), b, n,
        None if greedy else uniforms.data_ptr(), temperature, draft_temperature,
        accepted.data_ptr(), counts.data_ptr(), last.data_ptr(), nxt.data_ptr(), lp.data_ptr(),
        ws.data_ptr(), ws_bytes, _lib.current_stream(logits)), "aios_verify_drafts")
    return VerifiedDrafts(accepted, counts, last, nxt, lp)

"""Drafted tokens: what a drafter proposes behind a context, as a tree, and a
drafter of known phrases.

``CandidateGroupEngine.complete_drafted`` calls a drafter ``drafter(context,
room)`` with the tokens so far and the number that may still be added, and
checks every proposed continuation in one forward pass.
"""
from __future__ import annotations

from collections.abc import Iterable, Sequence
from dataclasses import dataclass

import torch

from aios_amd import _lib

# Drafts of one request in one pass (the decided token is a node too).
MAX_DRAFTS = _lib.TREE_MAX_NODES - 1


@dataclass(frozen=True)
class DraftTree:
    """Drafts behind a context.  Draft i is ``tokens[i]`` behind draft
    ``parents[i]`` < i, or behind the context itself (-1).  ``logits`` (GPU
    [1 + drafts, vocab], of the target's type): row 0 what the drafts behind
    the context were drawn from, row 1 + i those behind draft i, one after
    another, at the sampling temperature; None: no distribution drew them."""

    tokens: Sequence[int]
    parents: Sequence[int]
    logits: torch.Tensor | None = None

    def validate(self, vocab: int) -> None:
        if len(self.tokens) != len(self.parents):
            raise ValueError("every draft needs a parent")
        if len(self.tokens) > MAX_DRAFTS:
            raise ValueError(f"at most {MAX_DRAFTS} drafts are checked at once")
        if any(not -1 <= p < i for i, p in enumerate(self.parents)):
            raise ValueError("a draft's parent is an earlier draft, or -1")
        if any(not 0 <= t < vocab for t in self.tokens):
            raise ValueError("drafted token outside the vocabulary")
        if self.logits is not None and self.logits.shape != (1 + len(self.tokens), vocab):
            raise ValueError("draft logits must be [1 + drafts, vocab]")

    def depths(self) -> list[int]:
        """Tokens from the context to each draft, itself included."""
        out: list[int] = []
        for p in self.parents:
            out.append(1 + (out[p] if p >= 0 else 0))
        return out


def draft_tree(continuations: Iterable[Sequence[int]], max_drafts: int = 63) -> DraftTree:
    """Continuations of one context as a tree: shared beginnings become one
    draft, earlier continuations first; at most ``max_drafts`` drafts."""
    tokens: list[int] = []
    parents: list[int] = []
    seen: dict[tuple[int, int], int] = {}
    for cont in continuations:
        at = -1
        for t in cont:
            child = seen.get((at, int(t)))
            if child is None:
                if len(tokens) >= max_drafts:
                    break
                child = seen[at, int(t)] = len(tokens)
                tokens.append(int(t))
                parents.append(at)
            at = child
    return DraftTree(tokens, parents)


class PhraseDrafter:
    """Drafts from phrases that were typed before: behind a context whose last
    tokens (at least ``min_match``) occur in a phrase, the phrase goes on.
    Longer matches come first, then phrases in the order given."""

    def __init__(self, phrases: Iterable[Sequence[int]], min_match: int = 1, max_match: int = 8,
                 max_drafts: int = 63) -> None:
        if not 1 <= min_match <= max_match:
            raise ValueError("min_match must be within 1..max_match")
        if not 0 <= max_drafts <= MAX_DRAFTS:
            raise ValueError(f"max_drafts must be within 0..{MAX_DRAFTS}")
        self.min_match, self.max_match, self.max_drafts = min_match, max_match, max_drafts
        self.phrases = [tuple(int(t) for t in p) for p in phrases]
        # (phrase, position behind it) of every token
        self._behind: dict[int, list[tuple[int, int]]] = {}
        for i, p in enumerate(self.phrases):
            for j, t in enumerate(p[:-1]):
                self._behind.setdefault(t, []).append((i, j + 1))

    def __call__(self, context: Sequence[int], room: int) -> DraftTree:
        found = []
        for i, j in self._behind.get(int(context[-1]), ()) if len(context) else ():
            p, k = self.phrases[i], 1
            while k < self.max_match and k < j and k < len(context) and \
                    p[j - 1 - k] == context[-1 - k]:
                k += 1
            if k >= self.min_match:
                found.append((-k, i, j))
        return draft_tree((self.phrases[i][j : j + room] for _, i, j in sorted(found)),
                          self.max_drafts)

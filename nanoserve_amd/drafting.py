"""Drafted tokens for a decode step, from the request's own text.

A drafter is anything with

    draft(seq, limit, depth) -> (tokens, parents)

for a sequence (scheduling.Sequence): at most `limit` drafted tokens that may follow
its last one, no chain of them longer than `depth`.  Token i is row i + 1 of the
sequence's tree, parents[i] is the row it follows (0: the last token), and parents come
before their children.  A drafter decides only how fast a request goes: a step
keeps the drafted tokens that the model itself chooses (tree.commit_drafts).

The reference decodes without drafts (nanoserve/engine.py:140-190).
"""

from __future__ import annotations


def check_draft(tokens: list[int], parents: list[int], limit: int, depth: int, vocab_size: int) -> None:
    """Raise unless (tokens, parents) is what a drafter may return."""
    if len(tokens) != len(parents):
        raise ValueError(f"a draft of {len(tokens)} tokens with {len(parents)} parents")
    if len(tokens) > max(limit, 0):
        raise ValueError(f"a draft of {len(tokens)} tokens, at most {limit} were asked for")
    at = [0]  # depth of every row
    for i, (t, p) in enumerate(zip(tokens, parents)):
        if not 0 <= t < vocab_size:
            raise ValueError(f"drafted token {t} is outside the vocabulary of {vocab_size}")
        if not 0 <= p <= i:
            raise ValueError(f"drafted token {i} names row {p} as its parent: an earlier one of its tree is needed")
        at.append(at[p] + 1)
    if max(at) > max(depth, 0):
        raise ValueError(f"a draft with a chain of {max(at)} tokens, at most {depth} were asked for")


class NgramDrafter:
    """What followed the same last tokens earlier in the prompt or the output.

    The longest n-gram (up to max_ngram) that ends the sequence and stands in it
    before gives the first chain, its latest places first; shorter ones and earlier
    places add branches, up to `branches` chains in all.  Chains that begin alike
    share their rows.  It keeps the text of the requests that it has seen, by their
    ids: an engine needs one of its own."""

    def __init__(self, max_ngram: int = 3, branches: int = 2) -> None:
        if max_ngram < 1 or branches < 1:
            raise ValueError(f"max_ngram and branches must be positive, got {max_ngram} and {branches}")
        self.max_ngram = max_ngram
        self.branches = branches
        # Per sequence: the tokens indexed so far, and for every n-gram the places behind it.
        self._known: dict[int, tuple[list[int], dict[tuple, list[int]]]] = {}

    def forget(self, seq) -> None:
        self._known.pop(seq.seq_id, None)

    def _index(self, seq) -> tuple[list[int], dict[tuple, list[int]]]:
        text, places = self._known.setdefault(seq.seq_id, ([], {}))
        done = len(text)
        text += seq.token_slice(done, seq.num_tokens)
        for end in range(done + 1, len(text) + 1):
            for n in range(1, min(self.max_ngram, end) + 1):
                places.setdefault(tuple(text[end - n:end]), []).append(end)
        return text, places

    def draft(self, seq, limit: int, depth: int) -> tuple[list[int], list[int]]:
        text, places = self._index(seq)
        tokens: list[int] = []
        parents: list[int] = []
        child: dict[tuple[int, int], int] = {}  # (row, token) -> the row that holds it
        if limit <= 0 or depth <= 0:
            return tokens, parents
        chains = 0
        seen: set[int] = set()
        for n in range(min(self.max_ngram, len(text)), 0, -1):
            for at in reversed(places[tuple(text[len(text) - n:])]):
                if at == len(text) or at in seen:
                    continue  # the end itself; a place that a longer n-gram gave
                seen.add(at)
                row = 0
                for t in text[at:at + depth]:
                    nxt = child.get((row, t))
                    if nxt is None:
                        if len(tokens) == limit:
                            return tokens, parents
                        tokens.append(t)
                        parents.append(row)
                        nxt = child[row, t] = len(tokens)
                    row = nxt
                chains += 1
                if chains == self.branches:
                    return tokens, parents
        return tokens, parents

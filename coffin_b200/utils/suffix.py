"""Host-side suffix-match drafter for speculative decoding.

Keeps the token history of one sequence and proposes the continuation that followed the most
recent earlier occurrence of the current suffix (longest suffix first, ``min_match`` ..
``max_match`` tokens).  Every draft is therefore a true continuation of something already seen;
repetitive outputs (code, lists, quoted context) accept long drafts at zero model cost.
Reference: ``ops/suffix.py`` (``SuffixDrafter(max_match=4, min_match=2).reset/observe/draft``).
"""
from __future__ import annotations


class SuffixDrafter:
    KEEP = 4                                             # earlier occurrences of an n-gram that a tree of drafts looks at

    def __init__(self, max_match: int = 4, min_match: int = 2) -> None:
        if not 1 <= min_match <= max_match:
            raise ValueError("need 1 <= min_match <= max_match")
        self.max_match, self.min_match = max_match, min_match
        self.reset()

    def reset(self) -> None:
        self.history: list[int] = []
        self._index: dict[tuple[int, ...], int] = {}     # n-gram -> end position of its latest earlier occurrence
        self._before: dict[int, int] = {}                # end position of an occurrence (by n-gram length) -> of the one before it

    def observe(self, tokens) -> None:
        for t in tokens:
            self.history.append(int(t))
            n = len(self.history)
            # index the n-grams that end just before the new token, so that a lookup never
            # returns the suffix's own occurrence
            for k in range(self.min_match, self.max_match + 1):
                if n - 1 >= k:
                    gram = tuple(self.history[n - 1 - k:n - 1])
                    if gram in self._index:
                        self._before[(n - 1) * self.max_match + k - 1] = self._index[gram]
                    self._index[gram] = n - 1

    def draft(self, k: int) -> list[int]:
        """Up to ``k`` proposed next tokens (possibly none; none for ``k <= 0``)."""
        if k <= 0:
            return []
        h = self.history
        for m in range(min(self.max_match, len(h)), self.min_match - 1, -1):
            end = self._index.get(tuple(h[-m:]))
            if end is not None and end < len(h):
                return h[end:end + k]
        return []

    def draft_tree(self, depth: int, nodes: int) -> tuple[list[int], list[int]]:
        """Up to ``nodes`` proposed tokens as a tree at most ``depth`` deep: ``(tokens, parents)`` with parent -1 for a first token and a
        parent before its children.  The continuation that ``draft`` proposes comes first; those of earlier occurrences, and of
        shorter suffixes, branch off where they differ from it."""
        tokens: list[int] = []
        parents: list[int] = []
        child: dict[tuple[int, int], int] = {}
        h = self.history
        for m in range(min(self.max_match, len(h)), self.min_match - 1, -1):
            end = self._index.get(tuple(h[-m:]))
            for _ in range(self.KEEP):
                if end is None or len(tokens) >= nodes:
                    break
                at = -1
                for t in h[end:end + max(0, depth)]:
                    nxt = child.get((at, t))
                    if nxt is None:
                        if len(tokens) >= nodes:
                            break
                        nxt = child[(at, t)] = len(tokens)
                        tokens.append(t)
                        parents.append(at)
                    at = nxt
                end = self._before.get(end * self.max_match + m - 1)
        return tokens, parents

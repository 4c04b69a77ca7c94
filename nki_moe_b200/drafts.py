"""Drafts of what a sequence may go on with, for steps that check several tokens at once.

A draft is a tree of token ids, given in an order in which every node comes
after its parent: ``(tokens, parents)``, ``parents[i]`` being the index of node
``i``'s parent or -1 for one that follows the sequence's last token.  Whoever
checks it (:meth:`nki_moe_b200.qwen_stack.Qwen3MoEStack.generate_paged`) keeps the
path that the model itself takes, so a wrong draft never gets into a text; a draft
changes how many steps it takes.  (To the arithmetic: a step with drafts rounds in
other places than one without, so among nearly equal logits the choice may differ.)

The reference decodes one token a step; nothing there corresponds to this module.
"""

from __future__ import annotations

__all__ = ["LookupDrafts"]


class LookupDrafts:
    """Drafts from the text itself: what followed the last time that it ended as it
    ends now, and the times before, the longest repetitions first."""

    def __init__(self, text=(), longest: int = 4):
        if longest < 1:
            raise ValueError("longest must be positive")
        self.longest = longest
        self.text: list[int] = []
        self._after: dict[tuple, list[int]] = {}  # where what follows these tokens begins
        self.extend(text)

    def extend(self, tokens) -> None:
        """Appends tokens to the text."""
        for t in tokens:
            self.text.append(int(t))
            n = len(self.text)
            for k in range(1, min(self.longest, n) + 1):
                self._after.setdefault(tuple(self.text[n - k:]), []).append(n)

    def tree(self, nodes: int, runs: int = 16) -> tuple[list[int], list[int]]:
        """A draft of at most ``nodes`` nodes: up to ``runs`` earlier continuations,
        as far as they agree sharing their nodes.  The first one may take all nodes
        but a quarter, which later ones that part from it take if there are any."""
        tokens, parents, children = [], [], {}
        n, seen = len(self.text), set()

        def add(start: int, most: int) -> None:
            at = -1
            for t in self.text[start:start + nodes]:
                child = children.get((at, t))
                if child is None:
                    if len(tokens) >= most:
                        return
                    child = children[at, t] = len(tokens)
                    tokens.append(t)
                    parents.append(at)
                at = child

        starts = []
        for k in range(min(self.longest, n), 0, -1):
            for start in reversed(self._after.get(tuple(self.text[n - k:]), [])):
                if start < n and start not in seen:
                    seen.add(start)
                    starts.append(start)
                    if len(starts) == runs:
                        break
            if len(starts) == runs:
                break
        for i, start in enumerate(starts):
            add(start, nodes - nodes // 4 if i == 0 and len(starts) > 1 else nodes)
        if starts:
            add(starts[0], nodes)  # what the others left
        return tokens, parents

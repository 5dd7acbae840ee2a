"""Drafted trees for BatchedEngine's drafted decoding.

A drafter proposes likely continuations of a token list as a tree of (token,
parent) pairs, parents first and -1 for a child of the list's last token.
``PromptLookup`` needs no second model: it continues the last tokens as the
text itself continued them where they stood before.
"""

from __future__ import annotations


def tree_of(drafted, limit, depth, vocab):
    """A drafter's (token, parent) pairs as the engine uses them: at most `limit`
    nodes, none deeper than `depth`, no tokens outside the vocabulary and no two
    children of a node with one token (the later one's own children move to the
    earlier); children of a node that is left out are left out too."""
    out, place, level, children = [], {-1: -1}, {-1: 0}, {}
    for index, (token, parent) in enumerate(drafted):
        if not -1 <= parent < index:
            raise ValueError("a drafted node's parent must come before it")
        at = place.get(parent)
        if at is None or not 0 <= token < vocab or level[at] >= depth:
            continue
        known = children.get((at, token))
        if known is None:
            if len(out) >= limit:
                continue
            known = children[at, token] = len(out)
            out.append((token, at))
            level[known] = level[at] + 1
        place[index] = known
    return out


class PromptLookup:
    """Drafts the continuations of earlier occurrences of the last tokens.

    For n = longest, ..., shortest it looks for the last n tokens earlier in the
    list, latest occurrence first, and proposes the `depth` tokens that followed
    each of up to `branches` occurrences (over all n), as one tree."""

    def __init__(self, depth: int = 8, branches: int = 4, longest: int = 3, shortest: int = 1):
        if depth < 1 or branches < 1 or not 1 <= shortest <= longest:
            raise ValueError("depth, branches and lengths must be positive, shortest <= longest")
        self.depth, self.branches = depth, branches
        self.longest, self.shortest = longest, shortest

    def propose(self, tokens, limit):
        tokens, found, ends = list(tokens), [], set()
        for n in range(self.longest, self.shortest - 1, -1):
            if n >= len(tokens):
                continue
            tail = tokens[-n:]
            for end in range(len(tokens) - 1, n - 1, -1):  # the occurrence's end
                if len(found) == self.branches:
                    break
                if end not in ends and tokens[end - n:end] == tail:
                    ends.add(end)
                    found.append(tokens[end:end + self.depth])
        out, children = [], {}
        for continuation in found:
            parent = -1
            for token in continuation:
                node = children.get((parent, token))
                if node is None:
                    if len(out) == limit:
                        break
                    node = children[parent, token] = len(out)
                    out.append((token, parent))
                parent = node
        return out

"""PromptLookup over growing texts: the same trees as a search from the definition, without
a walk over the whole text in every turn (host only)."""

import random
from types import SimpleNamespace

import pytest

from hisparse_b200 import PromptLookup
from hisparse_b200.engine import BatchedEngine, Request


def by_definition(lookup, tokens, limit):
    """Every size from the longest, every earlier end from the latest."""
    ends = []
    for n in range(lookup.longest, lookup.shortest - 1, -1):
        for end in range(len(tokens) - 1, n - 1, -1):
            if len(ends) < lookup.branches and end not in ends \
                    and tokens[end - n:end] == tokens[len(tokens) - n:]:
                ends.append(end)
    nodes = {}
    for end in ends:
        path = ()
        for token in tokens[end:end + lookup.depth]:
            if path + (token,) not in nodes and len(nodes) == limit:
                break
            path += (token,)
            nodes.setdefault(path, (token, list(nodes).index(path[:-1]) if path[1:] else -1))
    return list(nodes.values())


@pytest.mark.parametrize("seed", range(6))
def test_growing_text_equals_the_definition(seed):
    rng = random.Random(seed)
    for _ in range(60):
        shortest = rng.randrange(1, 4)
        lookup = PromptLookup(depth=rng.randrange(1, 6), branches=rng.randrange(1, 6),
                              shortest=shortest, longest=shortest + rng.randrange(3))
        vocab, limit = rng.choice([1, 2, 3, 6]), rng.choice([0, 1, 4, 63])
        tokens = [rng.randrange(vocab) for _ in range(rng.randrange(1, 30))]
        text = lookup.follow(tokens)
        for _ in range(4):
            want = by_definition(lookup, tokens, limit)
            assert text.propose(limit) == lookup.propose(tokens, limit) == want
            more = [rng.randrange(vocab) for _ in range(rng.randrange(4))]
            tokens = tokens + more
            text.extend(more)


class Counted(int):
    """A token that counts how often it is compared."""

    compared = 0

    def __eq__(self, other):
        Counted.compared += 1
        return int(self) == int(other)

    __hash__ = int.__hash__


def stand_in_engine(drafter):
    engine = object.__new__(BatchedEngine)
    engine.drafter, engine._texts, engine.eos_token_id = drafter, {}, None
    engine.model = SimpleNamespace(config=SimpleNamespace(vocab_size=1 << 20))
    engine.cache = SimpleNamespace(release_request=lambda *a, **k: None)
    engine.requests, engine.waiting, engine.running = {}, [], []
    return engine


def test_turns_do_not_walk_the_whole_text():
    """20 turns over 5,000 tokens without a match: a comparison for every place of the
    text and size, in Python, would be 300,000."""
    engine = stand_in_engine(PromptLookup())
    request = Request("r", [Counted(i) for i in range(5000)], 100)
    Counted.compared = 0
    for turn in range(20):
        request.generated.append(Counted(6000 + turn))
        assert engine._draft(request) == []
    assert Counted.compared < 5000


class Following:
    """Records what it is handed."""

    def __init__(self):
        self.log = []

    def follow(self, tokens):
        self.log.append(("follow", list(tokens)))
        return self

    def extend(self, tokens):
        self.log.append(("extend", list(tokens)))

    def propose(self, limit):
        return [(7, -1)]


def test_engine_hands_over_new_tokens_only_and_forgets_ended_requests():
    drafter = Following()
    engine = stand_in_engine(drafter)
    a, b = Request("a", [1, 2], 9, generated=[3]), Request("b", [4], 3, generated=[5])
    for r in (a, b):
        engine.requests[r.request_id] = r
        assert engine._draft(r) == [(7, -1)]
    assert drafter.log == [("follow", [1, 2, 3]), ("follow", [4, 5])]
    a.generated += [6, 8]
    assert engine._draft(a) == engine._draft(a) == [(7, -1)]
    assert drafter.log[2:] == [("extend", [6, 8])]
    assert set(engine._texts) == {"a", "b"}
    engine._emit(b, 1)
    assert engine._draft(b) == [] and not b.finished  # one token left: nothing to draft
    engine._emit(b, 1)
    assert b.finished and set(engine._texts) == {"a"}
    engine.running.append(a)
    engine.cancel("a")
    assert engine._texts == {}


def test_a_propose_of_its_own_is_what_counts():
    class Mine(PromptLookup):
        def propose(self, tokens, limit):
            return [(len(tokens), -1)]

    one = PromptLookup()
    one.propose = lambda tokens, limit: [(len(tokens), -1)]
    for drafter in (Mine(), one, SimpleNamespace(propose=lambda t, limit: [(len(t), -1)])):
        engine = stand_in_engine(drafter)
        request = Request("r", [1, 1, 1], 9, generated=[1])
        assert engine._draft(request) == [(4, -1)]
        request.generated.append(1)
        assert engine._draft(request) == [(5, -1)]
    engine.drafter = PromptLookup(depth=1, branches=1)  # exchanged while the request runs
    assert engine._draft(request) == [(1, -1)]

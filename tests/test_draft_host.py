"""Drafted trees on the host: PromptLookup and the engine's reading of a draft."""

import pytest

from hisparse_b200 import PromptLookup
from hisparse_b200.draft import tree_of


def paths(tree):
    """Every root-to-node token path of (token, parent) pairs."""
    out = []
    for token, parent in tree:
        out.append((out[parent] if parent >= 0 else ()) + (token,))
    return out


def test_prompt_lookup_continues_earlier_occurrences():
    tokens = [1, 2, 3, 4, 9, 1, 2, 3, 5, 6, 1, 2, 3]
    tree = PromptLookup(depth=2, branches=2, longest=3).propose(tokens, 63)
    assert paths(tree) == [(5,), (5, 6), (4,), (4, 9)]  # the latest occurrence first
    one = PromptLookup(depth=3, branches=1, longest=3).propose(tokens, 63)
    assert paths(one) == [(5,), (5, 6), (5, 6, 1)]
    assert paths(PromptLookup(depth=8, branches=4).propose(tokens, 3)) == \
        [(5,), (5, 6), (5, 6, 1)]


def test_prompt_lookup_merges_and_falls_back_to_shorter_matches():
    tokens = [7, 8, 1, 7, 8, 2, 5, 8, 3, 7, 8]
    tree = PromptLookup(depth=1, branches=4, longest=2, shortest=1).propose(tokens, 63)
    assert paths(tree) == [(2,), (1,), (3,)]
    same = PromptLookup(depth=2, branches=3, longest=1).propose([4, 4, 4, 4], 63)
    assert paths(same) == [(4,), (4, 4)]
    assert PromptLookup().propose([1, 2, 3], 63) == []
    assert PromptLookup().propose([1], 63) == []


@pytest.mark.parametrize("bad", [dict(depth=0), dict(branches=0), dict(shortest=0),
                                 dict(longest=1, shortest=2)])
def test_prompt_lookup_refusals(bad):
    with pytest.raises(ValueError):
        PromptLookup(**bad)


def test_tree_of_limits():
    draft = [(5, -1), (6, 0), (7, 1), (5, -1), (8, 3), (99, -1), (1, 5), (-1, 0), (9, 2)]
    assert tree_of(draft, 63, 9, 50) == [(5, -1), (6, 0), (7, 1), (8, 0), (9, 2)]
    assert tree_of(draft, 63, 2, 50) == [(5, -1), (6, 0), (8, 0)]
    assert tree_of(draft, 2, 9, 50) == [(5, -1), (6, 0)]
    assert tree_of([], 63, 9, 50) == []
    for bad in ([(1, 0)], [(1, -2)], [(1, -1), (2, 1)]):
        with pytest.raises(ValueError):
            tree_of(bad, 63, 9, 50)


def test_decoder_weights_with_head_norms_round_trip():
    import torch

    from hisparse_b200.engine import DecoderConfig, DecoderWeights

    shape = dict(vocab_size=32, hidden_size=16, intermediate_size=24, num_hidden_layers=2,
                 num_attention_heads=4, num_key_value_heads=2)
    plain = DecoderWeights.random(DecoderConfig(**shape), 5, device="cpu", dtype=torch.float32)
    assert not any("q_norm" in k for k in plain.state_dict())
    config = DecoderConfig(**shape, qk_norm=True)
    weights = DecoderWeights.random(config, 5, device="cpu", dtype=torch.float32)
    state = weights.state_dict()
    assert state["model.layers.1.self_attn.k_norm.weight"].shape == (4,)
    again = DecoderWeights(config, state).state_dict()
    assert state.keys() == again.keys()
    assert all(torch.equal(state[k], again[k]) for k in state)

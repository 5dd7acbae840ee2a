"""Calls at the edges of what the verification operators' documentation allows."""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


def flags():
    from hisparse_b200 import _lib

    return _lib.device_flags(DEV)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("width", [0, 40])
def test_tree_marks_of_values_that_are_not_finite(dtype, dim, width):
    """The marks of such values are written by the warps that copy them and read by the
    softmax warps as soon as the products are done. The shortest way from one to the
    other: one or two blocks of keys, the value in the last one, on every SM at once."""
    from hisparse_b200 import attend_tree, tree_mask
    from test_gpu_verify_ops import tree_inputs

    batch, nodes = 96, 30
    (q, k, v), _, pool, rows, config = tree_inputs(batch, nodes, 8, 4, dim, 16, width, dtype, 51)
    mask = tree_mask([[-1] + [(t - 1) // 2 for t in range(1, nodes)]] * batch, DEV)
    clean = attend_tree(q, k, v, mask, pool, rows, config)
    v[:, 29, 3, dim - 1] = math.inf  # a leaf: only it sees its value
    v[:, 0, 1, 0] = math.nan         # the root: every node does
    for _ in range(20):
        got = attend_tree(q, k, v, mask, pool, rows, config)
        assert bool((got[:, 29, 6:, dim - 1] == math.inf).all())
        assert bool(got[:, :, 2:4, 0].isnan().all())
        same = torch.ones_like(got, dtype=torch.bool)
        same[:, 29, 6:, dim - 1] = False
        same[:, :, 2:4, 0] = False
        assert torch.equal(got[same], clean[same])
    assert not flags()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("offset", [0, 1, 3])
def test_logprobs_of_the_longest_row(dtype, offset):
    """2^31 - 1 entries, the most that is accepted, from a 16-byte boundary and off it:
    few entries above -inf, at both ends and in the middle, so that every sum is short."""
    from hisparse_b200 import token_logprobs

    v = 2 ** 31 - 1
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    buffer = torch.full((v + offset,), -math.inf, dtype=dtype, device=DEV)
    logits = buffer[offset:].view(1, v)
    at = {0: 1.0, 1: 0.5, v // 2: 0.25, v - 2: 1.5, v - 1: 2.0}
    for index, value in at.items():
        logits[0, index] = value
    tokens = torch.tensor([[*at, 7, v, -1]], device=DEV)
    got = token_logprobs(logits, tokens, top=6)
    lse = math.log(sum(math.exp(x) for x in at.values()))
    want = [x - lse for x in at.values()]
    # five exps (2 f each and f of an exponent of at most 1.75), their sums, a logarithm and
    # two differences of at most 2: under 32 f
    bound = 32 * 2.0 ** -24
    have = got.logprobs[0].tolist()
    assert all(abs(a - b) < bound for a, b in zip(have, want))
    assert have[5] == -math.inf and math.isnan(have[6]) and have[7] == 0
    entropy = -sum(math.exp(x) * x for x in want)
    assert abs(got.entropy.item() - entropy) < bound
    order = sorted(at, key=lambda i: -at[i])
    assert got.top_tokens[0].tolist() == order + [2]
    top = got.top_logprobs[0].tolist()
    assert all(abs(a - (at[i] - lse)) < bound for a, i in zip(top, order)) and top[5] == -math.inf
    assert flags()  # the token past the vocabulary


def test_operators_refuse_forward_mode_tangents():
    from torch.autograd import forward_ad

    from hisparse_b200 import attend_tree, qk_norm_rope, rope_frequencies, token_logprobs, tree_mask
    from test_gpu_verify_ops import tree_inputs

    (q, k, v), parents, pool, rows, config = tree_inputs(1, 3, 4, 2, 32, 16, 20, torch.float32, 52)
    mask, positions = tree_mask(parents, DEV), torch.arange(3, device=DEV)
    freq = rope_frequencies(32, 1e4, DEV)
    want = attend_tree(q, k, v, mask, pool, rows, config)
    with forward_ad.dual_level():
        tangent = forward_ad.make_dual(v, torch.ones_like(v))
        for call in (lambda: attend_tree(q, k, tangent, mask, pool, rows, config),
                     lambda: qk_norm_rope(q[0], tangent[0], positions, freq),
                     lambda: token_logprobs(tangent[0, :, 0], positions, top=1)):
            with pytest.raises(ValueError, match="no derivative"):
                call()
        # inside a level, tensors without a tangent are taken as ever
        assert torch.equal(attend_tree(q, k, v, mask, pool, rows, config), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("rows,kbytes,threads,top", [
    (2, 512, 256, 32), (2, 512, 256, 7), (300, 60, 256, 32), (601, 60, 128, 32), (601, 60, 128, 2)])
def test_logprobs_large_entries_of_few_threads(dtype, rows, kbytes, threads, top):
    """Entries that pass the threshold are collected up to 1,024 a block. Rows whose large
    entries all fall to fewer than `top` threads pass with more: the threshold is then a
    small entry's, and the alternatives are found by one pass each. In 8 blocks a row (512
    KB), in one block, and in one of half the threads."""
    from hisparse_b200 import token_logprobs
    from test_gpu_verify_ops import logprobs_check

    size = torch.tensor([], dtype=dtype).element_size()
    vocab, n = kbytes * 1024 // size, 16 // size
    i = torch.arange(vocab)
    large = i // n % threads < top - 1
    values = torch.stack([(1 + r % 5) * 100 + (i * 7919 + r) % 601 for r in range(min(rows, 6))])
    logits = torch.where(large, values, torch.randn(len(values), vocab)).to(dtype)
    blocks = 8 if kbytes == 512 else 1
    if top == 32:
        assert all(part.sum() > 1024 for part in large.view(blocks, -1))
    logits = logits.repeat(-(-rows // len(values)), 1)[:rows].contiguous().to(DEV)
    tokens = torch.arange(rows, device=DEV) * 31 % vocab
    got = token_logprobs(logits, tokens, top=top)
    for part in (slice(0, 6), slice(rows - 6, rows)) if rows > 6 else (slice(0, rows),):
        logprobs_check(type(got)(*(x[part] for x in got)), logits[part], tokens[part], top)
    again = token_logprobs(logits, tokens, top=top)
    assert all(torch.equal(x, y) for x, y in zip(got, again))
    assert not flags()

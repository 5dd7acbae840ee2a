"""The operators of a verification step against their formulas in fp64.

Tolerances are bounds on the arithmetic, written beside each comparison: u is
half a step of the output type (bf16 2^-8, fp16 2^-11, fp32 2^-24), f = 2^-24
the fp32 rounding of an intermediate.
"""

from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
F = 2.0 ** -24
FP32, FP16, BF16 = torch.float32, torch.float16, torch.bfloat16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_within(got, want, bound):
    """|got - want| <= bound elementwise, infinities and NaN in the same places."""
    got, want, bound = got.double().cpu(), want.double().cpu(), bound.double().cpu()
    finite = torch.isfinite(want)
    same = (got == want) | (got.isnan() & want.isnan())
    assert bool(same[~finite].all()), "infinities or NaN differ"
    excess = ((got - want).abs() - bound)[finite]
    assert not excess.isnan().any(), "a finite value came out as NaN"
    assert excess.numel() == 0 or excess.max().item() <= 0, \
        f"error above its bound by {excess.max().item():.3e}"


def flags():
    from hisparse_b200 import _lib

    return _lib.device_flags(DEV)


# ---- norms and rotation --------------------------------------------------------------------
def norm_rope_reference(x, weight, positions, inv_freq, eps):
    """(out, |y_i| + |y_{i+R}| for every element) in fp64."""
    y = x.double().cpu()
    if weight is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double().cpu()
    angle = positions.double().cpu()[:, None] * inv_freq.cpu()[None, :]
    c, s = angle.cos()[:, None], angle.sin()[:, None]
    a, b = y.chunk(2, -1)
    size = a.abs() + b.abs()
    return torch.cat((a * c - b * s, b * c + a * s), -1), torch.cat((size, size), -1)


def norm_rope_check(got, x, weight, positions, inv_freq, eps):
    """fp32 errors: the squares' mean (<= 12 f), rsqrt (2 f), two products of the
    norm (2 f), cos and sin (4 f: the fraction's rounding and the function's),
    the two products and the sum (2 f): under 32 f of |y_i| + |y_{i+R}|; then one
    rounding, with fp16's smallest step for results below its normal range."""
    want, size = norm_rope_reference(x, weight, positions, inv_freq, eps)
    arithmetic = 32 * F * size
    bound = arithmetic + half_step(got.dtype) * (want.abs() + arithmetic)
    if got.dtype == FP16:
        bound = bound + 2.0 ** -25
    assert got.is_contiguous() and got.shape == x.shape and got.dtype == x.dtype
    assert_within(got, want, bound)


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("tokens,hq,hkv,dim", [
    (1, 8, 2, 32), (1, 1, 1, 2), (5, 10, 2, 80), (3, 3, 3, 6), (130, 28, 4, 128),
    (7, 12, 1, 256), (33, 5, 5, 96), (2, 16, 16, 64), (3, 7, 1, 250), (1025, 32, 8, 128)])
@pytest.mark.parametrize("normed", [True, False])
def test_norm_rope(dtype, tokens, hq, hkv, dim, normed):
    from hisparse_b200 import qk_norm_rope, rope_frequencies

    gen = torch.Generator().manual_seed(tokens * 1000 + dim)
    fused = torch.randn(tokens, (hq + 2 * hkv) * dim, generator=gen).to(dtype).to(DEV)
    q, k = fused[:, :hq * dim].view(tokens, hq, dim), \
        fused[:, hq * dim:(hq + hkv) * dim].view(tokens, hkv, dim)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen)
    positions[0] = (1 << 20) - 1
    inv_freq = rope_frequencies(dim, 10000.0, DEV)
    wq = wk = None
    if normed:
        wq = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype).to(DEV)
        wk = (1 + 0.2 * torch.randn(dim, generator=gen)).to(dtype).to(DEV)
    for integer in (torch.int32, torch.int64):
        p = positions.to(integer).to(DEV)
        oq, ok = qk_norm_rope(q, k, p, inv_freq, wq, wk, eps=1e-6)
        norm_rope_check(oq, q, wq, p, inv_freq, 1e-6)
        norm_rope_check(ok, k, wk, p, inv_freq, 1e-6)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_norm_rope_strides_and_alignment(dtype):
    """Head-major views, rows that start off a 16-byte boundary, a transposed
    inner dimension, strided positions and an expanded token."""
    from hisparse_b200 import qk_norm_rope, rope_frequencies

    gen = torch.Generator().manual_seed(5)
    n, hq, hkv, dim = 9, 4, 2, 64
    base = torch.randn(hq, n, dim, generator=gen).to(dtype).to(DEV)
    odd = torch.randn(n * hkv * dim + 1, generator=gen).to(dtype).to(DEV)
    positions = torch.arange(2 * n, device=DEV)[::2]
    inv_freq = rope_frequencies(2 * dim, 1e6, DEV)[::2]
    w = torch.linspace(0.5, 1.5, 2 * dim, device=DEV).to(dtype)
    for q, k in ((base.transpose(0, 1), odd[1:].view(n, hkv, dim)),
                 (odd[1:].view(n, hkv, dim), base[:, :, :].transpose(0, 1)),
                 (base.transpose(0, 1).transpose(1, 2).contiguous().transpose(1, 2),
                  base[:1, :1].expand(n, hkv, dim))):
        for wq, wk in ((w[::2], w[1:dim + 1]), (None, w[:dim])):
            oq, ok = qk_norm_rope(q, k, positions, inv_freq, wq, wk, eps=1e-5)
            norm_rope_check(oq, q, wq, positions, inv_freq, 1e-5)
            norm_rope_check(ok, k, wk, positions, inv_freq, 1e-5)


def test_norm_rope_far_and_negative_positions():
    """Angles keep their fraction of a turn at positions past 2^31; a negative
    position turns the other way. (The fp64 product itself is off by 2^-53 of
    the angle: 2.5e-7 rad at 2^31, so the reference reduces the exact product.)"""
    from hisparse_b200 import qk_norm_rope, rope_frequencies

    gen = torch.Generator().manual_seed(6)
    positions = torch.tensor([-1, -70000, 0, 2 ** 31 - 1, 2 ** 31 + 12345, 10 ** 9])
    x = torch.randn(len(positions), 2, 128, generator=gen).to(DEV)
    inv_freq = rope_frequencies(128, 10000.0, DEV)
    out, _ = qk_norm_rope(x, x, positions.to(DEV), inv_freq)
    import numpy as np

    angle = np.outer(positions.numpy().astype(np.longdouble),
                     inv_freq.cpu().numpy().astype(np.longdouble))
    c, s = torch.tensor(np.cos(angle).astype(np.float64)), torch.tensor(
        np.sin(angle).astype(np.float64))
    a, b = x.double().cpu().chunk(2, -1)
    want = torch.cat((a * c[:, None] - b * s[:, None], b * c[:, None] + a * s[:, None]), -1)
    size = torch.cat((a.abs() + b.abs(),) * 2, -1)
    # 32 f as above and the fp64 product's error, three half steps of up to 2^31 rad
    assert_within(out, want, (33 * F + 3 * 2.0 ** 31 * 2.0 ** -53) * size)


def test_norm_rope_extreme_values():
    """A zero row keeps to zero through eps; large and small rows keep their
    direction; NaN stays within its head; nothing at all is a no-op."""
    from hisparse_b200 import qk_norm_rope, rope_frequencies

    inv_freq = rope_frequencies(64, 10000.0, DEV)
    x = torch.ones(4, 3, 64, device=DEV)
    x[0] = 0
    x[1] *= 1e15
    x[2] *= 1e-3
    x[3, 1, 7] = float("nan")
    w = torch.ones(64, device=DEV)
    p = torch.arange(4, device=DEV)
    out, _ = qk_norm_rope(x, x, p, inv_freq, w, w, eps=1e-12)
    assert bool((out[0] == 0).all())
    good = [0, 1, 2]
    norm_rope_check(out[good].contiguous(), x[good], w, p[good], inv_freq, 1e-12)
    assert bool(out[3, 1].isnan().any()) and not bool(out[3, [0, 2]].isnan().any())
    q, k = qk_norm_rope(x[:0], x[:0, :1], p[:0], inv_freq)
    assert q.shape == (0, 3, 64) and k.shape == (0, 1, 64)


def test_norm_rope_refusals():
    from hisparse_b200 import qk_norm_rope, rope_frequencies

    x = torch.zeros(2, 2, 32, device=DEV)
    p, f = torch.zeros(2, dtype=torch.int64, device=DEV), rope_frequencies(32, 1e4, DEV)
    w = torch.ones(32, device=DEV)
    with pytest.raises(ValueError, match="one dtype"):
        qk_norm_rope(x, x.half(), p, f)
    with pytest.raises(ValueError, match="key must be"):
        qk_norm_rope(x, x[:1], p, f)
    with pytest.raises(ValueError, match="query must be"):
        qk_norm_rope(x[0], x, p, f)
    with pytest.raises(ValueError, match="positions"):
        qk_norm_rope(x, x, p.float(), f)
    with pytest.raises(ValueError, match="positions"):
        qk_norm_rope(x, x, p[:1], f)
    with pytest.raises(ValueError, match="inv_freq"):
        qk_norm_rope(x, x, p, f.float())
    with pytest.raises(ValueError, match="norm weights"):
        qk_norm_rope(x, x, p, f, w[:31], w)
    with pytest.raises(ValueError, match="norm weights"):
        qk_norm_rope(x, x, p, f, w, w.half())
    with pytest.raises(ValueError, match="even"):
        qk_norm_rope(x[..., :31], x[..., :31], p, f[:15])
    with pytest.raises(ValueError, match="not supported"):
        big = torch.zeros(2, 2, 258, device=DEV)
        qk_norm_rope(big, big, p, rope_frequencies(258, 1e4, DEV))
    with pytest.raises(ValueError, match="eps"):
        qk_norm_rope(x, x, p, f, w, w, eps=-1.0)
    with pytest.raises(ValueError, match="unsupported element type"):
        qk_norm_rope(x.double(), x.double(), p, f)
    with pytest.raises(ValueError, match="CUDA"):
        qk_norm_rope(x, x, p.cpu(), f)


# ---- log probabilities -----------------------------------------------------------------------
def logprobs_reference(logits, tokens, top):
    x = logits.double().cpu()
    empty = (x == -math.inf).all(-1)
    logp = torch.log_softmax(x, -1)
    logp[empty] = -math.inf
    p = logp.exp()
    entropy = -torch.special.xlogy(p, p).sum(-1)
    entropy[empty] = 0
    given = None
    if tokens is not None:
        tokens = tokens.cpu().long()
        given = logp.gather(1, tokens.clamp(min=0).view(len(x), -1)).view(tokens.shape)
        given = given.masked_fill(tokens < 0, 0.0)
    rank = torch.where(x.isnan(), torch.full_like(x, math.inf), x)
    nan_first = x.isnan().long()
    order = []
    for row, nans in zip(rank, nan_first):
        keyed = sorted(range(len(row)), key=lambda i: (-nans[i].item(), -row[i].item(), i)) \
            if len(row) <= 4096 else torch.sort(row, descending=True, stable=True).indices.tolist()
        order.append(keyed[:top])
    order = torch.tensor(order, dtype=torch.int64).view(len(x), top)
    return given, entropy, logp.gather(1, order), order


def logprobs_check(got, logits, tokens, top):
    """log s: every exp is off by 2 f and by f of its exponent's size (which its
    weight exp(d) |d| < 0.37 takes back under f), and a sum of vocab entries over
    at least 128 partial sums by (vocab / 128 + 32) f of s; (x - m) and the last
    difference by f of their size each. The entropy's quotient t / s has the
    sums' error twice, of at most log(vocab)."""
    vocab = logits.shape[1]
    sums = (vocab / 128 + 64) * F
    given, entropy, top_lp, top_tok = logprobs_reference(logits, tokens, top)
    if given is None:
        assert got.logprobs.shape == (logits.shape[0], 0)
    else:
        assert got.logprobs.shape == given.shape
        assert_within(got.logprobs, given, sums + 4 * F * given.abs())
    assert_within(got.entropy, entropy, 2 * sums * (1 + math.log(vocab)) * torch.ones_like(entropy))
    assert torch.equal(got.top_tokens.cpu(), top_tok)
    assert_within(got.top_logprobs, top_lp, sums + 4 * F * top_lp.abs())
    assert got.logprobs.dtype == got.entropy.dtype == got.top_logprobs.dtype == FP32


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("rows,vocab,given,top", [
    (1, 1, 1, 1), (1, 2, 1, 2), (3, 7, 2, 7), (2, 31, 1, 20), (5, 257, 4, 32), (1, 1024, 1, 4),
    (4, 1003, 3, 0), (2, 50257, 1, 5), (1, 128256, 1, 20), (19, 4099, 2, 1), (300, 2049, 1, 3)])
def test_logprobs(dtype, rows, vocab, given, top):
    from hisparse_b200 import token_logprobs

    gen = torch.Generator().manual_seed(rows * vocab)
    logits = (3 * torch.randn(rows, vocab, generator=gen)).to(dtype).to(DEV)
    tokens = torch.randint(-1, vocab, (rows, given), generator=gen)
    tokens[0, 0] = vocab - 1
    for t in (tokens.to(DEV), tokens[:, 0].int().to(DEV), None):
        logprobs_check(token_logprobs(logits, t, top=top), logits, t, top)
    assert not flags()


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("rows,vocab,given,top", [
    (700, 4099, 3, 5), (1300, 4104, 1, 32), (650, 8190, 200, 1), (640, 30011, 1, 20)])
def test_logprobs_more_rows_than_places(dtype, rows, vocab, given, top):
    """More rows than the GPU holds blocks for: blocks of half the threads, also with
    more given tokens than those, odd row strides and every row twice."""
    from hisparse_b200 import token_logprobs

    gen = torch.Generator().manual_seed(rows * vocab)
    logits = (3 * torch.randn(rows // 2, vocab, generator=gen)).to(dtype)
    logits[1] = 0.5                       # all equal
    logits[2, ::2] = -math.inf
    logits[3] = torch.finfo(dtype).min
    logits[4] = (torch.arange(vocab) % 2).to(dtype)
    tokens = torch.randint(-1, vocab, (rows // 2, given), generator=gen)
    logits, tokens = logits.to(DEV), tokens.to(DEV)
    got = token_logprobs(logits.repeat(2, 1), tokens.repeat(2, 1), top=top)
    for half in (slice(0, rows // 2), slice(rows // 2, None)):
        logprobs_check(type(got)(*(x[half] for x in got)), logits, tokens, top)
    assert not flags()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_logprobs_ties_and_orders(dtype):
    """Equal logits go to the lower token, in constant, ascending, descending and
    two-valued rows (every entry an alternative's rival), -0 beside +0."""
    from hisparse_b200 import token_logprobs

    v = 3001
    rows = [torch.zeros(v), torch.arange(v).float() / 16, -torch.arange(v).float() / 16,
            (torch.arange(v) % 2).float(), (torch.arange(v) % 64).float(),
            torch.where(torch.arange(v) % 3 == 0, -0.0, 0.0),
            torch.where(torch.arange(v) > v - 10, 5.0, torch.randn(v)),
            torch.full((v,), torch.finfo(dtype).min), torch.full((v,), -1e4)]
    logits = torch.stack(rows).to(dtype).to(DEV)
    logprobs_check(token_logprobs(logits, top=32), logits, None, 32)


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
def test_logprobs_masked_and_nonfinite_rows(dtype):
    """-inf entries, a row with nothing else, rows of the type's lowest value
    beside -inf, and rows with +inf or NaN (all their results are NaN)."""
    from hisparse_b200 import token_logprobs

    v, inf, nan = 517, math.inf, math.nan
    gen = torch.Generator().manual_seed(3)
    logits = (2 * torch.randn(9, v, generator=gen)).to(dtype)
    logits[0, 1::2] = -inf
    logits[1, :] = -inf
    logits[2, :] = -inf
    logits[2, 300] = -4.0
    logits[3, :] = torch.finfo(dtype).min
    logits[3, 10:400] = -inf
    logits[4, 77] = nan
    logits[5, 0] = nan
    logits[5, 1:] = -inf
    logits[6, 200] = inf
    logits[7, 516] = nan
    logits[7, 3] = inf
    logits = logits.to(DEV)
    tokens = torch.tensor([[0, 1, 300, -1]] * 9, device=DEV)
    got = token_logprobs(logits, tokens, top=8)
    bad = [4, 5, 6, 7]
    fine = [0, 1, 2, 3, 8]
    pick = type(got)(*(x[fine] for x in got))
    logprobs_check(pick, logits[fine], tokens[fine], 8)
    assert bool(got.logprobs[bad][:, :3].isnan().all()) and bool(got.entropy[bad].isnan().all())
    assert bool((got.logprobs[:, 3] == 0).all())
    assert bool(got.top_logprobs[bad].isnan().all())
    want = logprobs_reference(logits[bad], None, 8)[3]
    assert torch.equal(got.top_tokens[bad].cpu(), want)


def test_logprobs_strides_and_tokens():
    """Rows off 16-byte boundaries, a strided inner dimension, an expanded row;
    a token past the vocabulary gives NaN and a device flag."""
    from hisparse_b200 import _lib, token_logprobs

    gen = torch.Generator().manual_seed(4)
    for dtype in (FP32, BF16):
        wide = torch.randn(6, 2 * 1031, generator=gen).to(dtype).to(DEV)
        for logits in (wide[:, 1:1030], wide[:, ::2], wide[:1, 3:700].expand(4, 697),
                       wide[::2, 5:6], wide.t()[:, :5]):
            top = min(6, logits.shape[1])
            logprobs_check(token_logprobs(logits, top=top), logits, None, top)
    assert not flags()
    got = token_logprobs(wide, torch.tensor([0, 5, 2062, 1 << 40, 3, -7], device=DEV))
    assert got.logprobs.isnan().tolist() == [False, False, True, True, False, False]
    assert got.logprobs[5].item() == 0
    assert flags() == [_lib.DEVICE_FLAGS[64]]
    none = token_logprobs(wide[:0], torch.zeros(0, 3, dtype=torch.int64, device=DEV), top=2)
    assert [tuple(t.shape) for t in none] == [(0, 3), (0,), (0, 2), (0, 2)]


def test_logprobs_rows_past_32_bits():
    """The last rows of logits with more than 2^32 elements."""
    from hisparse_b200 import token_logprobs

    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    rows, vocab = 34000, 128256
    logits = torch.zeros((rows, vocab), dtype=BF16, device=DEV)
    tail = (3 * torch.randn(3, vocab, generator=torch.Generator().manual_seed(9))).to(BF16).to(DEV)
    logits[-3:] = tail
    tokens = torch.full((rows,), 70000, device=DEV)
    got = token_logprobs(logits, tokens, top=4)
    # (few rows are split over blocks and many are not: their sums' order differs, so
    # the last rows are held against the formula, not against a call of their own)
    logprobs_check(type(got)(*(t[-3:] for t in got)), tail, tokens[-3:], 4)
    assert got.top_tokens[0].tolist() == [0, 1, 2, 3]
    assert abs(got.entropy[0].item() - math.log(vocab)) < 1e-4


def test_logprobs_refusals():
    from hisparse_b200 import token_logprobs

    x = torch.zeros(2, 40, device=DEV)
    with pytest.raises(ValueError, match="logits must be"):
        token_logprobs(x[0])
    with pytest.raises(ValueError, match="logits must be"):
        token_logprobs(x[:, :0])
    with pytest.raises(ValueError, match="top must be"):
        token_logprobs(x, top=41)
    with pytest.raises(ValueError, match="top must be"):
        token_logprobs(x, top=-1)
    with pytest.raises(ValueError, match="not supported"):
        token_logprobs(x, top=33)
    with pytest.raises(ValueError, match="tokens must be"):
        token_logprobs(x, torch.zeros(2, device=DEV))
    with pytest.raises(ValueError, match="tokens must be"):
        token_logprobs(x, torch.zeros(3, dtype=torch.int64, device=DEV))
    with pytest.raises(ValueError, match="unsupported element type"):
        token_logprobs(x.double())
    with pytest.raises(ValueError, match="CUDA"):
        token_logprobs(x.cpu())


# ---- tree attention --------------------------------------------------------------------------
def tree_inputs(batch, nodes, hq, hkv, dim, page, width, dtype, seed, scale=1.0):
    from hisparse_b200 import CacheConfig

    gen = torch.Generator().manual_seed(seed)
    pages = -(-max(width, 1) // page)
    blocks = batch * pages + 3
    pool = torch.randn(blocks, 2, page, hkv, dim, generator=gen).to(dtype)
    order = torch.randperm(blocks, generator=gen)[:batch * pages].view(batch, pages)
    rows = (order[:, :, None] * page + torch.arange(page)).reshape(batch, -1)[:, :width]
    q = (scale * torch.randn(batch, nodes, hq, dim, generator=gen)).to(dtype)
    k = torch.randn(batch, nodes, hkv, dim, generator=gen).to(dtype)
    v = torch.randn(batch, nodes, hkv, dim, generator=gen).to(dtype)
    parents = [[-1] + [int(torch.randint(0, t, (1,), generator=gen)) for t in range(1, nodes)]
               for _ in range(batch)]
    config = CacheConfig(gpu_pages=blocks, page_size=page, kv_heads=hkv, head_dim=dim,
                         device=DEV, dtype=dtype)
    return [x.to(DEV) for x in (q, k, v)], parents, pool.to(DEV), rows.contiguous().to(DEV), config


def tree_reference(q, k, v, mask, pool, rows, counts=None, nodes=None):
    """(out, sum p |v|, largest |q| |k| / sqrt(D)) in fp64, pair by pair."""
    q, k, v, pool, rows, mask = (x.cpu() for x in (q, k, v, pool, rows, mask))
    batch, width, hq, dim = q.shape
    page, hkv = pool.shape[2], pool.shape[3]
    out = torch.zeros(q.shape, dtype=torch.float64)
    size, reach = torch.zeros_like(out), 0.0
    for b in range(batch):
        n = width if nodes is None else max(0, min(width, int(nodes[b])))
        c = rows.shape[1] if counts is None else max(0, min(rows.shape[1], int(counts[b])))
        r = rows[b, :c]
        r = r[(r >= 0) & (r // page < pool.shape[0])]
        cache = [pool[r // page, i, r % page].double() for i in (0, 1)]
        for t in range(n):
            seen = [j for j in range(n) if int(mask[b, t]) >> j & 1]
            if not seen and not len(r):
                continue
            kk = torch.cat((cache[0], k[b, seen].double()))
            vv = torch.cat((cache[1], v[b, seen].double()))
            qq = q[b, t].double().view(hkv, hq // hkv, dim)
            p = torch.softmax(torch.einsum("hgd,nhd->hgn", qq, kk) / math.sqrt(dim), -1)
            out[b, t] = torch.einsum("hgn,nhd->hgd", p, vv).reshape(hq, dim)
            size[b, t] = torch.einsum("hgn,nhd->hgd", p, vv.abs()).reshape(hq, dim)
            reach = max(reach, (qq.norm(dim=-1).max() * kk.norm(dim=-1).max()).item())
    return out, size, reach / math.sqrt(dim)


def tree_check(got, inputs, mask, pool, rows, counts=None, nodes=None):
    """A score is off by (D + 4) f of |q| |k| / sqrt(D) at most, so a weight by that
    twice (its own and the sum's) and by 8 f for exp2 and the joins; a weight that
    is rounded to the type of the values by u; sums of K terms by K f. All of it
    applies to sum p |v|. One rounding of the result follows."""
    want, size, reach = tree_reference(*inputs, mask, pool, rows, counts, nodes)
    u = half_step(got.dtype)
    dim, keys = got.shape[3], rows.shape[1] + got.shape[1]
    relative = 2 * (dim + 4) * F * reach + (keys + 32) * F
    if got.dtype != FP32:
        relative += u
    bound = relative * size + u * (want.abs() + relative * size)
    if got.dtype == FP16:
        bound = bound + 2.0 ** -24
    assert got.is_contiguous() and got.dtype == inputs[0].dtype
    assert_within(got, want, bound)


SHAPES = [
    # batch, nodes, hq, hkv, dim, page, width
    (1, 1, 1, 1, 1, 1, 1), (2, 3, 4, 2, 2, 4, 5), (3, 5, 8, 2, 32, 16, 160),
    (1, 64, 8, 8, 64, 16, 300), (2, 7, 28, 4, 128, 64, 700), (1, 63, 28, 4, 128, 64, 1111),
    (2, 8, 32, 8, 128, 16, 513), (1, 17, 10, 2, 80, 12, 97), (2, 2, 12, 1, 256, 16, 130),
    (1, 33, 6, 6, 96, 5, 64), (1, 1, 16, 1, 200, 16, 257), (1, 4, 32, 8, 128, 16, 5000),
    (4, 16, 16, 4, 64, 16, 63), (2, 64, 16, 2, 128, 16, 190), (1, 5, 5, 1, 33, 3, 40),
    (1, 12, 8, 1, 128, 1, 129), (17, 3, 4, 4, 16, 16, 33),
    # an odd number of (row, split) pairs before the outputs of the splits
    (1, 1, 1, 1, 128, 16, 5000), (1, 3, 5, 1, 64, 16, 3000), (1, 1, 3, 3, 32, 16, 900),
    (1, 5, 1, 1, 256, 16, 2000), (1, 7, 3, 1, 20, 16, 700)]


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_tree(dtype, shape):
    from hisparse_b200 import attend_tree, tree_mask

    batch, nodes, *_, width = shape
    inputs, parents, pool, rows, config = tree_inputs(*shape, dtype, seed=sum(shape), scale=1.5)
    mask = tree_mask(parents, DEV)
    got = attend_tree(*inputs, mask, pool, rows, config)
    tree_check(got, inputs, mask, pool, rows)
    counts = torch.tensor([(width * (3 * b + 1)) // (3 * batch) for b in range(batch)],
                          dtype=torch.int32, device=DEV)
    lens = torch.tensor([max(0, nodes - 2 * b) for b in range(batch)], dtype=torch.int32,
                        device=DEV)
    got = attend_tree(*inputs, mask, pool, rows, config, counts=counts, nodes=lens)
    tree_check(got, inputs, mask, pool, rows, counts, lens)
    assert not flags()


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("dim", [64, 128, 72])
def test_tree_empty_rows_and_masks(dtype, dim):
    """No cache rows, rows that are all padding, a node that sees nothing, masks
    with bits beyond the tree, counts and node counts out of their range."""
    from hisparse_b200 import attend_tree

    inputs, _, pool, rows, config = tree_inputs(4, 64, 8, 2, dim, 16, 96, dtype, 11)
    mask = torch.full((4, 64), -1, dtype=torch.int64, device=DEV)
    mask[0, ::3] = 0
    mask[1] = torch.tensor([1 << 62, -2 ** 63, 3, 0] * 16, device=DEV)
    none = attend_tree(*inputs, mask, pool, rows[:, :0], config)
    tree_check(none, inputs, mask, pool, rows[:, :0])
    assert bool((none[0, ::3] == 0).all())
    padded = rows.clone()
    padded[0] = -1
    padded[1, 1:] = -5
    padded[2, ::2] = -1
    counts = torch.tensor([96, 96, 1 << 30, -3], dtype=torch.int32, device=DEV)
    lens = torch.tensor([64, 64, 65, -1], dtype=torch.int32, device=DEV)
    for c, n in ((None, None), (counts, None), (counts, lens),
                 (counts, torch.tensor([0, 1, 3, 40], dtype=torch.int32, device=DEV))):
        got = attend_tree(*inputs, mask, pool, padded, config, counts=c, nodes=n)
        tree_check(got, inputs, mask, pool, padded, c, n)
    assert not flags()


@pytest.mark.parametrize("dtype", [FP32, FP16, BF16])
@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dim", [128, 64, 36, 256])
def test_tree_nonfinite_values_out_of_sight(dtype, bad, dim):
    """What a node does not see takes no part, whatever it holds: other branches,
    padded nodes, rows behind counts and blocks that no row names. A node that
    sees a non-finite value gets it, in its own elements only."""
    from hisparse_b200 import attend_tree, tree_mask

    inputs, _, pool, rows, config = tree_inputs(2, 12, 8, 2, dim, 16, 96, dtype, 12)
    q, k, v = inputs
    parents = [[-1, 0, 1, 0, 3, 3, 0, 6, 7, 6, 6, 10]] * 2
    mask = tree_mask(parents, DEV)
    lens = torch.tensor([12, 9], dtype=torch.int32, device=DEV)
    counts = torch.tensor([96, 70], dtype=torch.int32, device=DEV)
    clean = attend_tree(q, k, v, mask, pool, rows, config, counts=counts, nodes=lens)
    k[:, 3] = bad            # seen by 3, 4, 5
    v[:, 6, 1, 9] = bad      # seen by 6 .. 11, KV head 1, element 9
    k[1, 9:], v[1, 9:], q[1, 9:] = bad, bad, bad
    hidden = rows[1, 70:]
    pool[hidden // 16, :, hidden % 16] = bad
    used = torch.zeros(pool.shape[0], dtype=torch.bool, device=DEV)
    used[(rows // 16).view(-1)] = True
    pool[~used] = bad
    got = attend_tree(q, k, v, mask, pool, rows, config, counts=counts, nodes=lens)
    same = torch.ones_like(got, dtype=torch.bool)
    same[:, 3:6] = False
    same[:, 6:12, 4:, 9] = False
    same[1, 9:] = True  # padded nodes: zero in both
    assert torch.equal(got[same], clean[same])
    assert bool((got[1, 9:] == 0).all())
    hit = got[0, 6:12, 4:, 9]
    assert bool(hit.isnan().all()) if math.isnan(bad) else bool((hit == bad).all())
    assert not flags()


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_tree_nonfinite_value_of_a_vanishing_weight(dtype):
    """A value that is not finite makes the result not finite however small its
    weight is, also when the splits are joined: 4,096 cache rows score 128, the
    node -128, so that its weight exp(-256) is 0 in fp32."""
    from hisparse_b200 import attend_tree, tree_mask

    (q, k, v), _, pool, rows, config = tree_inputs(1, 1, 2, 1, 64, 16, 4096, dtype, 21)
    q.fill_(8.0)
    pool[:, 0] = 2.0
    k.fill_(-2.0)
    v[..., 5] = math.inf
    got = attend_tree(q, k, v, tree_mask([[-1]], DEV), pool, rows, config)
    assert not got[..., 5].isfinite().any()
    rest = torch.arange(64, device=DEV) != 5
    assert got[..., rest].isfinite().all()
    want = pool[:, 1].double()[rows[0] // 16, rows[0] % 16].mean(0)  # equal scores
    # equal weights (exponents of up to 185 in fp32: 1 + 185 F each), an addition each of a
    # term of at most max |v| in fp32, one rounding
    bound = half_step(dtype) * want.abs() + 4400 * F * pool[:, 1].double().abs().max()
    assert_within(got[0, 0][:, rest], want[:, rest].expand(2, -1), bound[:, rest].expand(2, -1))


def test_tree_strided_inputs_and_bad_rows():
    """Views of a fused projection, an expanded row list, heads that are not
    adjacent; a row beyond the pool is skipped and flagged."""
    from hisparse_b200 import _lib, attend_tree, tree_mask

    for dtype, dim in ((FP32, 32), (BF16, 128), (BF16, 64), (FP16, 40), (BF16, 256)):
        inputs, parents, pool, rows, config = tree_inputs(3, 6, 8, 2, dim, 16, 100, dtype, 13)
        mask = tree_mask(parents, DEV)
        fused = torch.cat([x.flatten(2) for x in inputs], -1)
        views = [x.view(3, 6, -1, dim) for x in fused.split((8 * dim, 2 * dim, 2 * dim), -1)]
        want = attend_tree(*inputs, mask, pool, rows, config)
        assert torch.equal(attend_tree(*views, mask, pool, rows, config), want)
        apart = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in inputs]
        assert torch.equal(attend_tree(*apart, mask, pool, rows, config), want)
        odd = [torch.cat((x.flatten(), x.flatten()[:1]))[1:].view(x.shape) for x in inputs]
        tree_check(attend_tree(*odd, mask, pool, rows, config), odd, mask, pool, rows)
        shared = rows[:1].expand(3, -1)
        tree_check(attend_tree(*inputs, mask, pool, shared, config), inputs, mask, pool, shared)
        strided = rows.repeat_interleave(2, 1)[:, ::2]
        assert torch.equal(attend_tree(*inputs, mask, pool, strided, config), want)
        assert not flags()
        broken = rows.clone()
        broken[1, 50] = pool.shape[0] * 16
        broken[2, 3] = 1 << 60
        tree_check(attend_tree(*inputs, mask, pool, broken, config), inputs, mask, pool, broken)
        assert flags() == [_lib.DEVICE_FLAGS[1]]


def test_tree_rows_far_into_a_long_pool():
    """Rows of blocks whose elements lie past 2^31 (and bytes past 2^32) give what the
    same rows give at the start of a short pool, in runs and one by one."""
    from hisparse_b200 import CacheConfig, attend_tree, tree_mask

    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    for dtype, dim in ((BF16, 128), (FP16, 256), (FP32, 64)):
        inputs, parents, pool, rows, config = tree_inputs(2, 5, 8, 4, dim, 16, 200, dtype, 16)
        mask = tree_mask(parents, DEV)
        want = attend_tree(*inputs, mask, pool, rows, config)
        first = 2 ** 31 // pool[0].numel() + 11
        long_pool = torch.empty((first + pool.shape[0], *pool.shape[1:]), dtype=dtype, device=DEV)
        long_pool[first:] = pool
        far = CacheConfig(gpu_pages=long_pool.shape[0], page_size=16, kv_heads=4, head_dim=dim,
                          device=DEV, dtype=dtype)
        got = attend_tree(*inputs, mask, long_pool, rows + first * 16, far)
        assert torch.equal(got, want)
        mixed = torch.randperm(200, generator=torch.Generator().manual_seed(1)).to(DEV)
        want = attend_tree(*inputs, mask, pool, rows[:, mixed].contiguous(), config)
        got = attend_tree(*inputs, mask, long_pool, (rows + first * 16)[:, mixed].contiguous(), far)
        assert torch.equal(got, want)
        del long_pool
    assert not flags()


def test_tree_runs_equal_single_rows():
    """Rows in page order (tiled copies) and the same rows shuffled are the same set:
    equal within the bound of their sums."""
    from hisparse_b200 import attend_tree, tree_mask

    for dtype, dim in ((BF16, 128), (FP16, 64), (BF16, 256), (FP16, 192)):
        inputs, parents, pool, rows, config = tree_inputs(3, 40, 8, 2, dim, 64, 1000, dtype, 18)
        mask = tree_mask(parents, DEV)
        rows[1, 100:300] = -1
        rows[2, 5::7] = -1
        order = torch.randperm(1000, generator=torch.Generator().manual_seed(2)).to(DEV)
        for r in (rows, rows[:, order].contiguous(), rows[:, 3:].contiguous()):
            tree_check(attend_tree(*inputs, mask, pool, r, config), inputs, mask, pool, r)


def test_tree_peaked_scores():
    """Scores of +-400 (no overflow, weights down to zero) and equal scores."""
    from hisparse_b200 import attend_tree, tree_mask

    for dtype in (FP32, BF16):
        inputs, parents, pool, rows, config = tree_inputs(1, 9, 8, 2, 128, 16, 600, dtype, 14,
                                                          scale=60.0)
        mask = tree_mask(parents, DEV)
        tree_check(attend_tree(*inputs, mask, pool, rows, config), inputs, mask, pool, rows)
        inputs[0].zero_()
        tree_check(attend_tree(*inputs, mask, pool, rows, config), inputs, mask, pool, rows)


def test_tree_mask():
    from hisparse_b200 import tree_mask

    m = tree_mask([[-1, 0, 0, 2], [-1], [], list(range(-1, 63))], "cpu")
    assert m.shape == (4, 64)
    assert m[0, :5].tolist() == [1, 3, 5, 13, 0] and m[1].tolist() == [1] + [0] * 63
    assert m[2].count_nonzero() == 0 and m[3, 63].item() == -1 and m[3, 62].item() == 2 ** 63 - 1
    for bad in ([[0]], [[-1, 1]], [[-2]], [[-1] * 65]):
        with pytest.raises(ValueError):
            tree_mask(bad, "cpu")


def test_tree_refusals():
    from hisparse_b200 import attend_tree, tree_mask

    (q, k, v), parents, pool, rows, config = tree_inputs(2, 4, 8, 2, 32, 16, 40, FP32, 15)
    mask = tree_mask(parents, DEV)
    counts = torch.ones(2, dtype=torch.int32, device=DEV)
    with pytest.raises(ValueError, match="query must be"):
        attend_tree(q[0], k, v, mask, pool, rows, config)
    with pytest.raises(ValueError, match="GQA"):
        attend_tree(q[:, :, :7], k, v, mask, pool, rows, config)
    with pytest.raises(ValueError, match="key and value"):
        attend_tree(q, k[:, :3], v, mask, pool, rows, config)
    with pytest.raises(ValueError, match="one dtype"):
        attend_tree(q, k, v.half(), mask, pool, rows, config)
    with pytest.raises(ValueError, match="mask must be"):
        attend_tree(q, k, v, mask.int(), pool, rows, config)
    with pytest.raises(ValueError, match="mask must be"):
        attend_tree(q, k, v, mask[:1], pool, rows, config)
    with pytest.raises(ValueError, match="rows must be"):
        attend_tree(q, k, v, mask, pool, rows[0], config)
    with pytest.raises(ValueError, match="rows must be"):
        attend_tree(q, k, v, mask, pool, rows.int(), config)
    with pytest.raises(ValueError, match="pool must be"):
        attend_tree(q, k, v, mask, pool[:, :, :8], rows, config)
    with pytest.raises(ValueError, match="counts must be"):
        attend_tree(q, k, v, mask, pool, rows, config, counts=counts.long())
    with pytest.raises(ValueError, match="nodes must be"):
        attend_tree(q, k, v, mask, pool, rows, config, nodes=counts[:1])
    with pytest.raises(ValueError, match="at most 64"):
        wide = [x.repeat(1, 17, 1, 1) for x in (q, k, v)]
        attend_tree(*wide, mask.repeat(1, 17), pool, rows, config)
    with pytest.raises(ValueError, match="CUDA"):
        attend_tree(q, k, v, mask.cpu(), pool, rows, config)
    assert attend_tree(q[:0], k[:0], v[:0], mask[:0], pool, rows[:0], config).shape[0] == 0
    assert attend_tree(q[:, :0], k[:, :0], v[:, :0], mask[:, :0], pool, rows, config).numel() == 0


# ---- together: as a verification step uses them -------------------------------------------------
def _verify_inputs(dtype, seed):
    from hisparse_b200 import rope_frequencies, tree_mask

    batch, nodes, hq, hkv, dim, vocab = 3, 6, 8, 2, 64, 1003
    _, parents, pool, rows, config = tree_inputs(batch, nodes, hq, hkv, dim, 16, 200, dtype, seed)
    gen = torch.Generator().manual_seed(seed)
    fused = torch.randn(batch * nodes, (hq + 2 * hkv) * dim, generator=gen).to(dtype).to(DEV)
    head = (torch.randn(vocab, hq * dim, generator=gen) / 16).to(dtype).to(DEV)
    w = torch.ones(dim, dtype=dtype, device=DEV)
    positions = torch.randint(200, 300, (batch * nodes,), generator=gen).to(DEV)
    tokens = torch.randint(0, vocab, (batch * nodes, 2), generator=gen).to(DEV)
    return dict(fused=fused, head=head, w=w, positions=positions, tokens=tokens, pool=pool,
                rows=rows, config=config, mask=tree_mask(parents, DEV),
                freq=rope_frequencies(dim, 10000.0, DEV))


def _verify_step(s):
    from hisparse_b200 import attend_tree, qk_norm_rope, token_logprobs

    n, dim = s["fused"].shape[0], 64
    q, k, v = (x.view(n, -1, dim) for x in s["fused"].split((8 * dim, 2 * dim, 2 * dim), -1))
    q, k = qk_norm_rope(q, k, s["positions"], s["freq"], s["w"], s["w"])
    split = (3, 6)
    out = attend_tree(q.unflatten(0, split), k.unflatten(0, split), v.unflatten(0, split),
                      s["mask"], s["pool"], s["rows"], s["config"])
    logits = out.flatten(0, 1).flatten(1) @ s["head"].t()
    return (out, *token_logprobs(logits, s["tokens"], top=5)), (q, k, v, logits)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_operators_together(dtype):
    s = _verify_inputs(dtype, 21)
    (out, *scores), (q, k, v, logits) = _verify_step(s)
    fq, fk, fv = (x.view(18, -1, 64) for x in s["fused"].split((512, 128, 128), -1))
    norm_rope_check(q, fq, s["w"], s["positions"], s["freq"], 1e-6)
    norm_rope_check(k, fk, s["w"], s["positions"], s["freq"], 1e-6)
    inputs = [x.unflatten(0, (3, 6)) for x in (q, k, v)]
    tree_check(out, inputs, s["mask"], s["pool"], s["rows"])
    from hisparse_b200 import TokenLogprobs

    logprobs_check(TokenLogprobs(*scores), logits, s["tokens"], 5)


def test_operators_refuse_tensors_that_want_gradients():
    from hisparse_b200 import attend_tree, qk_norm_rope, token_logprobs

    s = _verify_inputs(FP32, 24)
    x = s["fused"].requires_grad_()
    with pytest.raises(ValueError, match="no backward"):
        _verify_step(s)
    with torch.no_grad():
        (out, *scores), (q, k, v, logits) = _verify_step(s)
    heads = [t.unflatten(0, (3, 6)) for t in (q, k, v.detach())]
    with pytest.raises(ValueError, match="no backward"):
        attend_tree(heads[0].requires_grad_(), *heads[1:], s["mask"], s["pool"], s["rows"],
                    s["config"])
    with pytest.raises(ValueError, match="no backward"):
        token_logprobs(logits.requires_grad_())
    with pytest.raises(ValueError, match="no backward"):
        qk_norm_rope(q.detach(), k.detach(), s["positions"], s["freq"],
                     s["w"].clone().requires_grad_(), s["w"])
    assert x.grad is None


def test_first_call_inside_a_capture(monkeypatch):
    """The device's status word is made outside graphs only: a first call inside one
    records no flags and works."""
    from hisparse_b200 import _lib, token_logprobs

    monkeypatch.setattr(_lib, "_status_words", {})
    monkeypatch.setattr(_lib, "_status_pointers", {})
    x = torch.randn(4, 100, device=DEV)
    tokens = torch.tensor([1, 2, 100, 3], device=DEV)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token_logprobs(x, tokens, top=2)
    graph.replay()
    assert _lib._status_words == {} and out.logprobs.isnan().tolist() == [False] * 2 + [True, False]
    want = token_logprobs(x, tokens, top=2)
    assert torch.equal(out.top_tokens, want.top_tokens)
    assert flags() == [_lib.DEVICE_FLAGS[64]]


def test_calls_on_two_streams_at_once():
    """Calls that overlap have workspaces of their own."""
    from hisparse_b200 import attend_tree, tree_mask

    cases = []
    for seed in (31, 32):
        inputs, parents, pool, rows, config = tree_inputs(2, 20, 8, 2, 128, 16, 4000, BF16, seed)
        cases.append((*inputs, tree_mask(parents, DEV), pool, rows, config))
    want = [attend_tree(*c) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(8):
        for i, (stream, case) in enumerate(zip(streams, cases)):
            with torch.cuda.stream(stream):
                got[i].append(attend_tree(*case))
    torch.cuda.synchronize()
    for outs, w in zip(got, want):
        assert all(torch.equal(o, w) for o in outs)


def test_operators_captured_and_on_another_stream():
    """A captured step replayed on new inputs, two captured steps replayed in turn,
    and a step on a side stream give the eager results bit for bit."""
    a, b = _verify_inputs(BF16, 22), _verify_inputs(BF16, 23)
    want_a, want_b = _verify_step(a)[0], _verify_step(b)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _verify_step(a)[0]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(got, want_a))
    graphs = []
    for s in (a, b):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = _verify_step(s)[0]
        graphs.append((graph, out))
    for _ in range(2):
        for graph, _ in graphs:
            graph.replay()
    for (_, out), want in zip(graphs, (want_a, want_b)):
        assert all(torch.equal(x, y) for x, y in zip(out, want))
    for name in ("fused", "pool", "rows", "positions", "tokens", "mask"):
        a[name].copy_(b[name])
    a["head"].copy_(b["head"])
    graphs[0][0].replay()
    assert all(torch.equal(x, y) for x, y in zip(graphs[0][1], want_b))
    again = _verify_step(b)[0]  # and the same call gives the same bits
    assert all(torch.equal(x, y) for x, y in zip(again, want_b))

"""Bounds for attention over a cache held in 8 bits that a missing row or a weight in fewer bits
exceeds, and inputs that make them tight: flat weights (every row counts alike) and sums that
nearly cancel (a result far below the terms it is made of shows their rounding)."""

from __future__ import annotations

import math

import numpy as np
import torch

import quantized_reference as ref

STEP = 2.0 ** -23  # of fp32
# What taking a query apart leaves of an element, as a share of the query's largest: each part
# leaves half a step, with the largest element at 2^7 or more and numbers below 2^-6 in steps
# of 2^-9. Part j works on 16^(j-1) of the rest, so n parts leave 2^-10 / 16^(n-1) / 2^7.
QUERY = {torch.bfloat16: 2.0 ** -21, torch.float16: 2.0 ** -25, torch.float32: 2.0 ** -37}


def smallest(dtype, group, dim):
    """What a weight loses besides its share, of the largest, which is kept at 2^7 or more. Its
    second fp16 number has steps of 2^-24, of which rounding loses half, and is kept times 2^11;
    with two quads of bf16 queries to a KV head it is kept as it is. (Weights stay in fp32
    where head_dim is no multiple of 16.)"""
    together = dtype == torch.bfloat16 and group > 4 and dim % 16 == 0
    return 2.0 ** -32 if together else 2.0 ** -43


def pool_of(blocks, page, heads, dim, seed, key_size=0.3, key_elements=None):
    """Records [blocks, 2, page, row_bytes]: V normal, K normal times key_size, zeros past its
    first key_elements."""
    rng = np.random.default_rng(seed)
    x = rng.standard_normal((blocks, 2, page, heads, dim))
    x[:, 0] *= key_size
    if key_elements is not None:
        x[:, 0, :, :, key_elements:] = 0
    return ref.records(x)


def attend(query, pool, rows, heads, dtype, counts=None):
    """float64 [B, Hq, D] of query [B, Hq, D] (float64, numbers of dtype) over rows [B, K] or
    [B, Hq, K], and how far a result of `dtype` may be from it.

    Scores: n products that are not zero and their scaling, each off by at most a step of
    fp32 of the sum of their sizes, 16 more for the parts' sums and factors, and what taking
    the query apart leaves. In powers of two, scores go through five roundings (in the
    numerator and in the sum) with the V exponent and the lift added. That changes a weight by its
    share, in the numerator and in the sum (twice). The power itself, the factors of a moved
    maximum and of a join, the weight as two fp16 numbers: 2^-20 together. Sums of n rows: a
    step each. What is small against a weight's second number counts with the codes of its
    row, up to 448 where the largest weight's row has at least 224: twice `smallest` of the
    largest element's sum of |v|. Then the result's own rounding."""
    b, hq, d = query.shape
    info = torch.finfo(dtype)
    out, bound = np.zeros(query.shape), np.zeros(query.shape)
    for i in range(b):
        for h in range(hq):
            at = rows[i] if rows.ndim == 2 else rows[i, h]
            at = at[:len(at) if counts is None else max(0, int(counts[i]))]
            at = at[(at >= 0) & (at < pool.shape[0] * pool.shape[2])]
            if not len(at):
                continue
            kh = h // (hq // heads)
            records = ref.row_records(pool, at, 1)
            k = ref.values(ref.row_records(pool, at, 0), heads, d)[:, kh]
            v = ref.values(records, heads, d)[:, kh]
            q, size = query[i, h], np.abs(k) @ np.abs(query[i, h]) / math.sqrt(d)
            s = k @ q / math.sqrt(d)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], spread = w @ v, w @ np.abs(v)
            n = np.count_nonzero(np.any(k != 0, axis=0))
            score = (n + 16) * STEP * size.max() + \
                QUERY[dtype] * np.abs(q).max() * np.abs(k).sum(1).max() / math.sqrt(d)
            exponents = records[:, heads * d + kh].astype(int) - 127
            number = np.abs(s).max() * 1.4427 + np.abs(exponents).max() + 32
            share = 2 * score + 5 * STEP / 2 * number + 2.0 ** -20 + (len(at) + 8) * STEP
            error = share * spread + 2 * smallest(dtype, hq // heads, d) * len(at) * spread.max() + 2.0 ** -126
            bound[i, h] = error + info.eps / 2 * (np.abs(out[i, h]) + error) + \
                info.smallest_normal * info.eps / 2
    return out, bound


def cancel(query, pool, rows, heads, head):
    """Writes the V rows of the last four of rows [K] so that the result of query head `head`
    of each KV head's group nearly cancels: each takes what the rows before it sum to, which
    leaves 2^-4 of it. Returns those heads of query [Hq, D]."""
    hq, d = query.shape
    out = []
    values = ref.values(ref.row_records(pool, rows, 1), heads, d)
    keys = ref.values(ref.row_records(pool, rows, 0), heads, d)
    for kh in range(heads):
        out.append(kh * (hq // heads) + head)
        s = keys[:, kh] @ query[out[-1]] / math.sqrt(d)
        w = np.exp(s - s.max())
        rest = w[:-4] @ values[:-4, kh]
        for i in range(len(rows) - 4, len(rows)):
            held = ref.values(ref.records(-rest[None, None] / w[i]), 1, d)[0, 0]
            values[i, kh] = held
            rest = rest + w[i] * held
    at = rows[-4:]
    pool[at // pool.shape[2], 1, at % pool.shape[2]] = ref.records(values[-4:])
    return out

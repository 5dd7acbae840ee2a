"""Plain 64-bit forms of a cache held in 8 bits, for the tests: the formulas of
include/hisparse_quantized.h over numpy arrays, written without the library."""

from __future__ import annotations

import math

import numpy as np
import torch

LOWEST = -100
# the numbers that the bytes stand for: 4 bits of exponent (bias 7), 3 of fraction
NUMBERS = np.array([math.nan if i & 127 == 127 else (-1.0 if i >> 7 else 1.0) * (
    math.ldexp(8 + (i & 7), (i >> 3 & 15) - 10) if i >> 3 & 15 else math.ldexp(i & 7, -9))
    for i in range(256)])
_BETWEEN = (NUMBERS[:126] + NUMBERS[1:127]) / 2  # halfway between neighbouring numbers


def encode(x):
    """Bytes of the e4m3 numbers nearest to x (float64, |x| <= 448 or not finite)."""
    size = np.abs(x)
    finite = np.isfinite(x)
    safe = np.where(finite, size, 0.0)
    index = np.searchsorted(_BETWEEN, safe, side="left")  # the lower one of a tie
    tie = (index < 126) & (safe == _BETWEEN[np.minimum(index, 125)]) & (index % 2 == 1)
    code = (index + tie) | (np.signbit(x).astype(np.int64) << 7)
    return np.where(finite, code, 127).astype(np.uint8)


def exponent(x):
    """Exponent of the scale of a head's elements x [..., D]."""
    largest = np.where(np.isfinite(x), np.abs(x), 0.0).max(-1)
    out = np.full(largest.shape, LOWEST, dtype=np.int64)
    for at in np.ndindex(largest.shape):
        e = LOWEST
        while largest[at] > math.ldexp(448.0, e):
            e += 1
        out[at] = e
    return out


def row_bytes(heads, dim):
    n = heads * (dim + 1)
    return n + -n % 32


def records(x):
    """uint8 [..., record] of float64 x [..., heads, D]."""
    *lead, heads, dim = x.shape
    e = exponent(x)
    out = np.zeros((*lead, row_bytes(heads, dim)), dtype=np.uint8)
    out[..., :heads * dim] = encode(x * np.exp2(-e.astype(float))[..., None]).reshape(*lead, heads * dim)
    out[..., heads * dim:heads * (dim + 1)] = e + 127
    return out


def values(record, heads, dim):
    """float64 [..., heads, D] that records [..., record] hold."""
    codes = NUMBERS[record[..., :heads * dim]].reshape(*record.shape[:-1], heads, dim)
    e = record[..., heads * dim:heads * (dim + 1)].astype(float) - 127
    return codes * np.exp2(e)[..., None]


def row_records(pool, rows, plane):
    """Records of physical rows (>= 0) of a pool [blocks, 2, P, record]."""
    p = pool.shape[2]
    return pool[rows // p, plane, rows % p]


def attend(query, pool, rows, heads, counts=None):
    """float64 [B, Hq, D] and, for its tolerance, the weighted sum of |v| and the
    largest sum of |q_d k_d| / sqrt(D) of every query. rows [B, K] or [B, Hq, K]."""
    b, hq, d = query.shape
    out, spread, size = np.zeros(query.shape), np.zeros(query.shape), np.zeros((b, hq, 1))
    for i in range(b):
        for h in range(hq):
            at = rows[i] if rows.ndim == 2 else rows[i, h]
            at = at[:len(at) if counts is None else max(0, int(counts[i]))]
            at = at[(at >= 0) & (at < pool.shape[0] * pool.shape[2])]
            if not len(at):
                continue
            kh = h // (hq // heads)
            k = values(row_records(pool, at, 0), heads, d)[:, kh]
            v = values(row_records(pool, at, 1), heads, d)[:, kh]
            s = k @ query[i, h] / math.sqrt(d)
            w = np.exp(s - s.max())
            w /= w.sum()
            out[i, h], spread[i, h] = w @ v, w @ np.abs(v)
            size[i, h] = (np.abs(k) @ np.abs(query[i, h])).max() / math.sqrt(d)
    return out, spread, size


def attend_tolerance(out, spread, size, dim, rows, dtype):
    """How far attention may be from `out`: a score of dim products and the scaling is off
    by at most (dim + 4) half steps of fp32 times the sum of its products' sizes, which
    changes a weight by that share, in the numerator and in the sum (so twice); a weight's
    power by 2^-21; sums of `rows` weights by that many steps (tensor cores may cut
    instead of rounding: whole steps). 16-bit queries: weights are rounded to fp16 for the
    second product, by half a step or, near zero, by 2^-25 of the largest (2^8 at most).
    fp32 queries: a weight is two fp16 numbers, whose rounding is part of the 2^-20 but for
    their smallest step, 2^-24, so half of that, 2^-25. The largest weight is kept at 2^7 or
    more, so this is 2^-32 of it; with codes up to 448 in the other rows and at least 224
    in its own row's largest element, each row adds at most 2^-32 * 448 / 224 = 2^-31 of the
    largest element's sum of |v| to any element, one with a far smaller sum among them.
    The result's own rounding is half a step of its type, and half the distance of its
    subnormal numbers (finfo's smallest normal times eps) where it is below the normal ones."""
    info = torch.finfo(dtype)
    step = 2.0 ** -23
    share = 2 * (dim + 4) * step * size + 2.0 ** -20 + (rows + 8) * step
    if dtype != torch.float32:
        share = share + 2.0 ** -11
    if dtype == torch.float32:
        absolute = 2.0 ** -31 * rows * spread.max(axis=-1, keepdims=True) + 2.0 ** -126
    else:
        absolute = 2.0 ** -25 * 2.0 ** 8 * rows * np.abs(spread).max(initial=0.0) + 2.0 ** -126
    absolute += info.smallest_normal * info.eps / 2
    return share * spread + absolute + info.eps / 2 * (np.abs(out) + share * spread)

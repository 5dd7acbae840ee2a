"""Operators of a cache held in 8 bits: what is measured, and their plain forms.

A cache whose rows are held in 8 bits moves half the bytes over the host link
and out of HBM. Every token's K (and V) of a KV head is held as e4m3 codes with
a power-of-two scale of its own, so that a row can move alone. Three operators
serve such a cache: rows are quantised as they are written, with their page's
bounds and mean (``append_quantized``), read back (``read_quantized``), and
attended to by decode queries (``attend_quantized``).

A row's record, for K and for V: kv_heads * head_dim codes, one byte a KV head
for the scale's exponent (plus 127), zeros up to a multiple of 32 bytes. The
exponent is the smallest e with |x| <= 448 * 2^e for every finite element x of
the head, and at least -100; a code is x * 2^-e rounded to e4m3.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import torch

own = False

_PACKAGE = str(Path(__file__).resolve().parent.parent / "nano-hisparse_b200")
_TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}
_DEVICE = "cuda:0"
_LOWEST = -100  # exponent of the smallest scale


# ---- the cases ---------------------------------------------------------------------------
def _append(name, chunks, tokens, last, within, kv_heads, head_dim, page_size, dtype):
    return {"name": name, "op": "append", "chunks": chunks, "tokens": tokens, "last": last,
            "within": within, "kv_heads": kv_heads, "head_dim": head_dim,
            "page_size": page_size, "dtype": dtype}


def _read(name, rows, kv_heads, head_dim, page_size, dtype, holes):
    return {"name": name, "op": "read", "rows": rows, "kv_heads": kv_heads,
            "head_dim": head_dim, "page_size": page_size, "dtype": dtype, "holes": holes}


def _attend(name, batch, rows, q_heads, kv_heads, head_dim, page_size, dtype, holes):
    return {"name": name, "op": "attend", "batch": batch, "rows": rows, "q_heads": q_heads,
            "kv_heads": kv_heads, "head_dim": head_dim, "page_size": page_size, "dtype": dtype,
            "holes": holes}


def listed():
    return [
        # a decode step of the small fp32 decoder: one row of three requests
        _append("append_step_3", 3, 1, 1, 5, 2, 32, 16, "float32"),
        # a decode step of 16 requests in bf16, pages nearly full
        _append("append_step_16", 16, 1, 1, 13, 8, 128, 16, "bfloat16"),
        # an odd prompt in pages of 64, the last page short, fp16
        _append("append_prompt_4099", 65, 64, 3, 0, 4, 128, 64, "float16"),
        # a whole 32k prompt
        _append("append_prompt_32768", 2048, 16, 16, 0, 8, 128, 16, "bfloat16"),
        # a few rows of the small fp32 decoder, some of them masked
        _read("read_small_24", 24, 2, 32, 16, "float32", True),
        # an 8,192-row budget of one long request in pages of 64
        _read("read_long_8192", 8192, 4, 128, 64, "float16", False),
        # the full history of 8 requests at 32k
        _read("read_full_262144", 262144, 8, 128, 16, "bfloat16", False),
        # the small fp32 decoder: three requests, 160 rows
        _attend("attend_small_fp32", 3, 160, 8, 2, 32, 16, "float32", True),
        # 16 requests with the 2,048-row Quest budget
        _attend("attend_budget_2048", 16, 2048, 32, 8, 128, 16, "bfloat16", False),
        # one long request with the 8,192-row budget in pages of 64 (28/4 heads)
        _attend("attend_long_8192", 1, 8192, 28, 4, 128, 64, "bfloat16", False),
        # heads that share nothing, an odd history, masked rows, fp16
        _attend("attend_heads_5003", 7, 5003, 16, 16, 64, 16, "float16", True),
        # the full history of 16 requests at 32k
        _attend("attend_full_32768", 16, 32768, 32, 8, 128, 16, "bfloat16", False),
    ]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


_HEADS = [(8, 2, 32), (32, 8, 128), (28, 4, 128), (16, 16, 64), (10, 2, 80), (12, 1, 256)]


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend"])
    dtype = rng.choice(["float32", "float16", "bfloat16", "bfloat16"])
    hq, hkv, d = rng.choice(_HEADS)
    page = rng.choice([16, 64, 12])
    if op == "append":
        if rng.random() < 0.5:  # a decode step, or a piece of up to a few tokens
            tokens = rng.choice([1, 1, 2, 5])
            case = _append("", _spread(rng, 1, 256), tokens, rng.randint(1, tokens),
                           rng.randint(0, page - tokens), hkv, d, page, dtype)
        else:  # a prompt's pages
            limit = 32768 * 8 * 128 // (page * hkv * d * (2 if dtype == "float32" else 1))
            case = _append("", _spread(rng, 1, min(2048, limit)), page, rng.randint(1, page), 0,
                           hkv, d, page, dtype)
    elif op == "read":
        limit = 262144 * 8 * 128 // (hkv * d * (2 if dtype == "float32" else 1))
        case = _read("", _spread(rng, 1, min(262144, limit)), hkv, d, page, dtype,
                     rng.random() < 0.3)
    else:
        batch = _spread(rng, 1, 64)
        # at most the largest listed case's rows and products, an eighth of them in fp32
        limit = 16 * 32768 * 32 * 128 // (batch * max(hq, 4 * hkv) * d)
        limit = limit // 8 if dtype == "float32" else limit
        case = _attend("", batch, _spread(rng, 1, max(1, min(32768, limit))), hq, hkv, d, page,
                       dtype, rng.random() < 0.3)
    del case["name"]
    return case


# ---- ragged sizes, from the case alone ----------------------------------------------------
def _row_counts(case):
    """Rows each request attends to: the longest first, the shortest three quarters of
    it; with holes the last of several requests has none."""
    b, n = case["batch"], case["rows"]
    counts = [n - i * n // (4 * b) for i in range(b)]
    if case["holes"] and b > 1:
        counts[-1] = 0
    return counts


def _token_counts(case):
    """Rows each chunk appends: all but the last are full."""
    return [case["tokens"]] * (case["chunks"] - 1) + [case["last"]]


def _holes(case):
    """Columns of masked rows: every thirteenth."""
    return slice(4, None, 13) if case["holes"] else slice(0, 0)


def _record(case):
    heads, dim = case["kv_heads"], case["head_dim"]
    return -(-heads * (dim + 1) // 32) * 32


# ---- inputs -------------------------------------------------------------------------------
def _rows_like(gen, shape, dtype):
    """K or V [..., kv_heads, head_dim]: normal values, a few channels much larger."""
    x = torch.empty(shape, dtype=torch.float32, device=_DEVICE).normal_(generator=gen)
    gain = torch.empty(shape[-2:], device=_DEVICE).normal_(generator=gen).mul_(0.7).exp_()
    return x.mul_(gain).to(dtype)


def _filled_pool(case, blocks, gen):
    """A pool whose every row has been written, [blocks, 2, page_size, record] bytes."""
    p, heads, dim = case["page_size"], case["kv_heads"], case["head_dim"]
    pool = torch.empty((blocks, 2, p, _record(case)), dtype=torch.uint8, device=_DEVICE)
    step = max(1, (1 << 26) // (2 * p * heads * dim))
    for first in range(0, blocks, step):
        n = min(step, blocks - first)
        pool[first:first + n] = _quantise(_rows_like(gen, (n, 2, p, heads, dim), torch.float32))
    return pool


def _placed_rows(case, pages, blocks, gen):
    """Physical rows of `pages` pages [pages, page_size]: three quarters of the pages lie
    whole in the pool, the rows of the others each at a place of its own."""
    p = case["page_size"]
    order = torch.randperm(blocks, generator=gen, device=_DEVICE)[:pages]
    rows = order[:, None] * p + torch.arange(p, device=_DEVICE)
    loose = rows[-(-3 * pages // 4):]
    mixed = loose.reshape(-1)[torch.randperm(loose.numel(), generator=gen, device=_DEVICE)]
    rows[-(-3 * pages // 4):] = mixed.view(loose.shape)
    return rows


def prepare(case, seed):
    if own and _PACKAGE not in sys.path:
        sys.path.insert(0, _PACKAGE)
    gen = torch.Generator(device=_DEVICE).manual_seed(seed)
    dtype = _TYPES[case["dtype"]]
    p, heads, dim = case["page_size"], case["kv_heads"], case["head_dim"]
    state = {"case": case}
    if case["op"] == "append":
        n = case["chunks"]
        blocks = n + 3
        counts = _token_counts(case)
        state["pool"] = _filled_pool(case, blocks, gen)
        state["block"] = torch.randperm(blocks, generator=gen, device=_DEVICE)[:n].contiguous()
        state["k"] = _rows_like(gen, (n, case["tokens"], heads, dim), dtype)
        state["v"] = _rows_like(gen, (n, case["tokens"], heads, dim), dtype)
        state["within"] = torch.full((n,), case["within"], dtype=torch.int32, device=_DEVICE)
        state["count"] = torch.tensor(counts, dtype=torch.int32, device=_DEVICE)
        # the bounds of the page's earlier rows (none: an empty page's)
        held = _read_back(state["pool"][state["block"], 0], case)[:, :case["within"]]
        empty = torch.full((n, 1, heads, dim), math.inf, device=_DEVICE)
        state["minimum"] = torch.cat((held, empty), 1).amin(1).to(torch.bfloat16)
        state["maximum"] = torch.cat((held, -empty), 1).amax(1).to(torch.bfloat16)
        state["summary"] = torch.zeros((n, heads, dim), device=_DEVICE)
        for name in ("minimum", "maximum", "summary"):  # addresses of the pages' entries
            t = state[name]
            state[name + "_ptrs"] = t.data_ptr() + torch.arange(n, device=_DEVICE) * (
                heads * dim * t.element_size())
    elif case["op"] == "read":
        n = case["rows"]
        pages = -(-n // p)
        blocks = pages + 5
        state["pool"] = _filled_pool(case, blocks, gen)
        rows = _placed_rows(case, pages, blocks, gen).reshape(-1)[:n].contiguous()
        rows[_holes(case)] = -1
        state["rows"] = rows
    else:
        b, hq, width = case["batch"], case["q_heads"], case["rows"]
        pages = -(-width // p)
        blocks = b * pages + 7
        state["pool"] = _filled_pool(case, blocks, gen)
        rows = _placed_rows(case, b * pages, blocks, gen).view(pages, b, p)
        rows = rows.transpose(0, 1).reshape(b, pages * p)[:, :width].contiguous()
        counts = torch.tensor(_row_counts(case), dtype=torch.int32, device=_DEVICE)
        rows[torch.arange(width, device=_DEVICE)[None, :] >= counts[:, None]] = -1
        rows[:, _holes(case)] = -1
        state["rows"], state["counts"] = rows, counts
        # the queries in one fused projection's output
        fused = torch.empty((b, (hq + 2 * heads) * dim), dtype=dtype, device=_DEVICE)
        fused.normal_(generator=gen)
        state["query"] = fused[:, :hq * dim].unflatten(-1, (hq, dim))
    if own:
        from hisparse_b200 import CacheConfig

        state["config"] = CacheConfig(gpu_pages=blocks, page_size=p, kv_heads=heads,
                                      head_dim=dim, device=_DEVICE, dtype=torch.float8_e4m3fn)
    return state


# ---- one pass -----------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if op == "append":
        if own:
            import hisparse_b200 as hs

            hs.append_quantized(state["k"], state["v"], state["within"], state["count"],
                                state["block"], state["pool"], state["minimum_ptrs"],
                                state["maximum_ptrs"], state["summary_ptrs"], state["config"])
        else:
            _plain_append(state)
        # the codes as the e4m3 numbers that they are, and the scales' exponents
        codes = state["case"]["kv_heads"] * state["case"]["head_dim"]
        pool = state["pool"]
        return (pool[..., :codes].view(torch.float8_e4m3fn), pool[..., codes:],
                state["minimum"], state["maximum"], state["summary"])
    if own:
        import hisparse_b200 as hs

        if op == "read":
            return hs.read_quantized(state["pool"], state["rows"], state["config"],
                                     _TYPES[state["case"]["dtype"]])
        return hs.attend_quantized(state["query"], state["pool"], state["rows"],
                                   state["config"], counts=state["counts"])
    return _plain_read(state) if op == "read" else _plain_attend(state)


def _power(exponent):
    """2^exponent in fp32, for whole exponents from -126 to 127."""
    return ((exponent + 127) << 23).view(torch.float32)


def _quantise(x):
    """fp32 [..., kv_heads, head_dim] as records [..., record]."""
    *lead, heads, dim = x.shape
    finite = torch.isfinite(x)
    largest = torch.where(finite, x, torch.zeros_like(x)).abs().amax(-1)
    fraction, exponent = torch.frexp(largest)  # 448 is 0.875 * 2^9
    exponent = (exponent - 9 + (fraction > 0.875).int()).clamp(min=_LOWEST)
    exponent = torch.where(largest > 0, exponent, torch.full_like(exponent, _LOWEST))
    codes = torch.where(finite, x * _power(-exponent)[..., None], math.nan)
    codes = codes.to(torch.float8_e4m3fn).view(torch.uint8)
    record = torch.zeros((*lead, -(-heads * (dim + 1) // 32) * 32), dtype=torch.uint8,
                         device=x.device)
    record[..., :heads * dim] = codes.reshape(*lead, heads * dim)
    record[..., heads * dim:heads * (dim + 1)] = (exponent + 127).to(torch.uint8)
    return record


def _read_back(records, case):
    """fp32 [..., kv_heads, head_dim] of records [..., record]."""
    heads, dim = case["kv_heads"], case["head_dim"]
    codes = records[..., :heads * dim].contiguous().view(torch.float8_e4m3fn).float()
    scale = _power(records[..., heads * dim:heads * (dim + 1)].int() - 127)
    return codes.unflatten(-1, (heads, dim)).mul_(scale[..., None])


def _plain_append(state):
    case, pool, block = state["case"], state["pool"], state["block"]
    p, tokens = case["page_size"], case["tokens"]
    row = torch.arange(p, device=pool.device)
    first, count = state["within"][:, None], state["count"][:, None]
    new = (row >= first) & (row < first + count)
    token = (row - first).clamp(0, tokens - 1).long()  # the new row that a page's row takes
    chunk = torch.arange(case["chunks"], device=pool.device)[:, None]
    for plane, x in enumerate((state["k"], state["v"])):
        records = _quantise(x.float())
        page = pool[block, plane]
        pool[block, plane] = torch.where(new[..., None], records[chunk, token], page)
    keys = _read_back(pool[block, 0], case)
    outside = ~new[:, :, None, None]
    low = keys.masked_fill(outside, math.inf).amin(1)
    high = keys.masked_fill(outside, -math.inf).amax(1)
    state["minimum"].copy_(torch.minimum(state["minimum"].float(), low))
    state["maximum"].copy_(torch.maximum(state["maximum"].float(), high))
    valid = (row < first + count)[:, :, None, None]
    total = torch.where(valid, keys, torch.zeros_like(keys)).sum(1)
    state["summary"].copy_(total / (first + count)[:, :, None])


def _plain_read(state):
    case, pool, rows = state["case"], state["pool"], state["rows"]
    p = case["page_size"]
    at = rows.clamp(min=0)
    out = torch.empty((2, rows.shape[0], case["kv_heads"], case["head_dim"]),
                      dtype=_TYPES[case["dtype"]], device=pool.device)
    for plane in range(2):
        x = _read_back(pool[at // p, plane, at % p], case)
        out[plane] = torch.where((rows >= 0)[:, None, None], x, torch.zeros_like(x))
    return out


def _plain_attend(state):
    case, pool, rows, query = state["case"], state["pool"], state["rows"], state["query"]
    b, hq, d = query.shape
    p, hkv = case["page_size"], case["kv_heads"]
    width = rows.shape[1]
    column = torch.arange(width, device=rows.device)
    valid = ((rows >= 0) & (column[None, :] < state["counts"][:, None]))[:, None, None, :]
    at = rows.clamp(min=0)
    block, within = at // p, at % p
    q = query.float().view(b, hkv, hq // hkv, d)
    keys = _read_back(pool[block, 0, within], case)              # [b, width, hkv, d]
    scores = torch.matmul(q, keys.permute(0, 2, 3, 1)) / math.sqrt(d)
    del keys
    scores = scores.masked_fill(~valid, -math.inf)
    largest = scores.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    weights = torch.exp(scores - largest)
    total = weights.sum(-1, keepdim=True)
    values = _read_back(pool[block, 1, within], case)
    values = torch.where(valid[:, 0, 0, :, None, None], values, torch.zeros_like(values))
    out = torch.matmul(weights, values.permute(0, 2, 1, 3)) / total.clamp(min=1e-30)
    return out.view(b, hq, d).to(query.dtype)


# ---- the definitions in 64 bits -----------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "append":
        return _exact_append(state)
    if case["op"] == "read":
        keys, values = _exact_rows(state["pool"], state["rows"], case)
        return torch.stack((keys, values))
    return _exact_attend(state)


def _two_to(exponent):
    """2^exponent in 64 bits (a power function may be off in the last bit)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _e4m3_numbers():
    """The number that each byte stands for: 4 bits of exponent (bias 7), 3 of fraction."""
    byte = torch.arange(256, device=_DEVICE)
    sign = 1.0 - 2.0 * (byte >> 7).double()
    power, fraction = (byte >> 3) & 15, (byte & 7).double() / 8
    size = torch.where(power > 0, _two_to(power - 7) * (1 + fraction),
                       fraction / 64)
    size[127::128] = math.nan
    return sign * size


def _exact_rows(pool, rows, case):
    """K and V of physical rows in 64 bits, zeros where the row is negative."""
    p, heads, dim = case["page_size"], case["kv_heads"], case["head_dim"]
    numbers, out = _e4m3_numbers(), []
    flat = pool.view(-1, pool.shape[-1])
    for plane in range(2):
        record = flat[(rows.clamp(min=0) // p * 2 + plane) * p + rows.clamp(min=0) % p]
        codes = numbers[record[..., :heads * dim].int()].unflatten(-1, (heads, dim))
        scale = _two_to(record[..., heads * dim:heads * (dim + 1)].long() - 127)
        out.append(codes * scale[..., None] * (rows >= 0)[..., None, None])
    return out


def _exact_append(state):
    case, pool = state["case"], state["pool"]
    p, heads, dim, w = (case[k] for k in ("page_size", "kv_heads", "head_dim", "within"))
    n, width = case["chunks"], case["kv_heads"] * case["head_dim"]
    numbers = _e4m3_numbers()
    codes, tail = numbers[pool[..., :width].int()], pool[..., width:].long()
    held = torch.zeros((n, p, heads, dim), dtype=torch.float64, device=pool.device)
    held[:, :w] = (codes[state["block"], 0].unflatten(-1, (heads, dim)) * _two_to(
        tail[state["block"], 0, :, :heads] - 127)[..., None])[:, :w]
    count = state["count"].long()
    for plane, x in enumerate((state["k"].double(), state["v"].double())):
        size = x.abs().amax(-1)
        e = torch.ceil(torch.log2(size.clamp(min=1e-200) / 448.0))
        e = torch.where(size <= 448.0 * _two_to(e - 1), e - 1, e)  # log2 near a border
        e = torch.where(size > 448.0 * _two_to(e), e + 1, e).clamp(min=_LOWEST)
        scaled = x / _two_to(e)[..., None]
        # the distance of neighbouring codes: 2^-3 of the power of two below, at least 2^-9
        step = _two_to(torch.frexp(scaled).exponent - 4).clamp(min=2.0 ** -9)
        rounded = torch.round(scaled / step) * step
        for t in range(case["tokens"]):
            some = torch.nonzero(count > t)[:, 0]
            to = state["block"][some]
            codes[to, plane, w + t] = rounded[some, t].flatten(1)
            tail[to, plane, w + t] = 0
            tail[to, plane, w + t, :heads] = (e[some, t] + 127).long()
            if plane == 0:
                held[some, w + t] = rounded[some, t] * _two_to(e[some, t])[..., None]
    total, low, high = held[:, 0] * 0, state["minimum"].double(), state["maximum"].double()
    for r in range(p):
        inside = (r < w + count)[:, None, None]
        total = total + held[:, r] * inside
        if r >= w:
            low = torch.where(inside & (held[:, r] < low), held[:, r], low)
            high = torch.where(inside & (held[:, r] > high), held[:, r], high)
    return codes, tail, low, high, total / (w + count)[:, None, None]


def _exact_attend(state):
    case, query = state["case"], state["query"]
    group = case["q_heads"] // case["kv_heads"]
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    for b, count in enumerate(_row_counts(case)):
        rows = state["rows"][b, :count]
        rows = rows[rows >= 0]
        if not len(rows):
            continue
        keys, values = _exact_rows(state["pool"], rows, case)
        for h in range(case["kv_heads"]):
            q = query[b, h * group:(h + 1) * group].double()
            probabilities = torch.softmax(q @ keys[:, h].T / case["head_dim"] ** 0.5, -1)
            out[b, h * group:(h + 1) * group] = probabilities @ values[:, h]
    return out


# ---- what a pass cannot do without ---------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    heads, dim = case["kv_heads"], case["head_dim"]
    row = 2 * heads * (dim + 1)  # K and V as they are held
    if case["op"] == "append":
        n, tokens = case["chunks"], sum(_token_counts(case))
        moved = tokens * (2 * heads * dim * size + row) + n * case["within"] * (row // 2)
        # bounds read and written, the mean written, the chunk's places and addresses
        moved += n * (heads * dim * (2 * 4 + 4) + 40)
        return {"bytes": moved, "flops": 8 * tokens * heads * dim}
    if case["op"] == "read":
        rows = case["rows"] - len(range(case["rows"])[_holes(case)])
        moved = rows * row + case["rows"] * (8 + 2 * heads * dim * size)
        return {"bytes": moved, "flops": 2 * rows * heads * dim}
    counts = [n - len(range(n)[_holes(case)]) for n in _row_counts(case)]
    moved = sum(counts) * row + sum(_row_counts(case)) * 8
    moved += case["batch"] * (2 * case["q_heads"] * dim * size + 4)
    return {"bytes": moved, "flops": 4 * sum(counts) * case["q_heads"] * dim}

"""The work that the attention operators are measured on.

Four operators serve a stack's attention layers:

* ``prompt``   causal attention over packed prompts of different lengths, with
               grouped heads (``prompt_attention``);
* ``tables``   the page tables and token slots of a step, from the requests'
               lengths and new tokens (``extend_page_tables``);
* ``write``    keys and values into a paged cache in 8 bits, with a scale for
               each page and head (``write_kv_cache``);
* ``cached``   attention of each request's newest tokens over that cache
               (``cached_attention``).

The cache: codes are float8 (e4m3), a page's scale is a power of two.  A page
holds ``page`` tokens: keys as [pages, heads, page, padded width], values
transposed, [pages, heads, padded width, page]; scales are [pages, heads].

Sizes are those of the repository's configurations (64 requests, prefixes of
up to 2,048 tokens and 512 decode steps, width 128 over 4 heads) and generic
ones of serving.  ``own`` says whether ``run`` takes the framework's kernels
or the plain form, elementary torch operations in 32 bits.
"""

from __future__ import annotations

import math
import random

import numpy as np
import torch

DEVICE = "cuda"
FLOATS = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
CODES = torch.float8_e4m3fn
MOST_CODE = 448.0
WIDTHS = (32, 64, 96, 128, 192, 256)

own = False


# ------------------------------------------------------------------- cases


def listed():
    return [
        # a token each of 64 decoding requests: the smallest call, once a token
        dict(name="tables-decode", kind="tables", batch=64, page=64, longest=2560, most=1),
        # a large cohort admitted at once, small pages
        dict(name="tables-admit", kind="tables", batch=512, page=16, longest=2048, most=2048),
        # the decode write of one layer: a token each of 64 requests, pages partly filled
        dict(name="write-token", kind="write", batch=64, heads=8, width=128, page=64,
             floats="bfloat16", longest=2560, most=1),
        # a cohort's prompts into empty pages
        dict(name="write-prompts", kind="write", batch=48, heads=8, width=128, page=64,
             floats="bfloat16", longest=0, most=2048),
        # a small cohort of the repository's own width, 4 heads of 32: latency
        dict(name="prompt-b4-t128", kind="prompt", batch=4, longest=128, spread="equal",
             heads=4, kv_heads=4, width=32, floats="float32"),
        # prompts of 0 to 2,048 tokens packed into one call, grouped heads
        dict(name="prompt-packed", kind="prompt", batch=24, longest=2048, spread="ragged",
             heads=32, kv_heads=8, width=128, floats="bfloat16"),
        # two long prompts: the largest call
        dict(name="prompt-long", kind="prompt", batch=2, longest=8192, spread="equal",
             heads=32, kv_heads=8, width=128, floats="bfloat16"),
        # a smaller model in float16: three query heads a key head, an odd longest length
        dict(name="prompt-f16-w64", kind="prompt", batch=8, longest=1111, spread="ragged",
             heads=12, kv_heads=4, width=64, floats="float16"),
        # one short request of the repository's own width: latency
        dict(name="cached-one", kind="cached", batch=1, tokens=1, longest=300, heads=4,
             kv_heads=4, width=32, page=64, floats="float32"),
        # the decode batch: 64 requests somewhere between prefix and capacity
        dict(name="cached-b64", kind="cached", batch=64, tokens=1, longest=2560, heads=32,
             kv_heads=8, width=128, page=64, floats="bfloat16"),
        # two very long contexts: few rows, the long axis has to be split
        dict(name="cached-long", kind="cached", batch=2, tokens=1, longest=131072, heads=32,
             kv_heads=8, width=128, page=64, floats="bfloat16"),
        # drafted tokens checked at once: 4 query tokens a request, smaller pages
        dict(name="cached-draft", kind="cached", batch=16, tokens=4, longest=4096, heads=16,
             kv_heads=2, width=64, page=32, floats="float16"),
    ]


def _log_int(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["tables", "write", "prompt", "prompt", "cached", "cached"])
    page = rng.choice([16, 32, 64, 64, 128])
    floats = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    width = rng.choice([32, 40, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 3, 4, 8])
    if kind == "tables":
        batch = _log_int(rng, 1, 1024)
        return dict(kind=kind, batch=batch, page=page, longest=_log_int(rng, 16, 8192),
                    most=_log_int(rng, 1, min(4096, (1 << 20) // batch)))
    if kind == "write":
        batch = _log_int(rng, 1, 64)
        return dict(kind=kind, batch=batch, heads=kv_heads, width=width, page=page,
                    floats=floats, longest=rng.choice([0, _log_int(rng, 1, 1024)]),
                    most=_log_int(rng, 1, 32768 // batch))
    if kind == "prompt":
        batch = _log_int(rng, 1, 64)
        heads = min(heads, 32 if floats != "float32" else 16)
        heads -= heads % kv_heads
        most = math.sqrt((2 * 8192 ** 2 * 32 * 128) / (batch * heads * width))
        most /= 3 if floats == "float32" else 1
        return dict(kind=kind, batch=batch, longest=_log_int(rng, 16, min(8192, int(most))),
                    spread=rng.choice(["equal", "ragged"]), heads=heads, kv_heads=kv_heads,
                    width=width, floats=floats)
    batch = _log_int(rng, 1, 64)
    tokens = rng.choice([1, 1, 1, 2, 4, 7])
    most = 2 * 131072 * 8 * 128 // (batch * kv_heads * width)
    return dict(kind=kind, batch=batch, tokens=tokens, longest=_log_int(rng, 32, min(131072, most)),
                heads=heads, kv_heads=kv_heads, width=width, page=page, floats=floats)


def _padded(width):
    return next(w for w in WIDTHS if w >= width)


def _spread(case, batch, longest, low):
    """Lengths from `low` to `longest`, the same for every seed: one of each end and an empty
    request among the larger batches, the others anywhere between."""

    r = random.Random(sum(ord(c) * (i + 7) for i, c in enumerate(case["kind"])) + 31 * batch
                      + 17 * longest)
    lengths = [r.randint(low, longest) for _ in range(batch)]
    lengths[r.randrange(batch)] = longest
    if batch >= 8:
        others = [i for i in range(batch) if lengths[i] != longest]
        for at, n in zip(r.sample(others, min(2, len(others))), (low, max(low, min(1, longest)))):
            lengths[at] = n
    return lengths


def _lengths(case):
    """(tokens held, tokens new) of every request."""

    batch, longest = case["batch"], case["longest"]
    if case["kind"] == "prompt":
        new = ([longest] * batch if case["spread"] == "equal"
               else _spread(case, batch, longest, 0))
        return [0] * batch, new
    if case["kind"] == "cached":
        return _spread(case, batch, longest, 0 if batch >= 8 else min(longest, case["tokens"])), None
    held = _spread(case, batch, longest, 0)
    low = 1 if case["kind"] == "write" else 0
    new = [1] * batch if case["most"] == 1 else _spread(case, batch, case["most"], low)
    return held, new


# ------------------------------------------------------------------ inputs


def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed) * 1_000_003 + 29)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEVICE)


def _offsets(counts):
    return _ints(np.concatenate(([0], np.cumsum(counts))).astype(np.int64).tolist())


def _projection(g, rows, heads, kv_heads, width, dtype):
    """Queries, keys and values as a fused projection leaves them: slices of one matrix.  Some
    channels of the keys are larger than others."""

    x = torch.randn(rows, heads + 2 * kv_heads, width, generator=g, device=DEVICE)
    x[:, heads:heads + kv_heads] *= torch.exp(
        0.4 * torch.randn(kv_heads, width, generator=g, device=DEVICE))
    x = x.to(dtype)
    return x[:, :heads], x[:, heads:heads + kv_heads], x[:, heads + kv_heads:]


def _pages_of(tokens, page):
    return -(-tokens // page)


def _tables(g, held, page, columns, spare):
    """The page tables of requests that hold `held` tokens, over a pool in no order, and the
    stack of the pages that are free."""

    counts = [_pages_of(n, page) for n in held]
    total = sum(counts)
    order = torch.randperm(total + spare, generator=g, device=DEVICE).to(torch.int32)
    table = torch.full((len(held), columns), -1, dtype=torch.int32, device=DEVICE)
    mine = torch.arange(columns, device=DEVICE) < _ints(counts)[:, None]
    table[mine] = order[:total]
    free = torch.full((total + spare,), -1, dtype=torch.int32, device=DEVICE)
    free[:spare] = order[total:]
    return table, free, _ints([spare])


def _cache(g, pages, heads, width, page):
    """Codes and scales of a pool in use: every page and head with a scale of its own."""

    padded = _padded(width)

    def codes(*shape, axis):
        scale = torch.exp2(torch.randint(-9, -6, (pages, heads), generator=g, device=DEVICE).float())
        x = torch.empty(pages, heads, *shape, dtype=CODES, device=DEVICE)
        for h in range(heads):
            y = torch.randn(pages, *shape, generator=g, device=DEVICE)
            y.narrow(axis + 1, width, padded - width).zero_()
            x[:, h] = (y / scale[:, h, None, None]).clamp_(-MOST_CODE, MOST_CODE).to(CODES)
        return x, scale

    keys, key_scales = codes(page, padded, axis=1)
    values, value_scales = codes(padded, page, axis=0)
    return dict(key_pages=keys, key_scales=key_scales, value_pages=values,
                value_scales=value_scales)


def prepare(case, seed):
    g, kind = _generator(seed), case["kind"]
    held, new = _lengths(case)
    if kind == "prompt":
        q, k, v = _projection(g, sum(new), case["heads"], case["kv_heads"], case["width"],
                              FLOATS[case["floats"]])
        return dict(kind=kind, query=q, key=k, value=v, offsets=_offsets(new),
                    longest=case["longest"])
    page = case["page"]
    if kind == "cached":
        table, _, _ = _tables(g, held, page, _pages_of(case["longest"], page), 3)
        pages = int(table.max()) + 1 if table.numel() else 1
        pages = max(pages, sum(_pages_of(n, page) for n in held) + 3)
        q = 1.2 * torch.randn(case["batch"], case["tokens"], case["heads"], case["width"],
                              generator=g, device=DEVICE)
        return dict(kind=kind, query=q.to(FLOATS[case["floats"]]), page_tables=table,
                    lengths=_ints(held), longest=case["longest"],
                    **_cache(g, pages, case["kv_heads"], case["width"], page))
    # the order of the requests differs from seed to seed
    order = torch.randperm(len(held), generator=g, device=DEVICE).tolist()
    held, new = [held[i] for i in order], [new[i] for i in order]
    need = sum(_pages_of(h + n, page) - _pages_of(h, page) for h, n in zip(held, new))
    columns = _pages_of(case["longest"] + case["most"], page)
    table, free, count = _tables(g, held, page, columns, need + 5)
    tokens = sum(new)
    plan = dict(lengths=_ints(held), added=_ints(new), page_tables=table, free_pages=free,
                free_count=count, page=page, tokens=tokens)
    if kind == "tables":
        batch = len(held)
        out = (torch.empty(batch, dtype=torch.int32, device=DEVICE),
               torch.empty(1, dtype=torch.int32, device=DEVICE),
               torch.empty(batch + 1, dtype=torch.int32, device=DEVICE),
               torch.empty(tokens, dtype=torch.int32, device=DEVICE),
               torch.empty(tokens, dtype=torch.int32, device=DEVICE),
               torch.empty(1, dtype=torch.int32, device=DEVICE))
        return dict(kind=kind, out=out, **plan)
    _, _, offsets, _, slots, _ = _extend_plain(plan)
    _, k, v = _projection(g, tokens, 0, case["heads"], case["width"], FLOATS[case["floats"]])
    return dict(kind=kind, key=k, value=v, slots=slots, offsets=offsets,
                **_cache(g, free.numel(), case["heads"], case["width"], page))


# ------------------------------------------------------- the plain forms


def _softmax_product(scores, visible, values):
    """sum_j softmax_j(scores) values over what is visible; a row that sees nothing gives 0."""

    scores = torch.where(visible, scores, -math.inf)
    most = scores.amax(dim=-1, keepdim=True).clamp(min=torch.finfo(scores.dtype).min)
    p = torch.exp(scores - most)
    total = p.sum(dim=-1, keepdim=True)
    return torch.matmul(p, values) / torch.where(total > 0, total, 1.0)


def _prompt_plain(s):
    query, offsets, longest = s["query"], s["offsets"].long(), s["longest"]
    rows, heads, width = query.shape
    kv_heads, batch = s["key"].shape[1], offsets.numel() - 1
    group = heads // kv_heads
    at = torch.arange(longest, device=query.device)
    valid = at < (offsets[1:] - offsets[:-1])[:, None]
    row = torch.where(valid, offsets[:-1, None] + at, rows)

    def padded(x):
        x = x[row.clamp(max=rows - 1)].float()
        return torch.where(valid[:, :, None, None], x, 0.0)

    q = padded(query).view(batch, longest, kv_heads, group, width).permute(0, 2, 3, 1, 4)
    k = padded(s["key"]).permute(0, 2, 3, 1).contiguous()
    v = padded(s["value"]).transpose(1, 2).contiguous()
    scores = torch.matmul(q.reshape(batch, kv_heads, group * longest, width), k)
    scores = (scores * width ** -0.5).view(batch, kv_heads, group, longest, longest)
    scores = torch.where(at[None, :] <= at[:, None], scores, -math.inf)
    scores = scores.view(batch, kv_heads, group * longest, longest)
    p = torch.exp(scores - scores.amax(dim=-1, keepdim=True))
    mixed = torch.matmul(p, v) / p.sum(dim=-1, keepdim=True)
    mixed = mixed.view(batch, kv_heads, group, longest, width).permute(0, 3, 1, 2, 4)
    out = torch.zeros(rows + 1, heads, width, device=query.device)
    out[row] = mixed.reshape(batch, longest, heads, width)
    return out[:rows].to(query.dtype)


def _extend_plain(s):
    lengths, added, table = s["lengths"].long(), s["added"].long(), s["page_tables"]
    free, count, page, tokens = s["free_pages"], s["free_count"].long(), s["page"], s["tokens"]
    batch, columns = table.shape
    held, want = (lengths + page - 1) // page, (lengths + added + page - 1) // page
    need = want - held
    fits = (need.sum() <= count) & (want <= columns).all() & (added.sum() <= tokens)
    before = torch.cumsum(need, 0) - need
    column = torch.arange(columns, device=table.device)
    fresh = (column >= held[:, None]) & (column < want[:, None]) & fits
    at = count - 1 - (before - held)[:, None] - column
    table.copy_(torch.where(fresh, free[at.clamp(0, free.numel() - 1)], table))
    ends = torch.cumsum(added, 0)
    starts = ends - added
    t = torch.arange(tokens, device=table.device)
    request = torch.zeros(tokens + 1, dtype=torch.int64, device=table.device)
    request.index_add_(0, ends.clamp(max=tokens), torch.ones_like(ends))
    request = torch.cumsum(request, 0)[:tokens].clamp(max=batch - 1)
    given = (t < ends[-1]) & fits
    position = torch.where(given, lengths[request] + t - starts[request], -1)
    entry = table[request, (position // page).clamp(0, columns - 1)]
    slot = torch.where(given, entry * page + position % page, -1)
    offsets = torch.cat((torch.zeros_like(ends[:1]), ends))

    def narrow(x):
        return x.to(torch.int32)

    return (narrow(torch.where(fits, lengths + added, lengths)),
            narrow(torch.where(fits, count - need.sum(), count)), narrow(offsets),
            narrow(position), narrow(slot), narrow((~fits).reshape(1)))


def _power_scale(most):
    """The least power of two, within 2**-100 to 2**119, by which `most` is at most 448."""

    mantissa, exponent = torch.frexp(most)          # most = mantissa * 2**exponent, mantissa < 1
    exponent = torch.where(mantissa <= 0.875, exponent - 9, exponent - 8)
    exponent = torch.where(most > 0, exponent, -100).clamp(-100, 119)
    return torch.ldexp(torch.ones_like(most), exponent)


def _encode(x, scale):
    return torch.where(torch.isfinite(x), (x / scale).clamp(-MOST_CODE, MOST_CODE),
                       math.nan).to(CODES)


def _write_plain(s):
    slots, starts = s["slots"].long(), s["offsets"][:-1].long()

    def write(x, codes, scales, transposed):
        pages, heads, page = codes.shape[0], codes.shape[1], codes.shape[3 if transposed else 2]
        padded = codes.shape[2 if transposed else 3]
        x = torch.nn.functional.pad(x.float(), (0, padded - x.shape[-1]))
        at, token = slots // page, slots % page
        finite = torch.where(torch.isfinite(x), x.abs(), 0.0)
        most = torch.zeros(pages, heads, device=x.device)
        most.scatter_reduce_(0, at[:, None].expand(-1, heads), finite.amax(dim=-1), "amax")
        needed = _power_scale(most)
        # a request's first page goes on where its earlier tokens ended: its codes are taken to
        # the new scale; every other page is a new one
        first, kept = at[starts], token[starts] > 0
        old = scales[first]
        taken = torch.where(kept[:, None], torch.maximum(old, needed[first]), needed[first])
        before = codes[first].float() * old[:, :, None, None]
        again = _encode(before, taken[:, :, None, None])
        bits = codes.view(torch.uint8)
        bits[first] = torch.where(kept[:, None, None, None], again.view(torch.uint8), bits[first])
        scales[at] = needed[at]
        scales[first] = taken
        new = _encode(x, scales[at][:, :, None]).view(torch.uint8)
        if transposed:
            bits.permute(0, 3, 1, 2)[at, token] = new
        else:
            bits.transpose(1, 2)[at, token] = new

    write(s["key"], s["key_pages"], s["key_scales"], False)
    write(s["value"], s["value_pages"], s["value_scales"], True)
    return [s["key_pages"], s["key_scales"], s["value_pages"], s["value_scales"]]


def _cached_plain(s):
    query, lengths = s["query"], s["lengths"].long()
    batch, tokens, heads, width = query.shape
    table = s["page_tables"].long().clamp(min=0)
    kv_heads, page = s["key_pages"].shape[1:3]
    group, span = heads // kv_heads, table.shape[1] * page

    def gathered(codes, scales):
        x = codes.view(torch.uint8)[table].view(CODES).float()
        return x * scales[table][..., None, None]

    k = gathered(s["key_pages"], s["key_scales"])[..., :width]
    k = k.permute(0, 2, 4, 1, 3).reshape(batch, kv_heads, width, span)
    v = gathered(s["value_pages"], s["value_scales"])[..., :width, :]
    v = v.permute(0, 2, 1, 4, 3).reshape(batch, kv_heads, span, width)
    q = query.float().view(batch, tokens, kv_heads, group, width).permute(0, 2, 1, 3, 4)
    scores = torch.matmul(q.reshape(batch, kv_heads, tokens * group, width), k) * width ** -0.5
    last = lengths[:, None] - tokens + torch.arange(tokens, device=query.device)
    at = torch.arange(span, device=query.device)
    visible = (at <= last[:, :, None])[:, None, :, None, :].expand(-1, -1, -1, group, -1)
    visible = visible.reshape(batch, 1, tokens * group, span)
    seen = (at < lengths[:, None])[:, None, :, None]
    mixed = _softmax_product(scores, visible, torch.where(seen, v, 0.0))
    mixed = mixed.view(batch, kv_heads, tokens, group, width).permute(0, 2, 1, 3, 4)
    return mixed.reshape(batch, tokens, heads, width).to(query.dtype)


# --------------------------------------------------------------------- run


def run(s):
    kind = s["kind"]
    if not own:
        if kind == "tables":
            return [s["page_tables"], *_extend_plain(s)]
        return {"prompt": _prompt_plain, "write": _write_plain, "cached": _cached_plain}[kind](s)
    import copy_on_write_sdm_amd as cow

    if kind == "prompt":
        return cow.prompt_attention(s["query"], s["key"], s["value"], s["offsets"],
                                    longest=s["longest"])
    if kind == "tables":
        step = cow.extend_page_tables(s["lengths"], s["added"], s["page_tables"],
                                      s["free_pages"], s["free_count"], page_tokens=s["page"],
                                      tokens=s["tokens"], out=s["out"])
        return [s["page_tables"], *step]
    if kind == "write":
        cow.write_kv_cache(s["key"], s["value"], s["slots"], s["key_pages"], s["key_scales"],
                           s["value_pages"], s["value_scales"])
        return [s["key_pages"], s["key_scales"], s["value_pages"], s["value_scales"]]
    return cow.cached_attention(s["query"], s["key_pages"], s["key_scales"], s["value_pages"],
                                s["value_scales"], s["page_tables"], s["lengths"],
                                longest=s["longest"])


def work(case):
    held, new = _lengths(case)
    kind, batch = case["kind"], case["batch"]
    size = {"float32": 4}.get(case.get("floats"), 2)
    if kind == "prompt":
        pairs = sum(n * (n + 1) // 2 for n in new)
        rows = sum(new) * case["width"]
        return dict(bytes=rows * size * 2 * (case["heads"] + case["kv_heads"]) + 4 * (batch + 1),
                    flops=4 * case["width"] * case["heads"] * pairs)
    page = case["page"]
    if kind == "cached":
        tokens = case["tokens"]
        pairs = sum(max(0, n - tokens + i + 1) for n in held for i in range(tokens))
        pages = sum(_pages_of(n, page) for n in held)
        rows = batch * tokens * case["heads"] * case["width"]
        return dict(bytes=2 * sum(held) * case["kv_heads"] * case["width"] + 4 * batch
                    + pages * (4 + 8 * case["kv_heads"]) + 2 * rows * size,
                    flops=4 * case["width"] * case["heads"] * pairs)
    need = sum(_pages_of(h + n, page) - _pages_of(h, page) for h, n in zip(held, new))
    if kind == "tables":
        return dict(bytes=4 * (4 * batch + 2) + 8 * need + 8 * sum(new), flops=0)
    touched = sum(_pages_of(h + n, page) - h // page for h, n in zip(held, new))
    elements = 2 * sum(new) * case["heads"] * case["width"]
    return dict(bytes=elements * (size + 1) + 8 * touched * case["heads"] + 4 * sum(new),
                flops=4 * elements)


# --------------------------------------------------- the same in 64 bits


def _attend64(q, k, v, last):
    """Rows q [n, D] over keys and values [m, D]; row i sees keys 0 .. last[i]."""

    out = torch.zeros(q.shape[0], v.shape[1], dtype=torch.float64, device=q.device)
    some = last >= 0
    if not k.shape[0] or not bool(some.any()):
        return out
    logits = (q[some] @ k.T) / math.sqrt(q.shape[1])
    logits.masked_fill_(torch.arange(k.shape[0], device=q.device) > last[some, None], -math.inf)
    out[some] = torch.softmax(logits, dim=-1) @ v
    return out


def _e4m3(x):
    """x, in 64 bits, to the nearest float8 e4m3 number (even on a tie)."""

    exponent = torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -6)))
    exponent = torch.where(torch.exp2(exponent) > x.abs(), exponent - 1, exponent).clamp(min=-6)
    step = torch.exp2(exponent - 3)
    return torch.round(x / step) * step


def _exact_scale(most):
    if most == 0.0:
        return 2.0 ** -100
    e = math.ceil(math.log2(most / MOST_CODE))
    while most > MOST_CODE * 2.0 ** e:
        e += 1
    while most <= MOST_CODE * 2.0 ** (e - 1):
        e -= 1
    return 2.0 ** min(119, max(-100, e))


def _exact_write(s):
    slots = s["slots"].tolist()
    page = s["key_pages"].shape[2]
    runs, at = [], 0                    # tokens that follow one another in one page
    while at < len(slots):
        end = at + 1
        while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % page:
            end += 1
        runs.append((at, end))
        at = end

    def written(x, codes, scales):
        # codes as [pages, heads, page, padded]
        codes, scales = codes.double(), scales.double()
        for begin, end in runs:
            into, first = divmod(slots[begin], page)
            rows = x[begin:end].double()
            for h, most in enumerate(rows.abs().amax(dim=(0, 2)).tolist()):
                scale = _exact_scale(most)
                if first:
                    old = float(scales[into, h])
                    if old > scale:
                        scale = old
                    elif old < scale:
                        codes[into, h] = _e4m3(codes[into, h] * (old / scale))
                scales[into, h] = scale
                codes[into, h, first:first + end - begin, :x.shape[2]] = _e4m3(rows[:, h] / scale)
                codes[into, h, first:first + end - begin, x.shape[2]:] = 0.0
        return codes, scales

    keys, key_scales = written(s["key"], s["key_pages"], s["key_scales"])
    values, value_scales = written(s["value"], s["value_pages"].float().transpose(2, 3),
                                   s["value_scales"])
    return [keys, key_scales, values.transpose(2, 3).contiguous(), value_scales]


def exact(case, seed):
    s, kind = prepare(case, seed), case["kind"]
    if kind == "tables":
        return None                     # whole numbers only
    if kind == "write":
        return _exact_write(s)
    if kind == "prompt":
        query = s["query"]
        out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
        group = case["heads"] // case["kv_heads"]
        ends = s["offsets"].tolist()
        for begin, end in zip(ends, ends[1:]):
            last = torch.arange(end - begin, device=query.device)
            for h in range(case["heads"]):
                out[begin:end, h] = _attend64(
                    query[begin:end, h].double(), s["key"][begin:end, h // group].double(),
                    s["value"][begin:end, h // group].double(), last)
        return out
    query, page, width = s["query"], case["page"], case["width"]
    batch, tokens, heads, _ = query.shape
    group = heads // case["kv_heads"]
    out = torch.zeros(query.shape, dtype=torch.float64, device=query.device)
    for b, n in enumerate(s["lengths"].tolist()):
        mine = s["page_tables"][b, :_pages_of(n, page)].long()
        for h in range(case["kv_heads"]):
            k = s["key_pages"][:, h].view(torch.uint8)[mine].view(CODES).double()
            k = (k * s["key_scales"][mine, h, None, None].double()).reshape(-1, k.shape[-1])
            v = s["value_pages"][:, h].view(torch.uint8)[mine].view(CODES).double()
            v = (v * s["value_scales"][mine, h, None, None].double()).transpose(1, 2)
            v = v.reshape(-1, v.shape[-1])
            rows = query[b, :, h * group:(h + 1) * group].reshape(-1, width).double()
            last = n - tokens + torch.arange(tokens, device=query.device)
            mixed = _attend64(rows, k[:n, :width], v[:n, :width], last.repeat_interleave(group))
            out[b, :, h * group:(h + 1) * group] = mixed.view(tokens, group, width)
    return out

"""Cases, plain forms and exact values of the operators that serve token sequences from a paged cache
(disentangledcolorization_amd/paged.py).

The cache is two pools of pages, k_cache and v_cache, (pages, kv_heads, page, dim) or with a layer axis in front.  A row of
`page_table` lists the pages of one sequence, `lens` how many tokens it holds, `refs` how many rows name each page.  The new tokens of
all sequences lie behind each other; `cu_new` holds where each sequence's begin.

    attention   the new tokens attend to their sequence's cache, themselves included
    rotary      positions enter a tensor of heads
    append      pages for the new tokens are taken (lowest first), queries and keys are rotated, keys and values are written
    fork        rows become copies of other rows, pages shared, the last page copied where it is not full
    compact     the pages in use move to the lowest numbers
"""
import math
import random

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


# ---- cases --------------------------------------------------------------------------------------------------------------------

def _attention(name, dtype, seqs, max_new, max_len, q_heads, kv_heads, dim, page, window=0, lse=False):
    return {"name": name, "kind": "attention", "dtype": dtype, "seqs": seqs, "max_new": max_new, "max_len": max_len, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "page": page, "window": window, "lse": lse}


def _rotary(name, dtype, tokens, heads, dim, rotated, interleaved, scaling, factor, far):
    return {"name": name, "kind": "rotary", "dtype": dtype, "tokens": tokens, "heads": heads, "dim": dim, "rotated": rotated,
            "interleaved": interleaved, "scaling": scaling, "factor": factor, "far": far}


def _append(name, dtype, seqs, max_new, max_len, q_heads, kv_heads, dim, rotated, interleaved, page):
    return {"name": name, "kind": "append", "dtype": dtype, "seqs": seqs, "max_new": max_new, "max_len": max_len, "q_heads": q_heads,
            "kv_heads": kv_heads, "dim": dim, "rotated": rotated, "interleaved": interleaved, "page": page}


def _pages(name, kind, dtype, rows, beam, max_len, layers, kv_heads, dim, page, spare):
    return {"name": name, "kind": kind, "dtype": dtype, "rows": rows, "beam": beam, "max_len": max_len, "layers": layers,
            "kv_heads": kv_heads, "dim": dim, "page": page, "spare": spare}


def listed():
    return [
        # one user's next token over a short history: what counts is latency
        _attention("attend one token", "bf16", 1, 1, 256, 8, 8, 64, 16),
        # a full server's step: many sequences of unlike lengths, one new token each
        _attention("attend a batch's step", "bf16", 64, 1, 4096, 32, 8, 128, 16),
        # a step over two very long histories: the work has to be split over the keys
        _attention("attend a long history", "fp16", 2, 1, 131072, 32, 4, 128, 64, lse=True),
        # a server that mixes prompts' chunks with single tokens, three query heads a key head, idle rows among them
        _attention("attend chunks and tokens", "fp16", 24, 257, 4111, 12, 4, 64, 32, lse=True),
        # a long prompt's chunk behind a long history: the matrix cores bound it
        _attention("attend a long chunk", "bf16", 1, 2048, 16384, 32, 8, 128, 64),
        # wide heads that see only the last 1 024 keys
        _attention("attend a window", "bf16", 3, 701, 9001, 8, 2, 256, 16, window=1024),
        # one token's queries and keys of one layer
        _rotary("rotate one token", "fp16", 1, 40, 128, 128, False, "none", 1.0, 4096),
        # a long prompt of a model whose positions were stretched, half of each head rotated, pairs side by side
        _rotary("rotate a long prompt", "bf16", 16384, 32, 128, 64, True, "parts", 8.0, 1 << 20),
        # the step before "attend a batch's step"
        _append("append a batch's step", "bf16", 64, 1, 4096, 32, 8, 128, 128, False, 16),
        # prompts' chunks before attention, heads of 80 of which 32 are rotated
        _append("append prompts", "fp16", 5, 2500, 6000, 16, 4, 80, 32, True, 32),
        # beams: each step the rows become copies of the better ones, in all layers
        _pages("fork beams", "fork", "bf16", 64, 4, 1000, 8, 8, 64, 16, 0.25),
        # a pool with holes, before its upper half is given back
        _pages("compact the pool", "compact", "bf16", 32, 1, 1024, 4, 8, 128, 16, 1.0),
    ]


def _span(rng, low, high):
    """A whole number, even over its logarithm."""
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high + 0.49)))))))


def draw(rng):
    kind = rng.choice(("attention", "attention", "attention", "attention", "rotary", "append", "append", "fork", "compact"))
    dtype = rng.choice(("bf16", "fp16"))
    kv_heads = rng.choice((1, 2, 3, 4, 8))
    q_heads = kv_heads * rng.choice((1, 1, 2, 3, 4, 8))
    dim = rng.choice((8, 32, 64, 64, 80, 96, 128, 128, 128, 192, 256))
    page = rng.choice((1, 8, 16, 16, 32, 64, 128))
    if kind == "attention":
        seqs, new = _span(rng, 1, 96), rng.choice((1, 1, _span(rng, 2, 16), _span(rng, 17, 2048)))
        most = min(131072, 2 ** 27 // (seqs * kv_heads * dim), 2 ** 29 // (seqs * new * q_heads))
        length = _span(rng, 1, max(1, most))
        c = _attention("", dtype, seqs, min(new, length), length, q_heads, kv_heads, dim, page, rng.choice((0, 0, 0, _span(rng, 1, 2048))),
                       rng.random() < 0.5)
    elif kind == "rotary":
        rotated = 2 * rng.randint(2, dim // 2)
        c = _rotary("", rng.choice(("bf16", "fp16", "fp32")), _span(rng, 1, 2 ** 26 // (q_heads * 256)), q_heads, dim, rotated, rng.random() < 0.5,
                    rng.choice(("none", "linear", "ntk", "parts")), rng.choice((2.0, 4.0, 16.0)), _span(rng, 64, 1 << 22))
    elif kind == "append":
        seqs, new = _span(rng, 1, 96), rng.choice((1, 1, _span(rng, 2, 2048)))
        length = new + _span(rng, 1, max(1, min(16384, 2 ** 26 // (seqs * kv_heads * dim) - new)))
        c = _append("", dtype, seqs, new, length, q_heads, kv_heads, dim, 2 * rng.randint(2, dim // 2), rng.random() < 0.5, page)
    else:
        rows, layers = _span(rng, 1, 96), rng.randint(1, 8)
        length = _span(rng, 1, max(1, min(4096, 2 ** 26 // (rows * layers * kv_heads * dim))))
        c = _pages("", kind, dtype, rows, rng.choice((1, 2, 4, 7)), length, layers, kv_heads, dim, max(page, 8), rng.choice((0.25, 0.5, 1.0)))
    del c["name"]
    return c


# ---- what a case says of its sequences: the same for every seed ------------------------------------------------------------------

def _lengths(case):
    """(tokens in the cache, new ones among them) of every sequence: one of the full size, one idle, one without a history."""
    r = random.Random(case["seqs"] * 1000003 + case["max_len"])
    lens = [case["max_len"]] + [r.randint(max(1, case["max_len"] // 8), case["max_len"]) for _ in range(case["seqs"] - 1)]
    new = [min(n, case["max_new"] if i == 0 else r.randint(1, case["max_new"])) for i, n in enumerate(lens)]
    if case["seqs"] >= 6:
        lens[2], new[2] = 0, 0
        lens[3] = new[3]
    return lens, new


def _rows(case):
    """(lengths, pages shared with the group's first row, parents) of the rows of a fork or a compaction."""
    r = random.Random(case["rows"] * 1000003 + case["max_len"])
    lens, shared, parents = [], [], []
    for i in range(case["rows"]):
        first = i - i % case["beam"]
        n = r.randint(max(1, case["max_len"] // 2), case["max_len"]) if i == first else lens[first]
        lens.append(n)
        shared.append(0 if i == first else r.randint(0, n // case["page"]))
        parents.append(min(case["rows"] - 1, first + r.randrange(case["beam"])) if r.random() < 0.9 else i)
    if case["rows"] >= 6:
        parents[4] = -1  # a sequence that has ended
    return lens, shared, parents


def _table(case):
    """The pages that the rows of a fork or a compaction name, counted up from 0: lists, and how many there are."""
    lens, shared, _ = _rows(case)
    table, count = [], 0
    for i, n in enumerate(lens):
        used = -(-n // case["page"])
        first = i - i % case["beam"]
        alone = used - shared[i]
        table.append((table[first][:shared[i]] if shared[i] else []) + list(range(count, count + alone)))
        count += alone
    return table, count


def _frequencies(case):
    """Radians a position, in 64 bits, and the factor of the rotated values."""
    n = case["rotated"]
    i = torch.arange(0, n, 2, dtype=torch.float64)
    f = 10000.0 ** (-i / n)
    s = case.get("factor", 1.0)
    kind = case.get("scaling", "none")
    if kind == "linear":
        return f / s, 1.0
    if kind == "ntk":
        return (10000.0 * s ** (n / (n - 2))) ** (-i / n), 1.0
    if kind == "parts":  # pairs that turn often keep their frequency, pairs that turn less than once are stretched
        kept = ((4096 * f / (2 * math.pi) - 1.0) / (32.0 - 1.0)).clamp(0, 1)
        return (1 - kept) * f / s + kept * f, 0.1 * math.log(s) + 1.0
    return f, 1.0


def _visible(n, length, window):
    """How many (query, key) pairs a sequence has, and how many keys are seen at all."""
    pairs = sum(min(p + 1, window) if window else p + 1 for p in range(length - n, length))
    return pairs, (min(length, n + window - 1) if window else length) if n else 0


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "attention":
        lens, new = _lengths(case)
        seen = [_visible(n, x, case["window"]) for x, n in zip(lens, new)]
        b = 2 * sum(new) * case["q_heads"] * case["dim"] * size + 2 * sum(k for _, k in seen) * case["kv_heads"] * case["dim"] * size
        b += 4 * sum(-(-k // case["page"]) for _, k in seen) + 8 * case["seqs"] + (4 * sum(new) * case["q_heads"] if case["lse"] else 0)
        return {"bytes": b, "flops": 4 * sum(p for p, _ in seen) * case["q_heads"] * case["dim"]}
    if case["kind"] == "rotary":
        n = case["tokens"] * case["heads"]
        return {"bytes": 2 * n * case["dim"] * size + 8 * case["tokens"] + 4 * case["rotated"], "flops": 3 * n * case["rotated"]}
    if case["kind"] == "append":
        lens, new = _lengths(case)
        pages = sum(-(-x // case["page"]) for x in lens)
        b = 2 * sum(new) * (case["q_heads"] + 2 * case["kv_heads"]) * case["dim"] * size + 4 * (2 * pages + 2 * pages) + 12 * case["seqs"]
        return {"bytes": b, "flops": 3 * sum(new) * (case["q_heads"] + case["kv_heads"]) * case["rotated"]}
    table, count = _table(case)
    slot = 2 * case["layers"] * case["kv_heads"] * case["dim"] * size
    if case["kind"] == "fork":
        lens, _, parents = _rows(case)
        copies = _forked(case)
        b = sum(2 * slot * f for f in copies) + 8 * sum(-(-lens[p] // case["page"]) for p in parents if p >= 0) + 12 * case["rows"]
        return {"bytes": b + 4 * _pool(case), "flops": 0}
    moved = sum(1 for p in _places(case) if p >= count)
    return {"bytes": 2 * slot * case["page"] * moved + 8 * sum(map(len, table)) + 4 * _pool(case), "flops": 0}


def _forked(case):
    """The filled slots of every last page that a fork has to copy."""
    lens, _, parents = _rows(case)
    keeper = {}
    for i, p in enumerate(parents):
        if p >= 0:
            keeper[p] = min(keeper.get(p, i), -1 if p == i else i)
    return [lens[p] % case["page"] for i, p in enumerate(parents) if p >= 0 and lens[p] % case["page"] and keeper[p] != (-1 if p == i else i)]


def _pool(case):
    count = _table(case)[1]
    return count + case["rows"] + int(count * case["spare"])


def _places(case):
    """Where in the pool the pages that are in use lie."""
    r = random.Random(case["rows"] * 7919 + case["max_len"])
    return r.sample(range(_pool(case)), _table(case)[1])


# ---- inputs ---------------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    s = {"case": case}

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32 if math.prod(shape) < 1 << 24 else dtype).mul_(scale).to(dtype)

    def ints(values):
        return torch.tensor(values, dtype=torch.int32, device="cuda")

    if kind in ("rotary", "append"):
        f, s["gain"] = _frequencies(case)
        s["inv_freq"] = f.cuda()
    if kind == "rotary":
        s["x"] = randn(case["tokens"], case["heads"], case["dim"])
        s["positions"] = torch.randint(0, case["far"], (case["tokens"],), generator=g, device="cuda")
        return s
    if kind in ("attention", "append"):
        lens, new = _lengths(case)
        ps, before = case["page"], [x - n if kind == "append" else x for x, n in zip(lens, new)]
        used = [-(-x // ps) for x in before]
        pool = sum(-(-x // ps) for x in lens) + 3
        order = torch.randperm(pool, generator=g, device="cuda").int()
        width = max(-(-x // ps) for x in lens) + 1
        at = torch.arange(width, device="cuda")
        first = ints([sum(used[:i]) for i in range(len(used))])
        held = at < ints(used)[:, None]
        s["table"] = torch.where(held, order[(first[:, None] + at).clamp(max=pool - 1)], -1).int()
        s["lens"] = ints(before)
        s["cu_new"] = ints([sum(new[:i]) for i in range(len(new) + 1)])
        s["max_new"], s["max_len"] = max(new), max(lens)
        heads, dim, total = case["q_heads"] + 2 * case["kv_heads"], case["dim"], sum(new)
        qkv = randn(total, heads, dim)  # as one product with the joined weights leaves it
        s["q"], s["k"], s["v"] = qkv.split([case["q_heads"], case["kv_heads"], case["kv_heads"]], dim=1)
        s["k_cache"], s["v_cache"] = randn(pool, case["kv_heads"], ps, dim, scale=1.5), randn(pool, case["kv_heads"], ps, dim)
        if kind == "append":
            s["refs"] = torch.zeros(pool, dtype=torch.int32, device="cuda")
            s["refs"][order[:sum(used)].long()] = 1
        return s
    table, _ = _table(case)
    lens, _, parents = _rows(case)
    places, pool = _places(case), _pool(case)
    width = max(map(len, table)) + 1
    s["table"] = ints([[places[p] for p in row] + [-1] * (width - len(row)) for row in table])
    s["lens"], s["parents"] = ints(lens), ints(parents)
    shape = (case["layers"], pool, case["kv_heads"], case["page"], case["dim"])
    s["k_cache"], s["v_cache"] = randn(*shape), randn(*shape)
    return s


# ---- the plain forms --------------------------------------------------------------------------------------------------------------

def _per_token(cu_new, total):
    """The sequence of every new token, and its place among that sequence's new tokens."""
    at = torch.arange(total, device=cu_new.device)
    seq = torch.searchsorted(cu_new[1:].long(), at, right=True)
    return seq, at - cu_new[seq]


def _plain_attention(s):
    case, q, lens = s["case"], s["q"], s["lens"]
    ps, dim, kv_heads = case["page"], case["dim"], case["kv_heads"]
    group, seqs = case["q_heads"] // kv_heads, case["seqs"]
    new = s["cu_new"][1:] - s["cu_new"][:-1]
    pages = s["table"][:, :-(-s["max_len"] // ps)].clamp(min=0).long()
    keys = pages.shape[1] * ps
    k, v = (c[pages].float().permute(0, 2, 1, 3, 4).reshape(seqs, kv_heads, keys, dim) for c in (s["k_cache"], s["v_cache"]))
    seq, off = _per_token(s["cu_new"], q.shape[0])
    rows = torch.zeros(seqs, kv_heads, group, s["max_new"], dim, device=q.device)
    rows[seq, :, :, off] = q.float().view(-1, kv_heads, group, dim)
    scores = rows.view(seqs, kv_heads, -1, dim) @ k.transpose(2, 3).contiguous()
    scores = scores.mul_(1 / math.sqrt(dim)).view(seqs, kv_heads, group, s["max_new"], keys)
    pos = (lens - new)[:, None] + torch.arange(s["max_new"], device=q.device)
    key = torch.arange(keys, device=q.device)
    seen = (key <= pos[:, :, None]) & (key < lens[:, None, None])
    if case["window"]:
        seen &= key > pos[:, :, None] - case["window"]
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    p = scores.sub_(top.clamp(min=-1e30)).exp_()
    total = p.sum(-1, keepdim=True)
    v = torch.where((key < lens[:, None])[:, None, :, None], v, 0)
    out = (p.view(seqs, kv_heads, -1, keys) @ v).view(seqs, kv_heads, group, s["max_new"], dim)
    out = torch.where(total > 0, out / total, 0)[seq, :, :, off].reshape(q.shape).to(q.dtype)
    if not case["lse"]:
        return out
    return out, (top + total.log())[seq, :, :, off].reshape(q.shape[:2])


def _plain_rotary(x, positions, inv_freq, gain, interleaved):
    n = 2 * inv_freq.numel()
    angle = positions.double()[:, None] * inv_freq
    c, d = (gain * angle.cos()).float()[:, None], (gain * angle.sin()).float()[:, None]
    y = x.float()
    a, b = (y[..., 0:n:2], y[..., 1:n:2]) if interleaved else (y[..., :n // 2], y[..., n // 2:n])
    turned = (a * c - b * d, a * d + b * c)
    turned = torch.stack(turned, -1).flatten(-2) if interleaved else torch.cat(turned, -1)
    return torch.cat((turned, y[..., n:]), -1).to(x.dtype)


def _plain_reserve(table, lens, refs, new, ps):
    rows, width = table.shape
    have, want = (lens + ps - 1) // ps, (lens + new + ps - 1) // ps
    at = torch.arange(width, device=table.device)
    taken = ((at >= have[:, None]) & (at < want[:, None])).flatten()
    free = refs == 0
    missing = (want - have).sum() - free.sum()
    by_rank = torch.argsort(free.int(), descending=True, stable=True).int()
    got = by_rank[(taken.cumsum(0) - 1).clamp(0, refs.numel() - 1)]
    done = (missing <= 0) & (want <= width).all()
    grown = torch.where((at < have[:, None]), table, -1).flatten()
    table_out = torch.where(taken & done, got, grown).view(rows, width).int()
    refs_out = refs + (free & (free.cumsum(0) <= taken.sum()) & done)
    info = torch.stack(((refs_out == 0).sum(), missing.clamp(min=0), torch.zeros_like(missing), torch.zeros_like(missing)))
    return table_out, lens + torch.where(done, new, 0), refs_out.int(), info.int()


def _plain_append(s):
    case, new = s["case"], s["cu_new"][1:] - s["cu_new"][:-1]
    table, lens, refs, info = _plain_reserve(s["table"], s["lens"], s["refs"], new, case["page"])
    seq, off = _per_token(s["cu_new"], s["q"].shape[0])
    pos = (lens - new)[seq] + off
    q, k = (_plain_rotary(x, pos, s["inv_freq"], s["gain"], case["interleaved"]) for x in (s["q"], s["k"]))
    page, slot = table[seq, pos // case["page"]].long(), pos % case["page"]
    s["k_cache"][page, :, slot] = k
    s["v_cache"][page, :, slot] = s["v"]
    return q, s["k_cache"], s["v_cache"], table, lens.int(), refs, info


def _count(table, held, pool):
    """How many rows name each page."""
    return torch.zeros(pool, dtype=torch.int32, device=table.device).scatter_add_(0, table.clamp(min=0).flatten().long(), held.flatten().int())


def _plain_fork(s):
    table, ps, k_cache, v_cache = s["table"], s["case"]["page"], s["k_cache"], s["v_cache"]
    rows, width = table.shape
    at, row = torch.arange(width, device=table.device), torch.arange(rows, device=table.device)
    src = s["parents"].clamp(min=0).long()
    lens = torch.where(s["parents"] >= 0, s["lens"][src], 0)
    used = (lens + ps - 1) // ps
    held = at < used[:, None]
    out = torch.where(held, table[src], -1)
    rank = torch.where(lens > 0, torch.where(row == src, -1, row), rows)
    keeper = torch.full((rows,), rows, device=table.device).scatter_reduce_(0, src, rank, "amin")
    need = (lens % ps > 0) & (rank != keeper[src])
    last = (used - 1).clamp(min=0).long()
    tail = out.gather(1, last[:, None])[:, 0]
    refs = _count(out, held & ~(need[:, None] & (at == last[:, None])), k_cache.shape[1])
    free = refs == 0
    by_rank = torch.argsort(free.int(), descending=True, stable=True).int()
    missing = need.sum() - free.sum()
    fresh = by_rank[(need.cumsum(0) - 1).clamp(min=0)]
    out = torch.where(need[:, None] & (at == last[:, None]), fresh[:, None], out)
    refs = refs + (free & (free.cumsum(0) <= need.sum()))
    pick = need.nonzero()[:, 0]
    a, b = tail[pick].long(), fresh[pick].long()
    filled = (torch.arange(ps, device=table.device) < (lens % ps)[pick][:, None])[None, :, None, :, None]
    k_cache[:, b] = torch.where(filled, k_cache[:, a], k_cache[:, b])
    v_cache[:, b] = torch.where(filled, v_cache[:, a], v_cache[:, b])
    info = torch.stack(((refs == 0).sum(), missing.clamp(min=0), torch.zeros_like(missing), need.sum()))
    return out.int(), lens.int(), refs.int(), info.int(), k_cache, v_cache


def _plain_compact(s):
    table, ps, k_cache, v_cache = s["table"], s["case"]["page"], s["k_cache"], s["v_cache"]
    held = torch.arange(table.shape[1], device=table.device) < ((s["lens"] + ps - 1) // ps)[:, None]
    refs = _count(table, held, k_cache.shape[1])
    page = torch.arange(refs.numel(), device=table.device)
    live = refs > 0
    count = live.sum()
    hole, mover = (~live & (page < count)).nonzero()[:, 0], (live & (page >= count)).nonzero()[:, 0]
    to = page.clone()
    to[mover] = hole
    k_cache[:, hole] = k_cache[:, mover]
    v_cache[:, hole] = v_cache[:, mover]
    out = torch.where(held, to[table.clamp(min=0).long()], -1).int()
    zero = torch.zeros_like(count)
    info = torch.stack((refs.numel() - count, zero, zero, zero + mover.numel()))
    return out, torch.zeros_like(refs).scatter_add_(0, to, torch.where(live, refs, 0)), info.int(), k_cache, v_cache


# ---- one pass ---------------------------------------------------------------------------------------------------------------------

def run(s):
    case = s["case"]
    if own:
        return _own(s)
    if case["kind"] == "attention":
        return _plain_attention(s)
    if case["kind"] == "rotary":
        return _plain_rotary(s["x"], s["positions"], s["inv_freq"], s["gain"], case["interleaved"])
    return {"append": _plain_append, "fork": _plain_fork, "compact": _plain_compact}[case["kind"]](s)


def _own(s):
    from disentangledcolorization_amd import paged

    case, kind = s["case"], s["case"]["kind"]
    if kind == "attention":
        return paged.cache_attention(s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["cu_new"], window=case["window"],
                                     max_new=s["max_new"], max_len=s["max_len"], return_lse=case["lse"])
    if kind == "rotary":
        return paged.rotary(s["x"], s["positions"], s["inv_freq"], gain=s["gain"], interleaved=case["interleaved"])
    if kind == "append":
        table, lens, refs, info = paged.cache_reserve(s["table"], s["lens"], s["refs"], s["cu_new"], case["page"])
        q = paged.cache_append(s["q"], s["k"], s["v"], s["k_cache"], s["v_cache"], table, lens, s["cu_new"], inv_freq=s["inv_freq"],
                               gain=s["gain"], interleaved=case["interleaved"])
        return q, s["k_cache"], s["v_cache"], table, lens, refs, info
    if kind == "fork":
        return (*paged.cache_select(s["table"], s["lens"], s["parents"], s["k_cache"], s["v_cache"]), s["k_cache"], s["v_cache"])
    return (*paged.cache_compact(s["table"], s["lens"], s["k_cache"], s["v_cache"]), s["k_cache"], s["v_cache"])


# ---- from the definitions, in 64 bits -----------------------------------------------------------------------------------------------

def _turn(x, positions, inv_freq, gain, interleaved):
    """Pairs as complex numbers, turned."""
    n, x = 2 * inv_freq.numel(), x.double()
    pairs = x[..., :n].unflatten(-1, (-1, 2) if interleaved else (2, -1))
    z = torch.complex(*pairs.unbind(-1 if interleaved else -2))
    z = z * torch.polar(torch.full_like(inv_freq, gain), inv_freq * positions.double()[:, None])[:, None]
    return torch.cat((torch.stack((z.real, z.imag), -1 if interleaved else -2).flatten(-2), x[..., n:]), -1)


def exact(case, seed):
    if case["kind"] in ("fork", "compact"):
        return None  # nothing is computed: pages move
    s = prepare(case, seed)
    if case["kind"] == "rotary":
        return _turn(s["x"], s["positions"], s["inv_freq"], s["gain"], case["interleaved"])
    lens, new = _lengths(case)
    starts = [sum(new[:i]) for i in range(len(new))]
    if case["kind"] == "append":
        ps, table, free = case["page"], s["table"].tolist(), (s["refs"] == 0).nonzero()[:, 0].tolist()
        k_cache, v_cache, q = s["k_cache"].double(), s["v_cache"].double(), []
        for b, (length, n) in enumerate(zip(lens, new)):
            for i in range(-(-(length - n) // ps), -(-length // ps)):
                table[b][i] = free.pop(0)
            pos, here = torch.arange(length - n, length, device="cuda"), slice(starts[b], starts[b] + n)
            page = torch.tensor(table[b], device="cuda")[pos // ps]
            k_cache[page, :, pos % ps] = _turn(s["k"][here], pos, s["inv_freq"], s["gain"], case["interleaved"])
            v_cache[page, :, pos % ps] = s["v"][here].double()
            q.append(_turn(s["q"][here], pos, s["inv_freq"], s["gain"], case["interleaved"]))
        return [torch.cat(q), k_cache, v_cache] + [None] * 4
    heads, kv_heads, dim = case["q_heads"], case["kv_heads"], case["dim"]
    group = heads // kv_heads
    out = torch.zeros(sum(new), heads, dim, dtype=torch.float64, device="cuda")
    lse = torch.full((sum(new), heads), -math.inf, dtype=torch.float64, device="cuda")
    for b, (length, n) in enumerate(zip(lens, new)):
        if not n:
            continue
        first = max(0, length - n - case["window"] + 1) if case["window"] else 0
        token = torch.arange(first, length, device="cuda")
        page, slot = s["table"][b].long()[token // case["page"]], token % case["page"]
        query = torch.arange(length - n, length, device="cuda")[:, None]
        hidden = token > query
        if case["window"]:
            hidden |= query - token >= case["window"]
        here = slice(starts[b], starts[b] + n)
        for h in range(kv_heads):
            k, v = s["k_cache"][page, h, slot].double(), s["v_cache"][page, h, slot].double()
            for j in range(h * group, (h + 1) * group):
                w = torch.where(hidden, -math.inf, s["q"][here, j].double() @ k.T / math.sqrt(dim))
                lse[here, j] = torch.logsumexp(w, 1)
                out[here, j] = torch.softmax(w, 1) @ v
    return (out, lse) if case["lse"] else out

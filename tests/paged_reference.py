"""Plain 64-bit implementations of the paged-cache operators, for tests/test_gpu_paged.py and tests/test_paged_cpu.py: loops over sequences and
rows on the CPU, written from the definitions."""
import math

import torch


def turned(x, positions, inv_freq, gain=1.0, interleaved=False, inverse=False):
    """(values, magnitudes |a| + |b| of the pair behind every element), float64."""
    x, n = x.double().cpu(), 2 * len(inv_freq)
    out, size = x.clone(), torch.zeros_like(x)
    sign = -1.0 if inverse else 1.0
    for i, f in enumerate(inv_freq.double().cpu().tolist()):
        a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + n // 2)
        angle = positions.double().cpu() * f
        c, s = (gain * angle.cos())[:, None], (sign * gain * angle.sin())[:, None]
        out[..., a] = x[..., a] * c - x[..., b] * s
        out[..., b] = x[..., a] * s + x[..., b] * c
        size[..., a] = size[..., b] = abs(gain) * (x[..., a].abs() + x[..., b].abs())
    return out, size


def attended(q, k_cache, v_cache, table, lens, cu, causal=True, window=0, scale=None):
    """(values, softmax-weighted |v|, lse, bound of the scores' fp32 error) of the tokens before cu[-1], float64."""
    q, kc, vc = q.double().cpu(), k_cache.double().cpu(), v_cache.double().cpu()
    table, lens, cu = table.tolist(), lens.tolist(), cu.tolist()
    pages, kv_heads, ps, dim = kc.shape
    heads, group = q.shape[1], q.shape[1] // kv_heads
    scale = 1 / math.sqrt(dim) if scale is None else scale
    out, size = torch.zeros(cu[-1], heads, dim, dtype=torch.float64), torch.zeros(cu[-1], heads, dim, dtype=torch.float64)
    lse, off = torch.full((cu[-1], heads), -math.inf, dtype=torch.float64), torch.zeros(cu[-1], heads, dtype=torch.float64)
    for b, length in enumerate(lens):
        n = cu[b + 1] - cu[b]
        if not n or not length:
            continue
        at = torch.arange(length)
        page = torch.tensor(table[b])[at // ps]
        bad = (page < 0) | (page >= pages)
        page = page.clamp(0, pages - 1)
        k, v = kc[page, :, at % ps], vc[page, :, at % ps]            # (length, kv_heads, dim)
        k[bad] = math.nan
        for i in range(n):
            p, t = length - n + i, cu[b] + i
            low, high = (max(0, p - window + 1) if window else 0), (p + 1 if causal else length)
            if p < 0 and causal:
                continue
            for h in range(heads):
                kk, vv = k[low:high, h // group], v[low:high, h // group]
                s = kk @ q[t, h] * scale
                lse[t, h] = torch.logsumexp(s, 0)
                w = torch.softmax(s, 0)
                out[t, h] = w @ vv
                size[t, h] = w @ vv.abs()
                off[t, h] = (kk.abs() @ q[t, h].abs()).max() * abs(scale) * (dim + 8) * 2.0 ** -24
    return out, size, lse, off


def reserved(table, lens, refs, cu, ps):
    """cache_reserve on lists: (table, lens, refs, [free, missing])."""
    width = len(table[0])
    used = [-(-n // ps) for n in lens]
    new = [max(0, cu[i + 1] - cu[i]) for i in range(len(lens))]
    want = [-(-(n + m) // ps) for n, m in zip(lens, new)]
    free = [p for p, r in enumerate(refs) if r == 0]
    held = [row[:u] + [-1] * (width - u) for row, u in zip(table, used)]
    long = sum(w - width for w in want if w > width)
    need = sum(w - u for w, u in zip(want, used) if w <= width)
    if need > len(free) or long:
        return held, list(lens), list(refs), [len(free), max(need - len(free), 0) + long]
    refs = list(refs)
    left = iter(free)
    for row, u, w in zip(held, used, want):
        for at in range(u, w):
            row[at] = next(left)
            refs[row[at]] = 1
    return held, [n + m for n, m in zip(lens, new)], refs, [refs.count(0), 0]


def selected(table, lens, parents, ps, pages):
    """cache_select on lists: (table, lens, refs, [free, missing, copied], copies [(src, dst, slots)])."""
    width = len(table[0])

    def count(rows):
        refs = [0] * pages
        for row in rows:
            for p in row:
                if 0 <= p < pages:
                    refs[p] += 1
        return refs

    new_lens = [lens[p] if p >= 0 else 0 for p in parents]
    new = [(table[p][:-(-lens[p] // ps)] if p >= 0 else []) for p in parents]
    keeper = {}
    for r, p in enumerate(parents):
        if p >= 0 and (p not in keeper or p == r):
            keeper[p] = r
    need = [r for r, p in enumerate(parents) if p >= 0 and lens[p] % ps and keeper[p] != r]
    refs = count([row[:-1] if r in need else row for r, row in enumerate(new)])
    free = [p for p in range(pages) if refs[p] == 0]
    if len(need) > len(free):
        held = [row[:-(-n // ps)] for row, n in zip(table, lens)]
        refs = count(held)
        return [row + [-1] * (width - len(row)) for row in held], list(lens), refs, [refs.count(0), len(need) - len(free), 0], []
    copies = []
    for r, page in zip(need, free):
        copies.append((new[r][-1], page, new_lens[r] % ps))
        new[r] = new[r][:-1] + [page]
        refs[page] = 1
    return [row + [-1] * (width - len(row)) for row in new], new_lens, refs, [refs.count(0), 0, len(copies)], copies


def selected_by_page(table, lens, parents, ps, pages):
    """The same for rows of any lengths whose pages (all of them inside the cache) may be shared in any way: of the rows that end inside a page one keeps it - a row
    that is its own parent, else the lowest - unless it is a full page of some row."""
    width = len(table[0])
    new_lens = [lens[p] if p >= 0 else 0 for p in parents]
    new = [(table[p][:-(-lens[p] // ps)] if p >= 0 else []) for p in parents]
    full = {page for row, n in zip(new, new_lens) for page in row[:n // ps]}
    ends = {}
    for r in sorted(range(len(parents)), key=lambda r: (parents[r] != r, r)):
        if new_lens[r] % ps:
            ends.setdefault(new[r][-1], []).append(r)
    need = sorted(r for page, rows in ends.items() for r in (rows if page in full else rows[1:]))

    def count(rows):
        refs = [0] * pages
        for row in rows:
            for p in row:
                refs[p] += 1
        return refs

    needs = set(need)
    refs = count([row[:-1] if r in needs else row for r, row in enumerate(new)])
    free = [p for p in range(pages) if refs[p] == 0]
    if len(need) > len(free):
        held = [row[:-(-n // ps)] for row, n in zip(table, lens)]
        refs = count(held)
        return [row + [-1] * (width - len(row)) for row in held], list(lens), refs, [refs.count(0), len(need) - len(free), 0], []
    copies = []
    for r, page in zip(need, free):
        copies.append((new[r][-1], page, new_lens[r] % ps))
        new[r] = new[r][:-1] + [page]
        refs[page] = 1
    return [row + [-1] * (width - len(row)) for row in new], new_lens, refs, [refs.count(0), 0, len(copies)], copies


def compacted(table, lens, ps, pages):
    """cache_compact on lists: (table, refs, [free, moved], moves [(src, dst)])."""
    width = len(table[0])
    held = [row[:-(-n // ps)] for row, n in zip(table, lens)]
    refs = [0] * pages
    for row in held:
        for p in row:
            refs[p] += 1
    live = sum(r > 0 for r in refs)
    moves = list(zip([p for p in range(live, pages) if refs[p]], [p for p in range(live) if not refs[p]]))
    to = dict(moves)
    new_refs = [0] * pages
    for p, r in enumerate(refs):
        new_refs[to.get(p, p)] += r
    return [[to.get(p, p) for p in row] + [-1] * (width - len(row)) for row in held], new_refs, [pages - live, len(moves)], moves

#!/usr/bin/env python
"""Timings of the paged-cache operators (disentangledcolorization_amd/paged.py) on one GPU.

    python tools/paged_bench.py cases [--draw N] [--seed S]   the cases of perf/operators.py: plain form and kernels in turn, and what both are off by
    python tools/paged_bench.py sweep                         attention over batch, new tokens, history, heads and windows, from a graph
    python tools/paged_bench.py steps                         steps of many sequences over wide tables without bounds: time and workspace
    python tools/paged_bench.py floor                         the rates that floors are taken from: a large copy, a large product
    python tools/paged_bench.py loop NAME [PASSES]            the kernels of the cases whose names hold NAME, for a profiler:
        cd /tmp && rocprofv3 --kernel-trace --stats -f csv -d OUT -o k -- python3 $REPO/tools/paged_bench.py loop "attend"
        cd /tmp && rocprofv3 --pmc SQ_BUSY_CYCLES SQ_INSTS_VALU SQ_INSTS_MFMA SQ_VALU_MFMA_BUSY_CYCLES -f csv -d OUT -o p -- python3 ... loop "a long chunk" 3
(profiles/paged_cases.txt, paged_sweep.txt, paged_kernel_stats.csv, paged_pmc.txt)"""
import argparse
import os
import random
import sys

import torch

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
sys.path[:0] = [REPO, os.path.join(REPO, "perf")]


def timed(f, passes):
    """us a pass, launched one behind the other."""
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    a, b = torch.cuda.Event(True), torch.cuda.Event(True)
    a.record()
    for _ in range(passes):
        f()
    b.record()
    torch.cuda.synchronize()
    return a.elapsed_time(b) / passes * 1e3


def timed_graph(f, calls=10, replays=10):
    """us a call inside a graph: no host in it."""
    for _ in range(10):
        f()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        for _ in range(calls):
            f()
    g.replay()
    torch.cuda.synchronize()
    return timed(g.replay, replays) / calls


def tensors(x):
    return [x] if torch.is_tensor(x) or x is None else [t for y in (x.values() if isinstance(x, dict) else x) for t in tensors(y)]


def off(a, b):
    """|a - b| over |b| of all elements, and the largest difference; whole values: how many differ."""
    if not a.is_floating_point():
        return "%d of %d differ" % ((a != b).sum().item(), a.numel())
    a, b = a.double(), b.double()
    d = torch.where((a == b) | (a.isnan() & b.isnan()), 0, a - b)
    return "%.2g (max %.2g)" % (d.norm() / b[b.isfinite()].norm().clamp(min=1e-300), d.abs().max())


def cases(args):
    import operators as M
    rng = random.Random(args.seed)
    listed = M.listed() + [dict(M.draw(rng), name="drawn %d" % i) for i in range(args.draw)]
    print("us a call with its Python and launches; off: from the 64-bit values, of all elements; both sides on the same inputs")
    for c in listed:
        s = M.prepare(c, 1)
        t = {False: [], True: []}
        for own in (False, True, True, False):
            M.own = own
            t[own].append(timed(lambda: M.run(s), 200 if own else 10))
        errors = []
        want = M.exact(c, 2)
        for own in (False, True):
            M.own = own
            got = tensors(M.run(M.prepare(c, 2)))
            errors.append([off(g, w.to(g.device)) for g, w in zip(got, tensors(want)) if w is not None] if want is not None else got)
        if want is None:
            errors = [["-"], [off(a, b) + " from the plain form's" for a, b in zip(*errors)]]
        print("%-26s plain %9.1f  kernels %8.1f   off: plain %s; kernels %s" % (c["name"], min(t[False]), min(t[True]), ", ".join(errors[0]), ", ".join(errors[1])), flush=True)
        if c["name"].startswith("drawn"):
            print("    %s" % {k: v for k, v in c.items() if k != "name"}, flush=True)
        del s, want, got, errors
        torch.cuda.empty_cache()


def served(lens, new, kv_heads, heads, dim, page, dtype, width=0):
    used = [-(-n // page) for n in lens]
    pool = sum(used) + 1
    k, v = (torch.randn(pool, kv_heads, page, dim, device="cuda", dtype=dtype) for _ in range(2))
    table, order, at = torch.full((len(lens), max(width, max(used))), -1, dtype=torch.int32), torch.randperm(pool).int(), 0
    for b, u in enumerate(used):
        table[b, :u] = order[at:at + u]
        at += u
    ints = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return torch.randn(sum(new), heads, dim, device="cuda", dtype=dtype), k, v, table.cuda(), ints(lens), ints([sum(new[:b]) for b in range(len(new) + 1)])


SWEEP = [
    # sequences, new tokens, keys, heads, key heads, elements, page, window
    (1, 1, 256, 8, 8, 64, 16, 0), (1, 1, 1024, 32, 8, 128, 16, 0), (1, 1, 4096, 32, 8, 128, 16, 0), (1, 1, 16384, 32, 8, 128, 16, 0), (1, 1, 65536, 32, 8, 128, 16, 0),
    (8, 1, 4096, 32, 8, 128, 16, 0), (64, 1, 2048, 32, 8, 128, 16, 0), (64, 1, 4096, 32, 8, 128, 64, 0), (256, 1, 1024, 32, 8, 128, 16, 0), (16, 1, 16384, 32, 8, 128, 16, 0),
    (64, 1, 2048, 32, 32, 128, 16, 0), (1, 8, 4096, 32, 8, 128, 16, 0), (1, 8, 65536, 32, 8, 128, 16, 0), (8, 16, 4096, 32, 1, 128, 16, 0), (1, 33, 4096, 32, 8, 128, 16, 0),
    (1, 256, 4096, 32, 8, 128, 16, 0), (1, 256, 18432, 32, 8, 128, 64, 0), (8, 128, 4096, 32, 8, 128, 64, 0), (1, 512, 8192, 32, 8, 128, 64, 0), (1, 1024, 1024, 32, 8, 128, 64, 0),
    (4, 1024, 1024, 32, 8, 128, 64, 0), (1, 2048, 2048, 32, 8, 128, 64, 0), (1, 2048, 16384, 32, 8, 128, 64, 0), (1, 8192, 8192, 32, 8, 128, 64, 0),
    (1, 2048, 16384, 16, 4, 64, 16, 0), (4, 2048, 8192, 16, 2, 64, 16, 0), (1, 512, 4096, 8, 8, 256, 64, 0), (1, 2048, 8192, 8, 2, 256, 64, 0),
    (3, 701, 9001, 8, 2, 256, 16, 1024), (64, 1, 8192, 32, 8, 128, 16, 1024), (1, 2048, 16384, 32, 8, 128, 64, 4096),
]


def sweep(args):
    from disentangledcolorization_amd import paged
    print("bf16, causal, bounds given; us a call from a graph; TB/s of the keys and values that are seen, TF of the products that are")
    for b, n, keys, heads, kv_heads, dim, page, window in SWEEP:
        x = served([keys] * b, [n] * b, kv_heads, heads, dim, page, torch.bfloat16)
        f = lambda precise=False: paged.cache_attention(*x, window=window, max_new=n, max_len=keys, precise=precise)
        seen = min(keys, n + window - 1) if window else keys
        pairs = sum(min(p + 1, window) if window else p + 1 for p in range(keys - n, keys))
        us, precise = timed_graph(f), timed_graph(lambda: f(True)) if n * heads // kv_heads > 16 else None
        print("%4d x %-5d over %-6d %2d/%-2d heads of %-3d page %-2d window %-5d %8.1f us %6.2f TB/s %6.0f TF%s" % (
            b, n, keys, heads, kv_heads, dim, page, window, us, 4 * b * seen * kv_heads * dim / us / 1e6, 4 * b * heads * dim * pairs / us / 1e6,
            "" if precise is None else "   precise %8.1f us" % precise), flush=True)


def steps(args):
    from disentangledcolorization_amd import paged
    r = random.Random(1)
    print("32 heads of 128 on 8, bf16, tables of 32 768 tokens (65 536 in the third); us a call, and what it allocates beside its result")
    for name, lens, new, width in (("1 000 x 1 over 1 024", [1024] * 1000, [1] * 1000, 2048), ("1 000 x 1 over up to 4 096", [r.randint(100, 4096) for _ in range(1000)], [1] * 1000, 2048),
                                   ("300 x 1, one over 65 536, the others over 500", [65536] + [500] * 299, [1] * 300, 4096),
                                   ("63 x 1 and one of 4 096, over up to 8 192", [r.randint(4096, 8192) for _ in range(64)], [4096] + [1] * 63, 2048),
                                   ("256 x 17 over 2 000", [2000] * 256, [17] * 256, 2048), ("256 x 17 over 20 000", [20000] * 256, [17] * 256, 2048),
                                   ("64 x 65 over up to 8 192", [r.randint(1000, 8192) for _ in range(64)], [65] * 64, 2048)):
        x = served(lens, new, 8, 32, 128, 16, torch.bfloat16, width)
        for kw in (dict(), dict(max_new=max(new), max_len=max(lens))):
            torch.cuda.empty_cache()
            torch.cuda.reset_peak_memory_stats()
            was = torch.cuda.memory_allocated()
            us = timed(lambda: paged.cache_attention(*x, **kw), 20)
            print("%-48s %-12s %8.1f us  %.2f GB" % (name, "with bounds" if kw else "without", us, (torch.cuda.max_memory_allocated() - was - x[0].nbytes) / 1e9), flush=True)


def floor(args):
    x = torch.empty(1 << 30, dtype=torch.uint8, device="cuda")
    y = torch.empty_like(x)
    print("copy of 1 GiB: %.2f TB/s" % (2 * x.nbytes / timed(lambda: y.copy_(x), 20) / 1e6))
    for dtype in (torch.bfloat16, torch.float16):
        a, b = (torch.randn(8192, 8192, device="cuda").to(dtype) for _ in range(2))
        print("%s product of 8 192^3: %.0f TF" % (str(dtype)[6:], 2 * 8192 ** 3 / timed(lambda: a @ b, 20) / 1e6))


def loop(args):
    import operators as M
    M.own = True
    for c in M.listed():
        if args.name in c["name"]:
            s = M.prepare(c, 1)
            for _ in range(args.passes):
                M.run(s)
            torch.cuda.synchronize()
            print(c["name"], flush=True)


if __name__ == "__main__":
    p = argparse.ArgumentParser(description=__doc__.split("\n")[0])
    sub = p.add_subparsers(dest="what", required=True)
    a = sub.add_parser("cases")
    a.add_argument("--draw", type=int, default=0)
    a.add_argument("--seed", type=int, default=1)
    for n in ("sweep", "steps", "floor"):
        sub.add_parser(n)
    a = sub.add_parser("loop")
    a.add_argument("name")
    a.add_argument("passes", type=int, nargs="?", default=20)
    args = p.parse_args()
    {"cases": cases, "sweep": sweep, "steps": steps, "floor": floor, "loop": loop}[args.what](args)

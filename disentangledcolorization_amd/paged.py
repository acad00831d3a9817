"""Token sequences served from a paged cache: rotary positions, attention of new tokens over the cache, and the cache's pages.

The cache is two tensors of pages, `k_cache` and `v_cache`, bf16 or fp16, (pages, kv_heads, page, dim) - or (layers, pages, kv_heads, page,
dim) for the page calls, whose layers share one table; other orders of the inner axes are fine as strides as long as the elements of a head
lie next to each other.  Row b of `page_table` (rows, width) int32 names the pages of sequence b, `lens` (rows,) int32 says how many tokens
it holds, `refs` (pages,) int32 how many rows name a page (0: free).  The new tokens of all sequences lie behind each other; `cu_new`
(rows + 1,) int32 holds where each sequence's begin; rows ahead of its first entry and behind its last belong to no sequence.

    inv_freq = rotary_frequencies(128, base=10000.0)
    page_table, lens, refs, info = cache_reserve(page_table, lens, refs, cu_new, page)      # pages for the new tokens
    q = cache_append(q, k, v, k_cache, v_cache, page_table, lens, cu_new, inv_freq=inv_freq, info=info)   # every layer
    out = cache_attention(q, k_cache, v_cache, page_table, lens, cu_new)
    page_table, lens, refs, info = cache_select(page_table, lens, parents, k_cache, v_cache)   # fork, reorder, free
    page_table, refs, info = cache_compact(page_table, lens, k_cache, v_cache)

Serving only: nothing here is differentiable, and tensors that ask for a gradient are refused (`rotary(inverse=True)` is the transposed
rotation).  Only rotary_frequencies synchronises, as its table is made on the host: it comes once, ahead of the steps.  All others run on the current stream of
the tensors' device and may be captured into a graph.  No CPU fallback: CPU tensors raise DiscoError.

Whether there were pages enough only the GPU knows when a step is under way: info[1] tells, and cache_append, given info, leaves the cache of
a step that found none as it was (what cache_attention then returns is not the new tokens').  The program looks at info when it suits it, frees pages and does
the step again.
"""
import ctypes as C
import math

import torch

from . import _ffi

_DTYPES = {torch.float16: _ffi.F16, torch.bfloat16: _ffi.BF16, torch.float32: _ffi.F32}
_SCALINGS = {None: _ffi.ROTARY_PLAIN, "linear": _ffi.ROTARY_LINEAR, "ntk": _ffi.ROTARY_NTK, "parts": _ffi.ROTARY_PARTS}
_INT32 = torch.int32
_MOST = 0x7fffffff


# (a step of a served model makes several of these calls a layer, each a few microseconds of GPU time: the checks are written to be quick)

def _device(values, ints=()):
    """The index of the one device that all tensors are on; floating tensors must not ask for a gradient."""
    device = values[0].get_device()
    if device < 0:
        raise _ffi.DiscoError("HIP path only: expected CUDA/HIP tensors (no CPU fallback)")
    for t in values:
        if t.get_device() != device:
            raise _ffi.DiscoError("tensors on several devices, or on the CPU (no CPU fallback)")
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("inference only: a tensor asks for a gradient")
    for t in ints:
        if t.get_device() != device:
            raise _ffi.DiscoError("tensors on several devices, or on the CPU (no CPU fallback)")
    return device


def _ints(name, t, shape):
    if t.dtype is not _INT32 or t.shape != shape or not t.is_contiguous():
        raise ValueError("%s must be contiguous int32 %s, got %s %s" % (name, tuple(shape), t.dtype, tuple(t.shape)))


def _call(device, fn, *args):
    """fn(*args, stream) on the current stream of the tensors' device, which need not be the current device."""
    if device == torch.cuda.current_device():
        rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    else:
        with torch.cuda.device(device):
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(device))
    if rc:
        _ffi.check(rc)


def _cache(k, v, page_table, layered=False):
    dims = 5 if layered and k.dim() == 5 else 4
    shape, st, other = k.shape, k.stride(), v.stride()
    if 1 in shape and v.shape == shape:                   # (the stride of an axis of one does not matter)
        st, other = (tuple(s if n > 1 else 0 for n, s in zip(shape, x)) for x in (st, other))
    if len(shape) != dims or v.shape != shape or v.dtype is not k.dtype or other != st:
        raise ValueError("k_cache and v_cache must be alike, (%spages, kv_heads, page, dim)" % ("[layers,] " if layered else ""))
    dtype = _DTYPES.get(k.dtype, _ffi.F32)
    if dtype == _ffi.F32:
        raise ValueError("the cache holds fp16 or bf16, got %s" % k.dtype)
    if st[-1] != 1 and shape[-1] > 1:
        raise ValueError("the elements of a head must lie next to each other")
    if page_table.dim() != 2:
        raise ValueError("page_table must be (rows, width)")
    rows, width = page_table.shape
    if max(*shape, rows, width) > _MOST:
        raise ValueError("a size beyond 2^31")
    if dims == 5:
        return _ffi.CacheDesc(dtype, shape[0], shape[1], shape[2], shape[3], shape[4], rows, width, st[0], st[1], st[2], st[3], k.data_ptr(), v.data_ptr())
    return _ffi.CacheDesc(dtype, 1, shape[0], shape[1], shape[2], shape[3], rows, width, 0, st[0], st[1], st[2], k.data_ptr(), v.data_ptr())


def _sequences(c, page_table, lens, cu_new):
    _ints("page_table", page_table, (c.rows, c.table_width))
    _ints("lens", lens, (c.rows,))
    _ints("cu_new", cu_new, (c.rows + 1,))


def _heads(name, t, tokens, heads, dim, dtype):
    """(tokens, heads, dim) with a head's elements next to each other: the two strides (0 of an axis of one, which has none that matters)."""
    if t.shape != (tokens, heads, dim) or t.dtype is not dtype:
        raise ValueError("%s must be (%d, %d, %d) %s, got %s %s" % (name, tokens, heads, dim, dtype, tuple(t.shape), t.dtype))
    token, head, one = t.stride()
    if one != 1 and dim > 1:
        raise ValueError("%s: the elements of a head must lie next to each other" % name)
    return token if tokens > 1 else 0, head if heads > 1 else 0


def _bound(n):
    """A whole number for an int32 argument whose check tells only too small from too large."""
    return max(-1, min(n, _MOST))


def _three(name, t):
    if t.dim() != 3:
        raise ValueError("%s must be (tokens, heads, dim)" % name)
    if t.shape[0] > _MOST:
        raise ValueError("%s: more than 2^31 tokens" % name)
    return t.shape


def _positions(positions, tokens):
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32 or int64 (%d,)" % tokens)
    return positions.dtype is torch.int64


def _frequencies(inv_freq):
    if inv_freq.dtype is not torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
        raise ValueError("inv_freq must be contiguous float64 (pairs,)")
    return 2 * inv_freq.numel()


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, original_length=4096, low=1.0, high=32.0, device="cuda"):
    """Radians a position of `dim` / 2 pairs, float64 on `device`.  For positions behind the trained length:
    scaling="linear" divides them all by `factor`; "ntk" changes the base so that the slowest pair is stretched by `factor` and the fastest
    kept; "parts" keeps pairs that make more than `high` turns over `original_length` positions, divides those with fewer than `low`, and
    blends in between (with a gain of 0.1 ln(factor) + 1 on the rotated values where the model was trained with one)."""
    if scaling not in _SCALINGS:
        raise ValueError("scaling must be None, 'linear', 'ntk' or 'parts'")
    out = torch.empty(max(int(dim) // 2, 1), dtype=torch.float64)
    _ffi.check(_ffi.lib().disco_op_rotary_frequencies(int(dim), _SCALINGS[scaling], base, factor, original_length, low, high, out.data_ptr()))
    return out.to(device)


def rotary(x, positions, inv_freq, gain=1.0, interleaved=False, inverse=False, out=None):
    """x (tokens, heads, dim) with the first 2 * len(inv_freq) elements of each head turned by its token's position and multiplied by
    `gain`; bf16, fp16 or fp32.  Pairs are (i, i + half), or (2i, 2i + 1) when interleaved.  inverse turns back.  out may be x."""
    device = _device((x, inv_freq), (positions,))
    tokens, heads, dim = _three("x", x)
    dtype = _DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError("x must be bf16, fp16 or fp32, got %s" % x.dtype)
    xs = _heads("x", x, tokens, heads, dim, x.dtype)
    wide, rotated = _positions(positions, tokens), _frequencies(inv_freq)
    if out is None:
        out = x.new_empty((tokens, heads, dim))
        os = (heads * dim if tokens > 1 else 0, dim if heads > 1 else 0)
    else:
        _device((x, out))
        os = _heads("out", out, tokens, heads, dim, x.dtype)
    if tokens and heads:
        d = _ffi.RotaryDesc(dtype, tokens, heads, dim, rotated, bool(interleaved), bool(inverse), wide, *xs, *os, gain)
        _call(device, _ffi.lib().disco_op_rotary, C.byref(d), x.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), out.data_ptr())
    return out


def cache_append(q, k, v, k_cache, v_cache, page_table, lens, cu_new, inv_freq=None, gain=1.0, interleaved=False, positions=None, q_out=None, info=None):
    """The new tokens' keys and values are written into their pages, keys (and queries, which are returned) turned by their positions on the
    way.  `lens` counts the new tokens already; `positions` replaces a token's place in its sequence as the angle's position; inv_freq=None turns
    nothing; q=None has no queries.  q_out may be q.

    info: cache_reserve's.  Where pages were missing nothing is written to the cache: a failed cache_reserve leaves `lens` as it was, and a step that goes on
    without info writes its tokens over the last cached ones of every sequence, and of those that share their pages."""
    device = _device((k, v, k_cache, v_cache), (page_table, lens, cu_new))
    c = _cache(k_cache, v_cache, page_table)
    _sequences(c, page_table, lens, cu_new)
    tokens, dtype = _three("k", k)[0], k_cache.dtype
    ks, vs = _heads("k", k, tokens, c.kv_heads, c.dim, dtype), _heads("v", v, tokens, c.kv_heads, c.dim, dtype)
    rotated, wide, q_heads, qs, os = 0, False, 0, (0, 0), (0, 0)
    if inv_freq is not None:
        _device((k, inv_freq))
        rotated = _frequencies(inv_freq)
    if positions is not None:
        _device((k,), (positions,))
        wide = _positions(positions, tokens)
    if info is not None:
        _device((k,), (info,))
        _ints("info", info, (4,))
    if q is not None:
        _device((k, q))
        q_heads = _three("q", q)[1]
        qs = _heads("q", q, tokens, q_heads, c.dim, dtype)
        if q_out is None:
            q_out, os = q.new_empty((tokens, q_heads, c.dim)), (q_heads * c.dim, c.dim)
        else:
            _device((k, q_out))
            os = _heads("q_out", q_out, tokens, q_heads, c.dim, dtype)
    elif q_out is not None:
        raise ValueError("q_out without q")
    if tokens:
        a = _ffi.AppendDesc(tokens, q_heads, rotated, bool(interleaved), wide, *qs, *ks, *vs, *os, gain)
        _call(device, _ffi.lib().disco_op_cache_append_reserved, C.byref(c), C.byref(a), q.data_ptr() if q_heads else None, k.data_ptr(), v.data_ptr(),
              page_table.data_ptr(), lens.data_ptr(), cu_new.data_ptr(), None if positions is None else positions.data_ptr(),
              None if inv_freq is None else inv_freq.data_ptr(), q_out.data_ptr() if q_heads else None, None if info is None else info.data_ptr())
    return q_out


def cache_attention(q, k_cache, v_cache, page_table, lens, cu_new, causal=True, window=0, scale=None, max_new=None, max_len=None,
                    return_lse=False, out=None, precise=False):
    """softmax(scale q k^T) v of every new token (tokens, q_heads, dim) over its sequence's cache, the new tokens among it (`lens` counts
    them).  Query head h reads key head h // (q_heads // kv_heads).  causal: the token at position p sees keys up to p, with `window` > 0 the last
    `window` of them; else the whole sequence.  A token that sees nothing gets zeros.  scale: 1 / sqrt(dim).

    precise: sequences of more than 16 rows (new tokens * query heads a key head) multiply the values with softmax weights of fp32 precision, as smaller ones
    always do; else with weights rounded to the cache's type, which is up to 1.4 times as fast and off by up to half a step of that type.

    max_new, max_len: what the caller knows of the largest number of new tokens and the largest length; they size launches and
    workspace, a sequence beyond them still comes out right.  With one row in the table, max_new = tokens says that every row of q is a new token of
    its sequence: fewer launches (a padded call leaves max_new out, or gives less).  Steps of hundreds of sequences over
    wide tables should give max_len: without it they take up to a gigabyte of workspace, and up to a quarter longer.  return_lse: also the logarithm of the softmax's sum, (tokens, q_heads)
    fp32.  `out` shares no memory with q.  Rows of no sequence are left as they are in a given `out`, and undefined in lse and an `out` of its own."""
    device = _device((q, k_cache, v_cache), (page_table, lens, cu_new))
    c = _cache(k_cache, v_cache, page_table)
    _sequences(c, page_table, lens, cu_new)
    tokens, q_heads, dim = _three("q", q)
    qs = _heads("q", q, tokens, q_heads, c.dim, k_cache.dtype)
    if out is None:
        out, os = q.new_empty((tokens, q_heads, dim)), (q_heads * dim, dim)
    else:
        _device((q, out))
        os = _heads("out", out, tokens, q_heads, dim, q.dtype)
    lse = q.new_empty((tokens, q_heads), dtype=torch.float32) if return_lse else None
    a = _ffi.AttentionDesc(tokens, q_heads, bool(causal), _bound(window), _bound(max_new or 0), _bound(max_len or 0),
                           1 / math.sqrt(dim) if scale is None else scale, *qs, *os)
    lib, need, cd, ad = _ffi.lib(), C.c_size_t(), C.byref(c), C.byref(a)
    _ffi.check(lib.disco_op_cache_attention_workspace_bytes(cd, ad, C.byref(need)))
    need = need.value
    ws = q.new_empty(need, dtype=torch.uint8) if need else None
    _call(device, lib.disco_op_cache_attention_precise if precise else lib.disco_op_cache_attention, cd, ad, q.data_ptr(), page_table.data_ptr(), lens.data_ptr(), cu_new.data_ptr(), out.data_ptr(),
          lse.data_ptr() if return_lse else None, ws.data_ptr() if need else None, need)
    return (out, lse) if return_lse else out


def _state(page_table, rows, width, pages):
    """New buffers for a table, its lengths, the pages' counts and info, in one allocation, and their addresses."""
    table = rows * width
    flat = page_table.new_empty(table + rows + pages + 4)
    at = flat.data_ptr()
    new, lens, refs, info = flat.split_with_sizes((table, rows, pages, 4))
    return ((new.view(rows, width), lens, refs, info), (at, at + 4 * table, at + 4 * (table + rows), at + 4 * (table + rows + pages)))


def cache_reserve(page_table, lens, refs, cu_new, page):
    """Pages for the new tokens of every row: (page_table, lens, refs, info) with them.  The lowest free pages are taken, rows ascending.
    info (4,) int32: free pages afterwards; pages that were missing - then the state returned is the old one -; lengths out of range; rows whose new
    tokens would go into a page that other rows name as well, each of which counts as a missing page.

    A row is cut back by a smaller length, as for drafted tokens that were rejected.  Where that leaves it inside a page which it shares, or for the pages behind
    its new end to become free, cache_select with every row its own parent comes first."""
    device = _device((page_table,), (lens, refs, cu_new))
    if page_table.dim() != 2 or refs.dim() != 1:
        raise ValueError("page_table must be (rows, width), refs (pages,)")
    rows, width = page_table.shape
    pages = refs.numel()
    if max(rows, width, pages) > _MOST:
        raise ValueError("a size beyond 2^31")
    _ints("page_table", page_table, (rows, width))
    _ints("lens", lens, (rows,))
    _ints("refs", refs, (pages,))
    _ints("cu_new", cu_new, (rows + 1,))
    new, at = _state(page_table, rows, width, pages)
    _call(device, _ffi.lib().disco_op_cache_reserve, rows, width, pages, _bound(page), page_table.data_ptr(), lens.data_ptr(), refs.data_ptr(), cu_new.data_ptr(), *at)
    return new


def _page_call(k_cache, v_cache, page_table, lens):
    c = _cache(k_cache, v_cache, page_table, True)
    _ints("page_table", page_table, (c.rows, c.table_width))
    _ints("lens", lens, (c.rows,))
    need = _ffi.lib().disco_op_cache_pages_workspace_bytes(c.rows, c.pages)
    return c, page_table.new_empty(need, dtype=torch.uint8), need


def cache_select(page_table, lens, parents, k_cache, v_cache):
    """Row r becomes what row parents[r] was, -1: empty; forks, reorders and frees rows in one call: (page_table, lens, refs, info).  Rows of one
    parent share its full pages; of a last page that is not full one row keeps the original and the others get copies, in all layers, also where
    it was a full page before its rows were cut back; and all get copies where it still is one for another row.
    info (4,) int32: free pages afterwards; pages that were missing - then the state returned is the old one -; entries out of range; pages copied."""
    device = _device((k_cache, v_cache), (page_table, lens, parents))
    c, ws, need = _page_call(k_cache, v_cache, page_table, lens)
    _ints("parents", parents, (c.rows,))
    new, at = _state(page_table, c.rows, c.table_width, c.pages)
    _call(device, _ffi.lib().disco_op_cache_select, C.byref(c), page_table.data_ptr(), lens.data_ptr(), parents.data_ptr(), *at, ws.data_ptr(), need)
    return new


def cache_compact(page_table, lens, k_cache, v_cache):
    """The n pages in use move to 0 .. n - 1, in all layers: (page_table, refs, info).  info as cache_select's."""
    device = _device((k_cache, v_cache), (page_table, lens))
    c, ws, need = _page_call(k_cache, v_cache, page_table, lens)
    (table, _, refs, info), at = _state(page_table, c.rows, c.table_width, c.pages)
    _call(device, _ffi.lib().disco_op_cache_compact, C.byref(c), page_table.data_ptr(), lens.data_ptr(), at[0], at[2], at[3], ws.data_ptr(), need)
    return table, refs, info


def cache_copy_pages(k_cache, v_cache, src, dst):
    """Page src[i] is copied to page dst[i], in all layers (src, dst int32).  No page of dst may be among src, or there twice;
    pairs out of range are skipped."""
    device = _device((k_cache, v_cache), (src, dst))
    if src.dim() != 1:
        raise ValueError("src must be (count,)")
    _ints("src", src, src.shape)
    _ints("dst", dst, src.shape)
    c = _cache(k_cache, v_cache, src[None], True)
    c.rows = c.table_width = 1
    if src.numel():
        _call(device, _ffi.lib().disco_op_cache_copy_pages, C.byref(c), src.data_ptr(), dst.data_ptr(), src.numel())

"""Token sequences served from a paged cache: rotary positions, attention of new tokens over the cache, and the cache's pages.

The cache is two tensors of pages, `k_cache` and `v_cache`, bf16 or fp16, (pages, kv_heads, page, dim) - or (layers, pages, kv_heads, page,
dim) for the page calls, whose layers share one table; other orders of the inner axes are fine as strides as long as the elements of a head
lie next to each other.  Row b of `page_table` (rows, width) int32 names the pages of sequence b, `lens` (rows,) int32 says how many tokens
it holds, `refs` (pages,) int32 how many rows name a page (0: free).  The new tokens of all sequences lie behind each other; `cu_new`
(rows + 1,) int32 holds where each sequence's begin.

    inv_freq = rotary_frequencies(128, base=10000.0)
    page_table, lens, refs, info = cache_reserve(page_table, lens, refs, cu_new, page)      # pages for the new tokens
    q = cache_append(q, k, v, k_cache, v_cache, page_table, lens, cu_new, inv_freq=inv_freq)   # every layer
    out = cache_attention(q, k_cache, v_cache, page_table, lens, cu_new)
    page_table, lens, refs, info = cache_select(page_table, lens, parents, k_cache, v_cache)   # fork, reorder, free
    page_table, refs, info = cache_compact(page_table, lens, k_cache, v_cache)

Serving only: nothing here is differentiable, and tensors that ask for a gradient are refused (`rotary(inverse=True)` is the transposed
rotation).  No call synchronises; on the current stream of the tensors' device all of them may be captured into a graph.  No CPU fallback:
CPU tensors raise DiscoError.
"""
import ctypes as C
import math

import torch

from . import _ffi

_DTYPES = {torch.float16: _ffi.F16, torch.bfloat16: _ffi.BF16, torch.float32: _ffi.F32}
_SCALINGS = {None: _ffi.ROTARY_PLAIN, "linear": _ffi.ROTARY_LINEAR, "ntk": _ffi.ROTARY_NTK, "parts": _ffi.ROTARY_PARTS}


def _check(device, **tensors):
    """One device, no gradient; integer tensors are int32 and contiguous."""
    for name, t in tensors.items():
        if not t.is_cuda:
            raise _ffi.DiscoError("HIP path only: expected CUDA/HIP tensors (no CPU fallback)")
        if t.device != device:
            raise ValueError("%s is on %s, expected %s" % (name, t.device, device))
        if t.requires_grad and torch.is_grad_enabled():
            raise NotImplementedError("inference only: %s asks for a gradient" % name)


def _ints(shape, **tensors):
    for name, t in tensors.items():
        if t.dtype != torch.int32 or not t.is_contiguous() or t.shape != shape:
            raise ValueError("%s must be contiguous int32 %s, got %s %s" % (name, tuple(shape), t.dtype, tuple(t.shape)))


class _on:
    """The tensors' device made current for a call (a no-op where it is), and its current stream."""

    def __init__(self, device):
        self.index = device.index

    def __enter__(self):
        self.back = torch.cuda.current_device()
        if self.back != self.index:
            torch.cuda.set_device(self.index)
        return torch.cuda.current_stream(self.index).cuda_stream

    def __exit__(self, *exc):
        if self.back != self.index:
            torch.cuda.set_device(self.back)


def _cache(k, v, page_table, layered):
    dims = 5 if layered and k.dim() == 5 else 4
    if k.dim() != dims or k.shape != v.shape or k.dtype != v.dtype or k.stride() != v.stride():
        raise ValueError("k_cache and v_cache must be alike, (%spages, kv_heads, page, dim)" % ("[layers,] " if layered else ""))
    if k.dtype not in (torch.float16, torch.bfloat16):
        raise ValueError("the cache holds fp16 or bf16, got %s" % k.dtype)
    st = k.stride()
    if st[-1] != 1:
        raise ValueError("the elements of a head must lie next to each other")
    if page_table.dim() != 2:
        raise ValueError("page_table must be (rows, width)")
    pages, kv_heads, page, dim = k.shape[-4:]
    layers, layer_stride = (k.shape[0], st[0]) if dims == 5 else (1, 0)
    rows, width = page_table.shape
    return _ffi.CacheDesc(_DTYPES[k.dtype], layers, pages, kv_heads, page, dim, rows, width, layer_stride, st[-4], st[-3], st[-2], k.data_ptr(), v.data_ptr())


def _heads(name, t, tokens, dim, dtype):
    """(tokens, heads, dim) with a head's elements next to each other: the two strides."""
    if t.dim() != 3 or t.shape[0] != tokens or t.shape[2] != dim or t.dtype != dtype:
        raise ValueError("%s must be (%d, heads, %d) %s, got %s %s" % (name, tokens, dim, dtype, tuple(t.shape), t.dtype))
    token, head, one = t.stride()
    if one != 1 and dim > 1:
        raise ValueError("%s: the elements of a head must lie next to each other" % name)
    return token, head


def _positions(positions, tokens):
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape != (tokens,) or not positions.is_contiguous():
        raise ValueError("positions must be contiguous int32 or int64 (%d,)" % tokens)
    return int(positions.dtype == torch.int64)


def _frequencies(inv_freq):
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not inv_freq.is_contiguous():
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
    _check(x.device, x=x, positions=positions, inv_freq=inv_freq)
    if x.dtype not in _DTYPES or x.dim() != 3:
        raise ValueError("x must be (tokens, heads, dim), bf16, fp16 or fp32")
    tokens, heads, dim = x.shape
    xs = _heads("x", x, tokens, dim, x.dtype)
    wide, rotated = _positions(positions, tokens), _frequencies(inv_freq)
    with _on(x.device) as stream:
        if out is None:
            out = torch.empty((tokens, heads, dim), dtype=x.dtype, device=x.device)
        else:
            _check(x.device, out=out)
            if out.shape != x.shape:
                raise ValueError("out must have the shape of x")
        os = _heads("out", out, tokens, dim, x.dtype)
        if tokens and heads:
            d = _ffi.RotaryDesc(_DTYPES[x.dtype], tokens, heads, dim, rotated, bool(interleaved), bool(inverse), wide, *xs, *os, gain)
            _ffi.check(_ffi.lib().disco_op_rotary(C.byref(d), x.data_ptr(), positions.data_ptr(), inv_freq.data_ptr(), out.data_ptr(), stream))
    return out


def cache_append(q, k, v, k_cache, v_cache, page_table, lens, cu_new, inv_freq=None, gain=1.0, interleaved=False, positions=None, q_out=None):
    """The new tokens' keys and values are written into their pages, keys (and queries, which are returned) turned by their positions on the
    way.  `lens` counts the new tokens already; `positions` replaces a token's place in its sequence as the angle's position; inv_freq=None turns
    nothing; q=None has no queries.  q_out may be q."""
    _check(k.device, k=k, v=v, k_cache=k_cache, v_cache=v_cache, page_table=page_table, lens=lens, cu_new=cu_new)
    c = _cache(k_cache, v_cache, page_table, False)
    _ints((c.rows, c.table_width), page_table=page_table)
    _ints((c.rows,), lens=lens)
    _ints((c.rows + 1,), cu_new=cu_new)
    tokens = k.shape[0]
    ks, vs = _heads("k", k, tokens, c.dim, k_cache.dtype), _heads("v", v, tokens, c.dim, k_cache.dtype)
    if k.shape[1] != c.kv_heads or v.shape[1] != c.kv_heads:
        raise ValueError("k and v must have the cache's %d heads" % c.kv_heads)
    rotated, wide = 0, 0
    if inv_freq is not None:
        _check(k.device, inv_freq=inv_freq)
        rotated = _frequencies(inv_freq)
    if positions is not None:
        _check(k.device, positions=positions)
        wide = _positions(positions, tokens)
    with _on(k.device) as stream:
        qs = os = (0, 0)
        q_heads = 0
        if q is not None:
            _check(k.device, q=q)
            qs = _heads("q", q, tokens, c.dim, k_cache.dtype)
            q_heads = q.shape[1]
            if q_out is None:
                q_out = torch.empty((tokens, q_heads, c.dim), dtype=q.dtype, device=q.device)
            else:
                _check(k.device, q_out=q_out)
                if q_out.shape != q.shape:
                    raise ValueError("q_out must have the shape of q")
            os = _heads("q_out", q_out, tokens, c.dim, k_cache.dtype)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if tokens:
            a = _ffi.AppendDesc(tokens, q_heads, rotated, bool(interleaved), wide, *qs, *ks, *vs, *os, gain)
            _ffi.check(_ffi.lib().disco_op_cache_append(
                C.byref(c), C.byref(a), q.data_ptr() if q_heads else None, k.data_ptr(), v.data_ptr(), page_table.data_ptr(), lens.data_ptr(),
                cu_new.data_ptr(), None if positions is None else positions.data_ptr(), None if inv_freq is None else inv_freq.data_ptr(),
                q_out.data_ptr() if q_heads else None, stream))
    return q_out


def cache_attention(q, k_cache, v_cache, page_table, lens, cu_new, causal=True, window=0, scale=None, max_new=None, max_len=None,
                    return_lse=False, out=None):
    """softmax(scale q k^T) v of every new token (tokens, q_heads, dim) over its sequence's cache, the new tokens among it (`lens` counts
    them).  Query head h reads key head h // (q_heads // kv_heads).  causal: the token at position p sees keys up to p, with `window` > 0 the last
    `window` of them; else the whole sequence.  A token that sees nothing gets zeros.  scale: 1 / sqrt(dim).

    max_new, max_len: what the caller knows of the largest number of new tokens and the largest length; they size launches and
    workspace, a sequence beyond them still comes out right.  return_lse: also the logarithm of the softmax's sum, (tokens, q_heads)
    fp32.  Rows behind cu_new[-1] are left as they are in a given `out` (and lse)."""
    _check(q.device, q=q, k_cache=k_cache, v_cache=v_cache, page_table=page_table, lens=lens, cu_new=cu_new)
    c = _cache(k_cache, v_cache, page_table, False)
    _ints((c.rows, c.table_width), page_table=page_table)
    _ints((c.rows,), lens=lens)
    _ints((c.rows + 1,), cu_new=cu_new)
    tokens, q_heads = q.shape[0], q.shape[1]
    qs = _heads("q", q, tokens, c.dim, k_cache.dtype)
    with _on(q.device) as stream:
        if out is None:
            out = torch.empty((tokens, q_heads, c.dim), dtype=q.dtype, device=q.device)
        else:
            _check(q.device, out=out)
            if out.shape != q.shape:
                raise ValueError("out must have the shape of q")
        os = _heads("out", out, tokens, c.dim, k_cache.dtype)
        lse = torch.empty((tokens, q_heads), dtype=torch.float32, device=q.device) if return_lse else None
        a = _ffi.AttentionDesc(tokens, q_heads, bool(causal), window, tokens if max_new is None else max_new, 0 if max_len is None else max_len,
                               1 / math.sqrt(c.dim) if scale is None else scale, *qs, *os)
        lib, need = _ffi.lib(), C.c_size_t()
        _ffi.check(lib.disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(need)))
        ws = torch.empty(need.value, dtype=torch.uint8, device=q.device) if need.value else None
        _ffi.check(lib.disco_op_cache_attention(C.byref(c), C.byref(a), q.data_ptr(), page_table.data_ptr(), lens.data_ptr(), cu_new.data_ptr(),
                                               out.data_ptr(), lse.data_ptr() if return_lse else None, ws.data_ptr() if need.value else None,
                                               need.value, stream))
    return (out, lse) if return_lse else out


def _state(page_table, pages):
    """New buffers for a table, its lengths, the pages' counts and info, in one allocation."""
    rows, width = page_table.shape
    flat = torch.empty(rows * width + rows + pages + 4, dtype=torch.int32, device=page_table.device)
    table, lens, refs, info = flat.split((rows * width, rows, pages, 4))
    return table.view(rows, width), lens, refs, info


def cache_reserve(page_table, lens, refs, cu_new, page):
    """Pages for the new tokens of every row: (page_table, lens, refs, info) with them.  The lowest free pages are taken, rows ascending.
    info (4,) int32: free pages afterwards; pages that were missing - then the state returned is the old one -; lengths out of range; 0."""
    _check(page_table.device, page_table=page_table, lens=lens, refs=refs, cu_new=cu_new)
    if page_table.dim() != 2 or refs.dim() != 1:
        raise ValueError("page_table must be (rows, width), refs (pages,)")
    rows, width = page_table.shape
    _ints((rows, width), page_table=page_table)
    _ints((rows,), lens=lens)
    _ints((rows + 1,), cu_new=cu_new)
    _ints(refs.shape, refs=refs)
    with _on(page_table.device) as stream:
        new = _state(page_table, refs.numel())
        _ffi.check(_ffi.lib().disco_op_cache_reserve(rows, width, refs.numel(), page, page_table.data_ptr(), lens.data_ptr(), refs.data_ptr(),
                                                    cu_new.data_ptr(), *[t.data_ptr() for t in new], stream))
    return new


def _page_call(k_cache, v_cache, page_table, **ints):
    _check(k_cache.device, k_cache=k_cache, v_cache=v_cache, page_table=page_table, **ints)
    c = _cache(k_cache, v_cache, page_table, True)
    _ints((c.rows, c.table_width), page_table=page_table)
    _ints((c.rows,), **ints)
    return c


def cache_select(page_table, lens, parents, k_cache, v_cache):
    """Row r becomes what row parents[r] was, -1: empty; forks, reorders and frees rows in one call: (page_table, lens, refs, info).  Rows of one
    parent share its full pages; of a last page that is not full one row keeps the original and the others get copies, in all layers.
    info (4,) int32: free pages afterwards; pages that were missing - then the state returned is the old one -; entries out of range; pages copied."""
    c = _page_call(k_cache, v_cache, page_table, lens=lens, parents=parents)
    with _on(k_cache.device) as stream:
        new = _state(page_table, c.pages)
        lib = _ffi.lib()
        ws = torch.empty(lib.disco_op_cache_pages_workspace_bytes(c.rows, c.pages), dtype=torch.uint8, device=k_cache.device)
        _ffi.check(lib.disco_op_cache_select(C.byref(c), page_table.data_ptr(), lens.data_ptr(), parents.data_ptr(), *[t.data_ptr() for t in new],
                                            ws.data_ptr(), ws.numel(), stream))
    return new


def cache_compact(page_table, lens, k_cache, v_cache):
    """The n pages in use move to 0 .. n - 1, in all layers: (page_table, refs, info).  info as cache_select's."""
    c = _page_call(k_cache, v_cache, page_table, lens=lens)
    with _on(k_cache.device) as stream:
        table, _, refs, info = _state(page_table, c.pages)
        lib = _ffi.lib()
        ws = torch.empty(lib.disco_op_cache_pages_workspace_bytes(c.rows, c.pages), dtype=torch.uint8, device=k_cache.device)
        _ffi.check(lib.disco_op_cache_compact(C.byref(c), page_table.data_ptr(), lens.data_ptr(), table.data_ptr(), refs.data_ptr(), info.data_ptr(),
                                             ws.data_ptr(), ws.numel(), stream))
    return table, refs, info


def cache_copy_pages(k_cache, v_cache, src, dst):
    """Page src[i] is copied to page dst[i], in all layers (src, dst int32).  No page of dst may be among src; pairs out of range are skipped."""
    _check(k_cache.device, k_cache=k_cache, v_cache=v_cache, src=src, dst=dst)
    c = _cache(k_cache, v_cache, src[None], True)
    if src.dim() != 1:
        raise ValueError("src must be (count,)")
    _ints(src.shape, src=src, dst=dst)
    count = src.numel()
    if count:
        c.rows = c.table_width = 1
        with _on(k_cache.device) as stream:
            _ffi.check(_ffi.lib().disco_op_cache_copy_pages(C.byref(c), src.data_ptr(), dst.data_ptr(), count, stream))

"""The paged-cache operators without a GPU: the rotary frequencies, the entry points' refusals, the binding's structs."""
import ctypes as C
import math
import os
import re

import pytest
import torch

from disentangledcolorization_amd import _ffi, paged

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.fixture(scope="module")
def lib():
    from disentangledcolorization_amd.build import build
    build(verbose=False)
    return _ffi.lib()


@pytest.mark.parametrize("dim", [2, 4, 8, 64, 96, 128])
def test_frequencies(lib, dim):
    i = torch.arange(dim // 2, dtype=torch.float64)
    f = 10000.0 ** (-2 * i / dim)
    near = lambda a, b: torch.allclose(a, b, rtol=1e-14, atol=0)
    assert near(paged.rotary_frequencies(dim, device="cpu"), f)
    assert near(paged.rotary_frequencies(dim, base=5e5, device="cpu"), 5e5 ** (-2 * i / dim))
    assert near(paged.rotary_frequencies(dim, scaling="linear", factor=4, device="cpu"), f / 4)
    if dim > 2:       # the slowest pair is stretched by the factor, the fastest kept
        g = paged.rotary_frequencies(dim, scaling="ntk", factor=4, device="cpu")
        assert g[0] == 1 and abs(g[-1] * 4 / f[-1] - 1) < 1e-13
    g = paged.rotary_frequencies(dim, scaling="parts", factor=8, original_length=4096, low=1, high=32, device="cpu")
    turns = 4096 * f / (2 * math.pi)
    for x, y, r in zip(g.tolist(), f.tolist(), turns.tolist()):
        if r >= 32:
            assert abs(x / y - 1) < 1e-14         # (two pow()s: an ulp each, and 9.2 = ln 10^4 roundings of the exponent: 1.4e-15)
        elif r <= 1:
            assert abs(x * 8 / y - 1) < 1e-14
        else:
            assert y / 8 < x < y
            assert abs(x - ((r - 1) / 31 * y + (32 - r) / 31 * y / 8)) < 1e-14 * y


@pytest.mark.parametrize("kw", [dict(dim=3), dict(dim=0), dict(dim=-2), dict(dim=8, base=1.0), dict(dim=8, base=math.nan), dict(dim=8, scaling="linear", factor=0.0),
                                dict(dim=8, scaling="linear", factor=math.inf), dict(dim=2, scaling="ntk", factor=2.0),
                                dict(dim=8, scaling="parts", factor=2.0, low=4.0, high=4.0), dict(dim=8, scaling="parts", factor=2.0, original_length=0)])
def test_frequencies_are_refused(lib, kw):
    with pytest.raises(_ffi.DiscoError, match="rotary_frequencies"):
        paged.rotary_frequencies(device="cpu", **kw)
    with pytest.raises(ValueError):
        paged.rotary_frequencies(8, scaling="other", device="cpu")


def cache(**kw):
    d = dict(dtype=_ffi.BF16, layers=1, pages=8, kv_heads=2, page_size=16, dim=64, rows=2, table_width=4, layer_stride=0, page_stride=2 * 16 * 64,
             head_stride=16 * 64, slot_stride=64, d_k=1 << 20, d_v=1 << 20)
    d.update(kw)
    return _ffi.CacheDesc(*[d[n] for n, _ in _ffi.CacheDesc._fields_])


BAD_CACHES = [dict(dtype=_ffi.F32), dict(dtype=7), dict(layers=0), dict(pages=0), dict(kv_heads=0), dict(page_size=24), dict(page_size=0), dict(page_size=-16),
              dict(dim=4), dict(dim=60), dict(dim=264), dict(rows=0), dict(rows=16385), dict(table_width=0), dict(table_width=1 << 27), dict(rows=16384, table_width=1 << 18, page_size=1), dict(d_k=None),
              dict(d_v=None), dict(d_k=(1 << 20) + 8), dict(page_stride=2044), dict(head_stride=1), dict(slot_stride=68), dict(page_stride=1 << 60)]


@pytest.mark.parametrize("kw", BAD_CACHES)
def test_bad_caches_are_refused(lib, kw):
    """No entry point gets as far as a launch with one (there is no GPU here: a launch would come back as DISCO_EHIP)."""
    c, p = cache(**kw), C.c_void_p(1 << 20)
    a = _ffi.AttentionDesc(4, 4, 1, 0, 0, 0, 0.125, 256, 64, 256, 64)
    d = _ffi.AppendDesc(4, 4, 64, 0, 0, 256, 64, 128, 64, 128, 64, 256, 64, 1.0)
    n = C.c_size_t()
    for rc in (lib.disco_op_cache_attention(C.byref(c), C.byref(a), p, p, p, p, p, None, p, 1 << 40, None),
               lib.disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)),
               lib.disco_op_cache_append(C.byref(c), C.byref(d), p, p, p, p, p, p, None, p, p, None),
               lib.disco_op_cache_select(C.byref(c), p, p, p, C.c_void_p(2 << 20), C.c_void_p(2 << 20), p, p, p, 1 << 40, None),
               lib.disco_op_cache_compact(C.byref(c), p, p, C.c_void_p(2 << 20), p, p, p, 1 << 40, None),
               lib.disco_op_cache_copy_pages(C.byref(c), p, p, 2, None)):
        assert rc in (-1, -2) and lib.disco_last_error().startswith(b"cache_"), (rc, lib.disco_last_error())


def test_pages_whose_pieces_an_int_does_not_count_are_refused(lib):
    """A head of a page is copied in pieces of 16 bytes, counted in 32 bits: where they do not fit nothing may be reported as copied."""
    p, o = C.c_void_p(1 << 20), C.c_void_p(2 << 20)
    need = lib.disco_op_cache_pages_workspace_bytes(2, 8)
    for page_size, dim in ((1 << 26, 256), (1 << 28, 64), (1 << 30, 16)):
        c = cache(page_size=page_size, dim=dim, table_width=1)
        for rc in (lib.disco_op_cache_select(C.byref(c), p, p, p, o, o, o, o, p, need, None), lib.disco_op_cache_compact(C.byref(c), p, p, o, o, o, p, need, None),
                   lib.disco_op_cache_copy_pages(C.byref(c), p, p, 1, None)):
            assert rc == -2 and b"pieces" in lib.disco_last_error()
    c = cache(page_size=1 << 25, dim=256, table_width=1)      # (just below: as far as the workspace's check)
    assert lib.disco_op_cache_select(C.byref(c), p, p, p, o, o, o, o, p, 0, None) == -6


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(q_heads=0), dict(q_heads=3), dict(window=-1), dict(window=4, causal=0), dict(max_new=-1), dict(max_len=-1),
                                dict(scale=math.nan), dict(scale=math.inf), dict(q_token=4), dict(out_head=1 << 60), dict(tokens=1 << 30)])
def test_bad_attention_is_refused(lib, kw):
    d = dict(tokens=4, q_heads=4, causal=1, window=0, max_new=0, max_len=0, scale=0.125, q_token=256, q_head=64, out_token=256, out_head=64)
    d.update(kw)
    a, c, p, n = _ffi.AttentionDesc(*[d[f] for f, _ in _ffi.AttentionDesc._fields_]), cache(), C.c_void_p(1 << 20), C.c_size_t()
    assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), p, p, p, p, p, None, p, 1 << 40, None) in (-1, -2)
    assert lib.disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)) in (-1, -2)


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(q_heads=3), dict(window=-1), dict(scale=math.nan), dict(q_token=4)])
def test_bad_precise_attention_is_refused(lib, kw):
    d = dict(tokens=4, q_heads=4, causal=1, window=0, max_new=0, max_len=0, scale=0.125, q_token=256, q_head=64, out_token=256, out_head=64)
    d.update(kw)
    a, c, p = _ffi.AttentionDesc(*[d[f] for f, _ in _ffi.AttentionDesc._fields_]), cache(), C.c_void_p(1 << 20)
    assert lib.disco_op_cache_attention_precise(C.byref(c), C.byref(a), p, p, p, p, p, None, p, 1 << 40, None) in (-1, -2)
    assert lib.disco_op_cache_attention_precise(None, C.byref(a), p, p, p, p, p, None, p, 1 << 40, None) == -1


def test_more_heads_than_units_can_be_counted_for(lib):
    c, p, n = cache(kv_heads=1025), C.c_void_p(1 << 20), C.c_size_t()
    a = _ffi.AttentionDesc(4, 1025, 1, 0, 0, 0, 0.125, 1025 * 64, 64, 1025 * 64, 64)
    assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), p, p, p, p, p, None, p, 1 << 40, None) == -2
    assert lib.disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)) == -2
    c.kv_heads = a.q_heads = 1024
    assert lib.disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)) == 0


def test_sizes_that_an_int32_does_not_hold_are_refused():
    """None of them may arrive as what is left of it in 32 bits (meta tensors: sizes without memory)."""
    far, meta = (1 << 32) + 4, dict(device="meta", dtype=torch.int32)
    with pytest.raises(ValueError, match="2\\^31"):
        paged._three("x", torch.empty(far, 1, 8, device="meta"))
    kv = torch.empty(far, 1, 16, 8, device="meta", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="2\\^31"):
        paged._cache(kv, kv, torch.empty(1, 2, **meta))
    kv = torch.empty(4, 1, 16, 8, device="meta", dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="2\\^31"):
        paged._cache(kv, kv, torch.empty(1, far, **meta))
    assert [paged._bound(n) for n in (-far, -1, 0, 7, far)] == [-1, -1, 0, 7, (1 << 31) - 1]


def test_attention_in_place_is_refused(lib):
    """Queries are read again where a result is not finite: they must still be there."""
    c, p, o = cache(), C.c_void_p(1 << 20), C.c_void_p(2 << 20)
    a = _ffi.AttentionDesc(4, 4, 1, 0, 0, 0, 0.125, 256, 64, 256, 64)
    assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), p, p, p, p, p, None, p, 1 << 40, None) == -1
    assert b"may not be q" in lib.disco_last_error()


@pytest.mark.parametrize("shape", [(1, 2, 16, 8), (4, 1, 16, 8), (4, 2, 1, 8), (1, 1, 1, 8), (1, 4, 2, 16, 8), (3, 1, 1, 4, 8)])
def test_the_stride_of_a_cache_axis_of_one_does_not_matter(shape):
    """Keys and values cut from different places are alike where the axes that have a stride have the same."""
    strides = torch.empty(shape, device="meta").stride()
    views = [torch.empty(1 << 14, device="meta", dtype=torch.bfloat16).as_strided(shape, tuple(st if n > 1 else odd for n, st in zip(shape, strides))) for odd in (5, 129)]
    table = torch.empty(2, 2, device="meta", dtype=torch.int32)
    c = paged._cache(*views, table, layered=len(shape) == 5)
    got = [c.layer_stride, c.page_stride, c.head_stride, c.slot_stride][-len(shape) + 1:]
    assert got == [st if n > 1 else 0 for n, st in zip(shape[:-1], strides)]
    other = torch.empty(1 << 14, device="meta", dtype=torch.bfloat16).as_strided(shape, tuple(2 * st if n > 1 else st for n, st in zip(shape[:-1], strides)) + (1,))
    if any(n > 1 for n in shape[:-1]):
        with pytest.raises(ValueError, match="alike"):
            paged._cache(views[0], other, table, layered=len(shape) == 5)


def test_missing_arguments_and_workspaces_are_refused(lib):
    c, p, o = cache(), C.c_void_p(1 << 20), C.c_void_p(2 << 20)
    a = _ffi.AttentionDesc(4, 4, 1, 0, 0, 0, 0.125, 256, 64, 256, 64)
    full = [p, p, p, p, p]
    for i in range(5):
        args = full[:i] + [None] + full[i + 1:]
        assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), *args, None, p, 1 << 40, None) == -1
    assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), C.c_void_p((1 << 20) + 2), p, p, p, p, None, p, 1 << 40, None) == -1
    c.table_width, n = 1 << 16, C.c_size_t()                 # a long table: the keys are split, which takes a workspace
    assert lib.disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)) == 0
    if n.value:
        assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), *full, None, None, 0, None) == -6
        assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), *full, None, p, n.value - 1, None) == -6
        assert lib.disco_op_cache_attention(C.byref(c), C.byref(a), *full, None, C.c_void_p((1 << 20) + 8), n.value, None) == -6
    assert lib.disco_op_cache_attention(None, C.byref(a), *full, None, p, 1 << 40, None) == -1
    assert lib.disco_op_cache_attention(C.byref(c), None, *full, None, p, 1 << 40, None) == -1
    c = cache()
    need = lib.disco_op_cache_pages_workspace_bytes(2, 8)
    assert need > 0 and lib.disco_op_cache_pages_workspace_bytes(0, 8) == 0
    assert lib.disco_op_cache_select(C.byref(c), p, p, p, o, o, o, o, p, need - 1, None) == -6
    assert lib.disco_op_cache_compact(C.byref(c), p, p, o, o, o, p, need - 1, None) == -6
    assert lib.disco_op_cache_select(C.byref(c), p, p, p, p, o, o, o, p, need, None) == -1           # in place
    assert lib.disco_op_cache_compact(C.byref(c), p, p, p, o, o, p, need, None) == -1
    assert lib.disco_op_cache_reserve(2, 4, 8, 16, p, p, p, p, o, p, o, o, None) == -1
    assert lib.disco_op_cache_reserve(2, 4, 8, 12, p, p, p, p, o, o, o, o, None) == -2
    assert lib.disco_op_cache_copy_pages(C.byref(c), None, p, 1, None) == -1
    assert lib.disco_op_cache_copy_pages(C.byref(c), p, p, -1, None) == -2


@pytest.mark.parametrize("kw", [dict(dtype=9), dict(tokens=-1), dict(heads=0), dict(dim=0), dict(rotated=0), dict(rotated=3), dict(rotated=66), dict(dim=1026), dict(heads=1 << 17), dict(x_token=1 << 60),
                                dict(tokens=(1 << 30) + 1), dict(tokens=(1 << 31) - 1)])
def test_bad_rotations_are_refused(lib, kw):
    d = dict(dtype=_ffi.F32, tokens=4, heads=2, dim=64, rotated=64, interleaved=0, inverse=0, wide_positions=0, x_token=128, x_head=64, out_token=128,
             out_head=64, gain=1.0)
    d.update(kw)
    r, p = _ffi.RotaryDesc(*[d[f] for f, _ in _ffi.RotaryDesc._fields_]), C.c_void_p(1 << 20)
    assert lib.disco_op_rotary(C.byref(r), p, p, p, p, None) in (-1, -2)
    ok = _ffi.RotaryDesc(_ffi.F32, 4, 2, 64, 64, 0, 0, 0, 128, 64, 64, 256, 1.0)
    assert lib.disco_op_rotary(C.byref(ok), p, p, p, p, None) == -1          # in place with other strides
    assert lib.disco_op_rotary(None, p, p, p, p, None) == -1


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(q_heads=-1), dict(rotated=-2), dict(rotated=5), dict(rotated=66), dict(k_token=1 << 60), dict(tokens=(1 << 31) - 1)])
def test_bad_appends_are_refused(lib, kw):
    d = dict(tokens=4, q_heads=4, rotated=64, interleaved=0, wide_positions=0, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64,
             out_token=256, out_head=64, gain=1.0)
    d.update(kw)
    a, c, p = _ffi.AppendDesc(*[d[f] for f, _ in _ffi.AppendDesc._fields_]), cache(), C.c_void_p(1 << 20)
    assert lib.disco_op_cache_append(C.byref(c), C.byref(a), p, p, p, p, p, p, None, p, p, None) in (-1, -2)


@pytest.mark.parametrize("kw", [dict(tokens=-1), dict(q_heads=-1), dict(rotated=5), dict(k_token=1 << 60)])
def test_bad_appends_behind_a_reserve_are_refused(lib, kw):
    """With and without the reserve's info the same checks."""
    d = dict(tokens=4, q_heads=4, rotated=64, interleaved=0, wide_positions=0, q_token=256, q_head=64, k_token=128, k_head=64, v_token=128, v_head=64,
             out_token=256, out_head=64, gain=1.0)
    d.update(kw)
    a, c, p = _ffi.AppendDesc(*[d[f] for f, _ in _ffi.AppendDesc._fields_]), cache(), C.c_void_p(1 << 20)
    for info in (None, p):
        assert lib.disco_op_cache_append_reserved(C.byref(c), C.byref(a), p, p, p, p, p, p, None, p, p, info, None) in (-1, -2)
        assert lib.disco_op_cache_append_reserved(None, C.byref(a), p, p, p, p, p, p, None, p, p, info, None) == -1


def test_cpu_tensors_are_refused():
    t = torch.zeros(2, 2, 64)
    with pytest.raises(_ffi.DiscoError, match="no CPU fallback"):
        paged.rotary(t, torch.zeros(2, dtype=torch.int64), torch.ones(32, dtype=torch.float64))
    kv, i = torch.zeros(4, 2, 16, 64, dtype=torch.bfloat16), torch.zeros(2, 2, dtype=torch.int32)
    for call in (lambda: paged.cache_attention(t, kv, kv, i, i[0], i[0]), lambda: paged.cache_append(t, t, t, kv, kv, i, i[0], i[0]),
                 lambda: paged.cache_select(i, i[0], i[0], kv, kv), lambda: paged.cache_compact(i, i[0], kv, kv),
                 lambda: paged.cache_reserve(i, i[0], i[0], i[0], 16), lambda: paged.cache_copy_pages(kv, kv, i[0], i[0])):
        with pytest.raises(_ffi.DiscoError, match="no CPU fallback"):
            call()


def test_structs_mirror_the_header():
    text = re.sub(r"/\*.*?\*/", "", open(os.path.join(REPO, "include", "disco_hip.h")).read(), flags=re.S)
    for cname, py in (("disco_cache_desc", _ffi.CacheDesc), ("disco_rotary_desc", _ffi.RotaryDesc), ("disco_append_desc", _ffi.AppendDesc),
                      ("disco_attention_desc", _ffi.AttentionDesc)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (cname, cname), text, re.S).group(1)
        kinds = {"int32_t": C.c_int32, "int64_t": C.c_int64, "float": C.c_float, "double": C.c_double, "void": C.c_void_p}
        want = [(n.strip().lstrip("*"), kinds[d.split()[0]]) for d in map(str.strip, body.split(";")) if d for n in d.split(None, 1)[1].split(",")]
        assert want == list(py._fields_)


def test_the_forwards_records_do_not_go_stale_with_the_paged_cache(tmp_path, monkeypatch):
    """bench.source_hash keys counters of the forward: a change of these operators, or of their section of the header, leaves it; one of the forward's files does not."""
    import shutil

    import bench
    from disentangledcolorization_amd import build as B
    csrc = tmp_path / "pkg" / "csrc"
    shutil.copytree(B.CSRC, csrc, ignore=shutil.ignore_patterns("build"))
    shutil.copytree(os.path.join(REPO, "include"), tmp_path / "include")
    was = bench.source_hash()
    monkeypatch.setattr(B, "CSRC", str(csrc))
    assert bench.source_hash() == was
    for name in (*B.PAGED_SOURCES, *B.PAGED_HEADERS):
        with open(csrc / name, "a") as f:
            f.write("// more\n")
    header = tmp_path / "include" / "disco_hip.h"
    text = header.read_text()
    header.write_text(text.replace("typedef struct disco_cache_desc {", "/* more */\ntypedef struct disco_cache_desc {"))
    assert header.read_text() != text and bench.source_hash() == was
    header.write_text(text.replace("#pragma once", "#pragma once\n\n", 1) if "#pragma once" in text else "\n" + text)
    assert bench.source_hash() != was
    header.write_text(text)
    for name in ("conv_mx_kernel.h", "tokens.hip", "util.cpp"):
        with open(csrc / name, "a") as f:
            f.write("// more\n")
        assert bench.source_hash() != was
        shutil.copy(os.path.join(REPO, "disentangledcolorization_amd", "csrc", name), csrc / name)
    assert bench.source_hash() == was

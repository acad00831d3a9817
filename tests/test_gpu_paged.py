"""-m gpu: the paged-cache operators (disentangledcolorization_amd/paged.py) against plain 64-bit implementations (tests/paged_reference.py).

Tolerances count roundings, eps / 2 each (eps of the tensors' type):
  rotary     one rounding of the result, and in fp32 the cosine and sine (3e-8 of the series, 2^-32 of a turn, 2^-24), the gain's rounding and three
             operations: 8 * 2^-24 of |a| + |b| together; far positions add their angle's 64-bit rounding.
  attention  one rounding of the result; the probabilities enter the second product rounded to the cache's type, so half a step of the weighted
             |v|; the scores' fp32 errors (bounded by the reference from |q| |k|) and the exponential's change every weight by a factor, twice (numerator
             and sum); fp16 probabilities below 2^-14 of the row's largest are off by at most 2^-25 of it each.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

import paged_reference as R  # noqa: E402
from disentangledcolorization_amd import _ffi, paged  # noqa: E402

DEV = "cuda:0"
BF, HF, FL = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module", autouse=True)
def device():
    assert torch.cuda.is_available(), "GPU tests need a HIP device"
    _ffi.lib()


def gen(seed):
    return torch.Generator().manual_seed(seed)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def half(dtype):
    return torch.finfo(dtype).eps / 2


# ---- rotary -----------------------------------------------------------------------------------------------------------------------------

def close_turned(got, x, positions, f, gain, interleaved, inverse=False):
    want, size = R.turned(x, positions, f, gain, interleaved, inverse)
    angle = positions.double().abs().max().item() * f.double().max().item()
    tol = half(x.dtype) * want.abs() + (8 * 2.0 ** -24 + angle * 2.0 ** -51) * size + torch.finfo(x.dtype).smallest_normal
    off = (got.double().cpu() - want).abs()
    assert (off <= tol).all(), (off - tol).max().item()


ROTARY = [
    # tokens, heads, dim, rotated
    (1, 1, 2, 2), (1, 5, 64, 64), (3, 40, 128, 128), (7, 3, 80, 32), (33, 4, 96, 50), (5, 2, 65, 6), (700, 6, 64, 62), (2, 7, 256, 256), (9, 3, 24, 8), (4100, 2, 40, 40),
    (2, 300, 8, 4), (1, 2, 512, 500),
]


@pytest.mark.parametrize("dtype", [BF, HF, FL])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("shape", ROTARY)
def test_rotary(shape, interleaved, dtype):
    tokens, heads, dim, rotated = shape
    x = torch.randn(tokens, heads, dim, generator=gen(tokens + dim)).to(dtype).to(DEV)
    f = paged.rotary_frequencies(rotated)
    positions = torch.randint(0, 1 << 20, (tokens,), generator=gen(3)).to(DEV)
    got = paged.rotary(x, positions, f, gain=1.25, interleaved=interleaved)
    assert got.dtype == dtype and got.is_contiguous()
    close_turned(got, x, positions, f, 1.25, interleaved)
    assert torch.equal(got[..., rotated:], x[..., rotated:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_rotary_places_and_strides(interleaved):
    """A slice of a joined projection, every alignment of its first element, another order of the axes, in place, int32 positions, negative and far ones."""
    joined = torch.randn(19, 9, 72, generator=gen(1)).half().to(DEV)
    f = paged.rotary_frequencies(32)
    positions = torch.arange(-9, 10, device=DEV)
    for at in (0, 1, 2, 3, 4, 8):
        x = joined[:, 2:7, at:at + 64]
        close_turned(paged.rotary(x, positions, f, interleaved=interleaved), x, positions, f, 1.0, interleaved)
    x = joined[:, :, :64].transpose(0, 1).contiguous().transpose(0, 1)
    got = paged.rotary(x, positions.int(), f, interleaved=interleaved)
    close_turned(got, x, positions, f, 1.0, interleaved)
    for far in (2 ** 31 - 1, 2 ** 40):
        p = far - torch.arange(19, device=DEV)
        close_turned(paged.rotary(x, p, f, interleaved=interleaved), x, p, f, 1.0, interleaved)
    y, before = joined.clone(), joined[:, 1:4].clone()
    out = y[:, 1:4, 2:66]
    assert paged.rotary(out, positions, f, interleaved=interleaved, out=out) is out
    close_turned(out, before[..., 2:66], positions, f, 1.0, interleaved)
    y[:, 1:4, 2:66] = joined[:, 1:4, 2:66]
    assert torch.equal(y, joined)                       # nothing else was touched


def test_far_positions_keep_their_angles():
    """fp32 against angles from whole numbers: position * frequency / 2 pi as fractions, with pi to 60 digits.  The tolerance has no part that grows with the position."""
    from fractions import Fraction
    pi = Fraction(314159265358979323846264338327950288419716939937510582097494, 10 ** 59)
    f = paged.rotary_frequencies(64, base=5e5)
    positions = [s * (far - i * 7919) for far in (1 << 20, 1 << 31, 1 << 40, 1 << 52) for i in range(20) for s in (1, -1)]
    x = torch.randn(len(positions), 2, 64, generator=gen(4)).to(DEV)
    got = paged.rotary(x, torch.tensor(positions, device=DEV), f).double().cpu()
    turn = torch.tensor([[float((p * Fraction(w) / (2 * pi)) % 1) for w in f.tolist()] for p in positions], dtype=torch.float64)[:, None]
    c, s, a, b = (2 * math.pi * turn).cos(), (2 * math.pi * turn).sin(), x[..., :32].double().cpu(), x[..., 32:].double().cpu()
    size = torch.cat((a.abs() + b.abs(),) * 2, -1)
    assert ((got - torch.cat((a * c - b * s, a * s + b * c), -1)).abs() <= (8 + 1) * 2.0 ** -24 * size).all()


def test_an_axis_of_one_has_any_stride():
    """A view's stride of an axis of one is what it was cut from: nothing may be refused, or read, because of it."""
    f, p = paged.rotary_frequencies(64), torch.tensor([77], device=DEV)
    x = torch.randn(1, 3, 64, generator=gen(0)).to(BF).to(DEV)
    odd = x.as_strided((1, 3, 64), (5, 64, 1))
    want = paged.rotary(x, p, f)
    assert torch.equal(paged.rotary(odd, p, f), want)
    y = x.clone()
    assert torch.equal(paged.rotary(y.as_strided((1, 3, 64), (7, 64, 1)), p, f, out=y), want)
    s = Served([50], [1], 1, 3, 64, 16, BF)
    out = torch.empty_like(s.q)
    paged.cache_attention(s.q.as_strided((1, 3, 64), (3, 64, 1)), *s.args(), out=out.as_strided((1, 3, 64), (1, 64, 1)))
    assert torch.equal(out, paged.cache_attention(s.q, *s.args()))


def test_a_cache_axis_of_one_has_any_stride():
    s = Served([50], [3], 1, 4, 64, 16, BF)
    want = paged.cache_attention(s.q, *s.args())
    k = torch.empty(s.pool, 3, 16, 64, dtype=BF, device=DEV)[:, 1:2]
    v = torch.empty(s.pool, 16, 3, 64, dtype=BF, device=DEV).transpose(1, 2)[:, :1]
    assert k.stride() != v.stride()
    k.copy_(s.k)
    with pytest.raises(ValueError, match="alike"):
        paged.cache_attention(s.q, k, v, *s.args()[2:])
    v = k.new_empty(s.pool, 3, 16, 64)[:, 1:2].as_strided(k.shape, (k.stride(0), 7, 64, 1))
    v.copy_(s.v)
    assert torch.equal(paged.cache_attention(s.q, k, v, *s.args()[2:]), want)


def test_rotary_there_and_back():
    """inverse is the transposed rotation: <y, rot(x)> = <rot'(y), x>, and without a gain it undoes the rotation."""
    x, y = (torch.randn(50, 3, 48, generator=gen(s)).to(DEV) for s in (1, 2))
    f, p = paged.rotary_frequencies(40, scaling="ntk", factor=4), torch.arange(50, device=DEV) * 1000
    for inter in (False, True):
        close_turned(paged.rotary(x, p, f, 0.9, inter, inverse=True), x, p, f, 0.9, inter, True)
        there = paged.rotary(x, p, f, 0.9, inter).double()
        back = paged.rotary(y, p, f, 0.9, inter, inverse=True).double()
        a, b = (there * y).sum(), (back * x).sum()
        assert abs(a - b) <= 16 * 2.0 ** -24 * (there.abs() * y.abs() + back.abs() * x.abs()).sum()
        z = paged.rotary(paged.rotary(x, p, f, interleaved=inter), p, f, interleaved=inter, inverse=True)
        assert (z - x).abs().max() <= 4 * 16 * 2.0 ** -24 * x.abs().max()


def test_rotary_of_nothing_and_refusals():
    f, p = paged.rotary_frequencies(8), torch.zeros(3, dtype=torch.int64, device=DEV)
    assert paged.rotary(torch.zeros(0, 4, 8, device=DEV), p[:0], f).shape == (0, 4, 8)
    assert paged.rotary(torch.zeros(3, 0, 8, device=DEV), p, f).shape == (3, 0, 8)
    x = torch.zeros(3, 2, 8, device=DEV)
    for bad in (lambda: paged.rotary(x.double(), p, f), lambda: paged.rotary(x[0], p, f), lambda: paged.rotary(x, p[:2], f), lambda: paged.rotary(x, p.float(), f),
                lambda: paged.rotary(x, p, f.float()), lambda: paged.rotary(x.transpose(1, 2), p, f), lambda: paged.rotary(x, p, f, out=x[:2]),
                lambda: paged.rotary(x, p, f, out=x.half()), lambda: paged.rotary(x, p.cpu(), f)):
        with pytest.raises((ValueError, _ffi.DiscoError)):
            bad()
    with pytest.raises(_ffi.DiscoError, match="rotated"):
        paged.rotary(x, p, paged.rotary_frequencies(10))
    with pytest.raises(NotImplementedError, match="inference only"):
        paged.rotary(x.requires_grad_(), p, f)
    with torch.no_grad():
        paged.rotary(x, p, f)


# ---- a cache to work on -----------------------------------------------------------------------------------------------------------------

class Served:
    """Sequences of given lengths whose pages lie anywhere in the pool; slots that no token uses hold NaN."""

    def __init__(self, lens, new, kv_heads=2, group=2, dim=64, page=16, dtype=BF, seed=0, spare=2, slot_major=False, q_scale=1.0, layers=None):
        g, rows = gen(seed), len(lens)
        used = [-(-n // page) for n in lens]
        pool, width = sum(used) + spare, max(max(used), 1) + 1
        order = torch.randperm(pool, generator=g).tolist()
        table, at = torch.full((rows, width), -1, dtype=torch.int32), 0
        for b, u in enumerate(used):
            table[b, :u] = torch.tensor(order[at:at + u], dtype=torch.int32)
            at += u
        shape = (pool, page, kv_heads, dim) if slot_major else (pool, kv_heads, page, dim)
        shape = shape if layers is None else (layers, *shape)
        self.k, self.v = (torch.randn(shape, generator=g).to(dtype) for _ in range(2))
        if slot_major:
            self.k, self.v = self.k.transpose(-3, -2), self.v.transpose(-3, -2)
        filled = torch.zeros(pool, page, dtype=torch.bool)
        for b, n in enumerate(lens):
            for i in range(used[b]):
                filled[table[b, i], :max(0, min(page, n - i * page))] = True
        for c in (self.k, self.v):
            c.transpose(-3, -2)[..., ~filled, :, :] = math.nan
        self.q = (torch.randn(sum(new), kv_heads * group, dim, generator=g) * q_scale).to(dtype)
        self.lens, self.cu = torch.tensor(lens, dtype=torch.int32), torch.tensor([sum(new[:i]) for i in range(rows + 1)], dtype=torch.int32)
        self.table, self.page, self.dtype, self.used, self.pool = table, page, dtype, used, pool
        for n in ("k", "v", "q", "lens", "cu", "table"):
            t = getattr(self, n)
            setattr(self, n, t.to(DEV) if t.dim() < 4 or not slot_major else t.transpose(-3, -2).to(DEV).transpose(-3, -2))

    def args(self):
        return self.k, self.v, self.table, self.lens, self.cu

    def refs(self):
        refs = torch.zeros(self.pool, dtype=torch.int32)
        for b, u in enumerate(self.used):
            for p in self.table[b, :u].tolist():
                refs[p] += 1
        return refs.to(DEV)


def close_attended(got, lse, q, k, v, table, lens, cu, **kw):
    want, size, want_lse, off = R.attended(q, k, v, table, lens, cu, **kw)
    n, dtype = want.shape[0], q.dtype
    got, lse = got[:n].double().cpu(), lse[:n].double().cpu()
    factor = 2 * off[..., None] + 2.0 ** -20
    tiny = int(lens.max()) * 2.0 ** -25 * v.double().nan_to_num(0, 0, 0).abs().max().item() if dtype == HF else 0.0
    tol = half(dtype) * want.abs() + (half(dtype) + factor) * size + tiny + torch.finfo(dtype).smallest_normal
    same = (got == want) | (got.isnan() & want.isnan())
    assert (same | ((got - want).abs() <= tol)).all(), ((got - want).abs() - tol).nan_to_num(0).max().item()
    same = (lse == want_lse) | (lse.isnan() & want_lse.isnan())
    assert (same | ((lse - want_lse).abs() <= off + 2.0 ** -22 * (1 + want_lse.abs()))).all()


def check(s, **kw):
    call = {n: kw[n] for n in ("causal", "window", "scale") if n in kw}
    got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, **kw)
    torch.cuda.synchronize()
    close_attended(got, lse, s.q, *s.args(), **call)
    return got, lse


# ---- attention ----------------------------------------------------------------------------------------------------------------------------

ATTENTION = [
    # lens, new, kv heads, group, dim, page
    ([1], [1], 1, 1, 8, 16),
    ([1], [1], 1, 1, 64, 1),
    ([17], [1], 2, 4, 64, 16),
    ([256], [1], 8, 1, 64, 16),
    ([1537], [1], 2, 8, 128, 16),
    ([700, 33, 0, 5, 512], [1, 1, 0, 1, 1], 2, 4, 128, 32),
    ([31, 32, 33, 64, 65, 1], [5, 1, 33, 2, 65, 1], 2, 3, 64, 8),
    ([40], [40], 1, 2, 80, 16),
    ([300], [130], 2, 2, 128, 64),
    ([129], [100], 1, 4, 256, 16),
    ([333, 20], [77, 20], 1, 1, 192, 4),
    ([200, 90], [64, 3], 2, 1, 96, 128),
    ([500], [3], 1, 16, 32, 16),
    ([90, 0, 0, 200, 7], [2, 0, 0, 9, 7], 3, 5, 40, 2),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", ATTENTION)
def test_attention(case, dtype):
    lens, new, kv_heads, group, dim, page = case
    check(Served(lens, new, kv_heads, group, dim, page, dtype, seed=len(lens) + dim))


@pytest.mark.parametrize("case", ATTENTION[2:10])
@pytest.mark.parametrize("kw", [dict(causal=False), dict(window=1), dict(window=37), dict(window=1000), dict(scale=0.7), dict(scale=0.0), dict(scale=-0.2)])
def test_attention_masks_and_scales(case, kw):
    lens, new, kv_heads, group, dim, page = case
    check(Served(lens, new, kv_heads, group, dim, page, BF, seed=5), **kw)


@pytest.mark.parametrize("new", [1, 3, 9, 70, 300])
def test_attention_of_a_long_history(new):
    """Lengths at which the keys are split over workgroups; peaked and flat rows."""
    for length, scale in ((2049, 1.0), (5000, 3.0), (12345, 0.0)):
        s = Served([length, 100], [min(new, 20) if length > 5000 else new, 1], 1, 4, 64, 16, HF, seed=new, q_scale=scale)
        check(s)


def test_attention_of_a_very_long_history():
    check(Served([70001], [1], 1, 2, 64, 16, BF, seed=3))


@pytest.mark.parametrize("new", [1, 50])
def test_attention_where_the_maximum_grows_late(new):
    """Scores that rise by hundreds along the keys: what was summed first has to vanish without a trace."""
    s = Served([900], [new], 1, 2, 64, 16, BF, seed=2)
    s.k.mul_(0.05)
    at = torch.arange(900, device=DEV)
    s.k[s.table[0].long()[at // 16], 0, at % 16] += (at[:, None] / 900 * 4).to(BF)
    s.q.copy_(s.q.abs() * 4)
    check(s)
    check(s, scale=-0.3)


@pytest.mark.parametrize("slot_major", [False, True])
def test_attention_strides(slot_major):
    """Pages laid out slot by slot, keys and values in one pool, queries as a slice of a joined projection, a given output."""
    s = Served([100, 37, 64], [3, 37, 1], 2, 2, 64, 16, HF, seed=1, slot_major=slot_major)
    check(s)
    both = torch.stack((s.k, s.v), 1)
    assert both[:, 0].stride()[0] == 2 * both[:, 0][0].numel()
    joined = torch.randn(41, 8, 72, generator=gen(9)).half().to(DEV)
    joined[:, 2:6, 8:] = s.q
    q = joined[:, 2:6, 8:]
    room = torch.full((41, 4, 128), 7.0, dtype=HF, device=DEV)
    got = paged.cache_attention(q, both[:, 0], both[:, 1], s.table, s.lens, s.cu, out=room[..., 64:])
    assert got.data_ptr() == room[..., 64:].data_ptr()
    assert torch.equal(got, paged.cache_attention(s.q, *s.args())) and (room[..., :64] == 7).all()


def test_attention_bounds_do_not_change_results():
    s = Served([700, 40, 0, 3000], [40, 1, 0, 2], 2, 4, 64, 16, BF, seed=8)
    want = paged.cache_attention(s.q, *s.args())
    for kw in (dict(max_new=40, max_len=3000), dict(max_len=3000), dict(max_new=40), dict(max_new=1, max_len=1), dict(max_new=4, max_len=100)):
        got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, **kw)
        close_attended(got, lse, s.q, *s.args())
        if kw.get("max_new") == 40 or "max_new" not in kw:
            if kw.get("max_len", 3000) == 3000:
                assert torch.equal(got, want)


@pytest.mark.parametrize("new", [1, 6, 90])
def test_a_sequence_does_not_depend_on_its_batch(new):
    lens, news = [777, 2100, 64, 5000], [new, 1, min(new, 64), new]
    s = Served(lens, news, 2, 4, 128, 16, BF, seed=4)
    together = paged.cache_attention(s.q, *s.args())
    for b in range(4):
        a, e = int(s.cu[b]), int(s.cu[b + 1])
        alone = paged.cache_attention(s.q[a:e], s.k, s.v, s.table[b:b + 1].contiguous(), s.lens[b:b + 1].contiguous(), ints([0, e - a]))
        assert torch.equal(alone, together[a:e])


def test_a_sequence_does_not_depend_on_a_longer_one():
    """Lengths around the most parts that a row's keys are cut into: the longer sequence of a call must not change how the shorter one is cut."""
    s = Served([16384, 16700, 16000, 24576, 24900], [1, 1, 40, 1, 1], 1, 1, 64, 64, BF, seed=4)
    together = paged.cache_attention(s.q, *s.args())
    for b in range(5):
        a, e = int(s.cu[b]), int(s.cu[b + 1])
        for kw in (dict(), dict(max_len=int(s.lens[b])), dict(max_len=int(s.lens[b]), max_new=e - a)):
            alone = paged.cache_attention(s.q[a:e], s.k, s.v, s.table[b:b + 1].contiguous(), s.lens[b:b + 1].contiguous(), ints([0, e - a]), **kw)
            assert torch.equal(alone, together[a:e])


def test_rows_behind_the_last_sequence_stay():
    s = Served([50, 20], [4, 1], 2, 2, 64, 16, BF)
    q = torch.cat((s.q, torch.full((7, 4, 64), math.nan, dtype=BF, device=DEV)))
    out = torch.full((12, 4, 64), 3.0, dtype=BF, device=DEV)
    paged.cache_attention(q, *s.args(), out=out)
    assert (out[5:] == 3).all() and torch.equal(out[:5], paged.cache_attention(s.q, *s.args()))


@pytest.mark.parametrize("rows", [40, 300, 1500])
@pytest.mark.parametrize("new", [1, 5, 33])
def test_one_sequence_with_rows_behind_it(rows, new):
    """A call of a fixed number of rows, as a captured one has, of which the one sequence uses the first few."""
    s = Served([700], [new], 2, 2, 64, 16, BF, seed=new)
    q = torch.cat((s.q, torch.full((rows - new, 4, 64), math.nan, dtype=BF, device=DEV)))
    for kw in (dict(), dict(max_len=700), dict(max_new=new), dict(window=100)):
        out = torch.full((rows, 4, 64), 3.0, dtype=BF, device=DEV)
        got, lse = paged.cache_attention(q, *s.args(), out=out, return_lse=True, **kw)
        assert (got[new:] == 3).all()
        close_attended(got, lse, s.q, *s.args(), **{n: kw[n] for n in kw if n == "window"})


@pytest.mark.parametrize("group,dim", [(2, 64), (16, 128), (3, 256)])
@pytest.mark.parametrize("new", [1, 5, 33, 400])
def test_one_sequence_is_cut_by_its_own_rows(new, group, dim):
    """The same bits as it is, in buffers of more rows, beside an idle row, and whatever true bounds are given."""
    s = Served([9000], [new], 1, group, dim, 16, BF, seed=new)
    want, sums = paged.cache_attention(s.q, *s.args(), return_lse=True)
    two = (s.k, s.v, torch.cat((s.table, s.table)), ints([9000, 50]), ints([0, new, new]))
    for rows in (new, 40, 300, 1500):
        q = torch.cat((s.q, s.q.new_zeros(max(0, rows - new), *s.q.shape[1:])))
        for args in (s.args(), two):
            for kw in (dict(), dict(max_new=new), dict(max_new=max(rows - 1, new), max_len=9000), dict(max_len=20000)):
                got, lse = paged.cache_attention(q, *args, return_lse=True, **kw)
                assert torch.equal(got[:new], want) and torch.equal(lse[:new], sums), (rows, kw)


@pytest.mark.parametrize("group,dim", [(2, 64), (16, 128)])
@pytest.mark.parametrize("new", [1, 5, 33])
def test_one_sequence_of_fewer_tokens_than_promised(new, group, dim):
    """max_new = tokens says that all rows are new tokens.  Where it is wrong the values are right all the same."""
    s = Served([9000], [new], 1, group, dim, 16, BF, seed=new)
    for rows in (40, 1500):
        q = torch.cat((s.q, s.q.new_full((rows - new, *s.q.shape[1:]), math.nan)))
        out = torch.full_like(q, 3.0)
        got, lse = paged.cache_attention(q, *s.args(), out=out, return_lse=True, max_new=rows)
        assert (got[new:] == 3).all()
        close_attended(got, lse, s.q, *s.args())


def test_a_mixed_call_with_long_prompts():
    """Every form in one call, keys split in each: long prompts, chunks, single tokens, idle rows, and parts kept by sequence and by token."""
    s = Served([3000, 5000, 0, 900, 2600, 40, 1200], [600, 1, 0, 70, 9, 3, 1100], 1, 2, 64, 16, BF, seed=3)
    check(s)
    check(s, window=1500)
    check(s, max_new=1100, max_len=5000)


def test_a_row_of_many_parts_is_joined_alike():
    """A few rows of many parts are joined by another kernel than many rows are: the same bits."""
    s = Served([20000, 26000, 700], [9, 1, 500], 2, 3, 64, 64, BF, seed=6)
    together, sums = paged.cache_attention(s.q, *s.args(), return_lse=True)
    alone, alone_sums = paged.cache_attention(s.q[:10], s.k, s.v, s.table[:2].contiguous(), s.lens[:2].contiguous(), ints([0, 9, 10]), return_lse=True)
    assert torch.equal(alone, together[:10]) and torch.equal(alone_sums, sums[:10])


@pytest.mark.parametrize("tokens,kv_heads,group,dim,dtype", [(16, 1, 4, 64, BF), (5, 2, 8, 128, HF), (9, 1, 2, 256, BF), (64, 1, 1, 96, HF), (128, 1, 1, 32, BF)])
def test_a_few_tokens_over_a_long_history(tokens, kv_heads, group, dim, dtype):
    """The many-rows form with the most parts: 17 to 128 rows over more keys than 64 parts of 512 hold."""
    s = Served([40001, 12345], [tokens, tokens - 1], kv_heads, group, dim, 64, dtype, seed=dim)
    check(s)
    check(s, window=30000, max_new=tokens)
    check(Served([40001], [tokens], kv_heads, group, dim, 64, dtype, seed=dim + 1), max_new=tokens, max_len=40001)


@pytest.mark.parametrize("lens,new,kv_heads,group,dim,window", [
    ([3000, 77], [300, 5], 2, 4, 256, 1024), ([1900, 1900], [500, 1], 1, 3, 64, 1300), ([1700], [1700], 1, 1, 192, 600), ([5000, 40, 2100], [120, 40, 3], 1, 8, 128, 2050),
    ([2600], [30], 1, 4, 96, 2560), ([2600], [17], 1, 1, 32, 2499), ([2049], [400], 1, 3, 128, 2047),
])
def test_windows_whose_keys_are_cut_by_tile(lens, new, kv_heads, group, dim, window):
    """What a tile of rows sees is split, from the first key of its first token on: windows longer than a part, shorter than the chunk, and almost everything."""
    s = Served(lens, new, kv_heads, group, dim, 16, BF, seed=window)
    got, _ = check(s, window=window)
    assert torch.equal(got, paged.cache_attention(s.q, *s.args(), window=window, max_new=max(new), max_len=max(lens)))
    a, e = int(s.cu[0]), int(s.cu[1])
    alone = paged.cache_attention(s.q[a:e], s.k, s.v, s.table[:1].contiguous(), s.lens[:1].contiguous(), ints([0, e - a]), window=window)
    assert torch.equal(alone, got[a:e])


@pytest.mark.parametrize("other", [[], [40]])
def test_a_long_chunk_of_many_heads_over_a_long_history(other):
    """As many rows as workgroups are at once, and their keys in two parts; the first and last tokens against the reference."""
    n, heads = 512, 64
    s = Served([16500, *other], [n, *[3 for _ in other]], heads, 1, 8, 64, BF, seed=7)
    got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True)
    table = s.table[:1].contiguous()
    for first in (0, 127, 250, n - 4):
        close_attended(got[first:first + 4], lse[first:first + 4], s.q[first:first + 4], s.k, s.v, table, ints([16500 - n + first + 4]), ints([0, 4]))
    assert got.isfinite().all() and torch.equal(got[:n], paged.cache_attention(s.q[:n], s.k, s.v, table, ints([16500]), ints([0, n])))


def test_attention_of_many_sequences():
    """More sequences than lanes look at at a time, in every form, idle ones among them."""
    g = gen(5)
    new = [0 if i % 9 == 4 else int(torch.randint(1, 12 if i % 50 else 60, (1,), generator=g)) for i in range(300)]
    check(Served([n + int(torch.randint(0, 40, (1,), generator=g)) if n or i % 2 else 0 for i, n in enumerate(new)], new, 1, 2, 32, 8, HF, seed=1))


def test_attention_workspace_stays_small():
    """What a call asks for in scratch does not grow with the page table's width times the rows of long prompts."""
    import ctypes as C
    n = C.c_size_t()
    c = _ffi.CacheDesc(_ffi.BF16, 1, 9000, 8, 16, 128, 8, 8192, 0, 8 * 16 * 128, 16 * 128, 128, 1 << 20, 1 << 20)
    a = _ffi.AttentionDesc(16384, 32, 1, 0, 0, 0, 0.1, 4096, 128, 4096, 128)
    assert _ffi.lib().disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)) == 0
    assert 0 < n.value < 1 << 29


@pytest.mark.parametrize("rows,tokens,width", [(256, 4351, 2048), (64, 4159, 2048), (1000, 1000, 2048), (1000, 1000, 8192), (256, 16384, 8192)])
def test_attention_workspace_of_many_sequences(rows, tokens, width):
    """Steps of many sequences over tables of up to 131 072 tokens, nothing known of their lengths, 32 heads of 128 on 8: less than a gigabyte, and with a bound on
    the lengths that single tokens and chunks have, less than half of one."""
    import ctypes as C
    n = C.c_size_t()
    c = _ffi.CacheDesc(_ffi.BF16, 1, 90000, 8, 16, 128, rows, width, 0, 8 * 16 * 128, 16 * 128, 128, 1 << 20, 1 << 20)
    for max_len, most in ((0, 3 << 30 if tokens > 5000 else 1 << 30), (4096, 1 << 29)):
        a = _ffi.AttentionDesc(tokens, 32, 1, 0, 0, max_len, 0.1, 4096, 128, 4096, 128)
        assert _ffi.lib().disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)) == 0
        assert 0 < n.value < most


@pytest.mark.parametrize("rows,kv_heads,group,dim,dtype", [(6000, 2, 4, 64, BF), (6000, 1, 8, 128, BF), (6000, 2, 4, 128, HF), (6000, 1, 3, 256, HF), (16000, 64, 1, 16, HF)])
def test_groups_of_parts_have_the_bits_of_parts(rows, kv_heads, group, dim, dtype):
    """A call of so many sequences that its workgroups add up groups of parts themselves: every form, windows, values that are not finite, pages outside the
    cache; bit for bit what each sequence has alone, where a join adds them up."""
    page, keys = 64, 30000
    lens, new = [70] * rows, [1] * rows
    for b, (n, m) in enumerate([(30000, 1), (9001, 2), (20000, 20), (700, 1), (29999, 60), (12345, 700 // group), (25000, 3000 // group), (26000, 5), (24000, 33), (17000, 400)]):
        lens[3 * b], new[3 * b] = n, m
    g = gen(dim)
    pages = keys // page + 1
    table = torch.stack([torch.randperm(pages, generator=g) for _ in range(40)]).int().repeat(rows // 40, 1)
    k, v = (torch.randn(pages, kv_heads, page, dim, generator=g).to(dtype).to(DEV) for _ in range(2))
    v[int(table[21, 300]), 0, 5, 3] = math.inf            # row 21 sees it whole, others somewhere
    table[24, 200] = -7
    table = table.contiguous().to(DEV)
    cu = [0]
    for m in new:
        cu.append(cu[-1] + m)
    q = torch.randn(cu[-1], kv_heads * group, dim, generator=g).to(dtype).to(DEV)
    import ctypes as C
    c, n = paged._cache(k, v, table), C.c_size_t()
    a = _ffi.AttentionDesc(cu[-1], kv_heads * group, 1, 0, 0, 0, 0.1, kv_heads * group * dim, dim, kv_heads * group * dim, dim)
    assert _ffi.lib().disco_op_cache_attention_workspace_bytes(C.byref(c), C.byref(a), C.byref(n)) == 0
    assert n.value < kv_heads * group * cu[-1] * 64 * (dim * 4 + 8)        # (less than a slot for every part of a row)
    for kw in (dict(), dict(window=11000)):
        got, sums = paged.cache_attention(q, k, v, table, ints(lens), ints(cu), return_lse=True, **kw)
        for b in (*range(0, 30, 3), 1, 2, rows - 1):
            at, to = cu[b], cu[b + 1]
            alone, alone_sums = paged.cache_attention(q[at:to], k, v, table[b:b + 1].contiguous(), ints(lens[b:b + 1]), ints([0, to - at]), return_lse=True, **kw)
            for x, y in ((got[at:to], alone), (sums[at:to], alone_sums)):
                assert torch.equal(x.isnan(), y.isnan()) and torch.equal(x.nan_to_num(7, 8, 9), y.nan_to_num(7, 8, 9)), b
        if not kw:
            assert got[cu[24]:cu[25]].isnan().all() and not got[cu[27]:cu[28]].isnan().any()


def close_heads(got, lse, s, pick, **kw):
    """Some heads and tokens of a large call against the plain form: `pick` [(sequence, first new token, how many)]."""
    kv_heads, group = s.k.shape[1], s.q.shape[1] // s.k.shape[1]
    for b, i, n in pick:
        at, length, new = int(s.cu[b]), int(s.lens[b]), int(s.cu[b + 1] - s.cu[b])
        h = (b + i) % kv_heads
        heads = slice(h * group, h * group + 1)
        k, v = s.k[:, h:h + 1], s.v[:, h:h + 1]
        end = torch.tensor([length - new + i + n], dtype=torch.int32) if kw.get("causal", True) else s.lens[b:b + 1]
        rows = slice(at + i, at + i + n)
        if not kw.get("causal", True):
            assert i + n == new
        close_attended(got[rows, heads], lse[rows, heads], s.q[rows, heads], k, v, s.table[b:b + 1], end, torch.tensor([0, n]), **kw)


LARGE = [
    # lens, new, kv heads, group, dim: rows of more than 1 024 in heads of 72 to 128
    ([1300], [1300], 1, 1, 128), ([2600], [1100], 1, 2, 72), ([700, 900], [600, 513], 2, 2, 80), ([40000], [300], 1, 4, 96), ([5000, 30, 0, 300], [520, 30, 0, 1], 2, 4, 104),
    ([1200], [1025], 8, 1, 120), ([3000, 3000], [1040, 1030], 4, 1, 128),
]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", LARGE)
@pytest.mark.parametrize("kw", [dict(), dict(window=333), dict(causal=False), dict(scale=-0.1)])
def test_the_form_of_256_rows(case, dtype, kw):
    """Split and not, heads that do not fill their blocks, alone and beside the other forms, masks and types."""
    lens, new, kv_heads, group, dim = case
    s = Served(lens, new, kv_heads, group, dim, 16, dtype, seed=dim)
    got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, **kw)
    pick = []
    for b, n in enumerate(new):
        if n:
            m = min(n, 7)
            pick += [(b, i, m) for i in ({0, n // 2, n - m} if kw.get("causal", True) else {n - m})]
    close_heads(got, lse, s, pick, **kw)
    if len(new) > 1:                                      # beside the others, and alone: the same bits
        alone = paged.cache_attention(s.q[:new[0]], s.k, s.v, s.table[:1].contiguous(), s.lens[:1].contiguous(), ints([0, new[0]]), **kw)
        assert torch.equal(alone, got[:new[0]])


def test_every_form_in_one_call():
    """Few, many and large rows of heads of 128, split and not, in one call and each alone: the same bits, and the plain form's values."""
    lens, new = [9000, 1200, 20000, 0, 3000, 700, 6000, 50], [1, 600, 40, 0, 5, 300, 1100, 50]
    s = Served(lens, new, 2, 4, 128, 16, BF, seed=7)
    for kw in (dict(), dict(window=777), dict(max_new=1100, max_len=20000)):
        got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, **kw)
        call = {n: kw[n] for n in kw if n == "window"}
        close_heads(got, lse, s, [(b, i, min(n, 5)) for b, n in enumerate(new) if n for i in {0, min(n // 3, n - min(n, 5)), n - min(n, 5)}], **call)
        for b, n in enumerate(new):
            at = int(s.cu[b])
            alone = paged.cache_attention(s.q[at:at + n], s.k, s.v, s.table[b:b + 1].contiguous(), s.lens[b:b + 1].contiguous(), ints([0, n]), **call)
            assert torch.equal(alone, got[at:at + n])


@pytest.mark.parametrize("dim,dtype", [(128, BF), (80, HF)])
@pytest.mark.parametrize("length", [1500, 20000])
def test_256_rows_and_what_they_do_not_see(dim, dtype, length):
    """Values and keys that are not finite, and pages outside the cache, reach only the rows that see them; split and not."""
    new = 1100
    s = Served([length], [new], 1, 1, dim, 16, dtype, seed=dim)
    pos = torch.arange(length - new, length, device=DEV)
    for kw, hit in ((dict(), length - 500), (dict(window=300), length - 700), (dict(window=300), length - new - 100)):
        sees = (pos >= hit) & (pos < hit + kw.get("window", 1 << 30))
        assert sees.any() and not sees.all()
        clean = paged.cache_attention(s.q, *s.args(), **kw)
        page, slot = int(s.table[0, hit // 16]), hit % 16
        for value in (math.nan, math.inf, -math.inf):
            keep = s.v[page, 0, slot].clone()
            s.v[page, 0, slot, 3:11] = value
            got = paged.cache_attention(s.q, *s.args(), **kw)
            assert torch.equal(got[~sees], clean[~sees])
            want = clean[sees].clone()
            want[..., 3:11] = value
            assert torch.equal(got[sees].nan_to_num(7, 8, 9), want.nan_to_num(7, 8, 9))
            s.v[page, 0, slot] = keep
        keep = s.k[page, 0, slot].clone()
        s.k[page, 0, slot, 5] = math.nan
        got = paged.cache_attention(s.q, *s.args(), **kw)
        assert torch.equal(got[~sees], clean[~sees]) and got[sees].isnan().all()
        s.k[page, 0, slot] = keep
        number, first = int(s.table[0, hit // 16]), hit // 16 * 16
        sees = (pos >= first) & (pos - kw.get("window", 1 << 30) < first + 15)
        s.table[0, hit // 16] = 1 << 30
        got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, **kw)
        assert torch.equal(got[~sees], clean[~sees]) and got[sees].isnan().all() and lse[sees].isnan().all()
        s.table[0, hit // 16] = number


@pytest.mark.parametrize("length", [50, 3000, 20000])
@pytest.mark.parametrize("new,group,dim", [(2, 1, 64), (40, 1, 64), (40, 2, 256), (1100, 1, 128)])
def test_rows_of_infinite_scores(new, group, dim, length):
    """One score of +inf: NaN, as exp(inf - inf), in the rows that see it.  One of -inf: a key without weight.  All of them -inf: NaN, unlike a row without keys.  Whichever
    part of a split row has them, and the other rows of their tiles are as they were."""
    length = max(length, new + 10)
    s = Served([length], [new], 1, group, dim, 16, BF, seed=dim)
    s.k[..., 0] = 0                                       # (times 3e38: every score but the one that is set stays as it is)
    s.q[..., 0] = 3e38
    clean = paged.cache_attention(s.q, *s.args())
    pos = torch.arange(length - new, length, device=DEV)
    for hit in (3, length - new + new // 2):              # a key that all see, in the first part, and one that the later half sees, in the last
        page, slot, sees = int(s.table[0, hit // 16]), hit % 16, pos >= hit
        s.k[page, 0, slot, 0] = 3e38
        got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True)
        assert got[sees].isnan().all() and not lse[sees].isfinite().any()
        assert torch.equal(got[~sees], clean[~sees]) and lse[~sees].isfinite().all()
        s.k[page, 0, slot, 0] = -3e38
        got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True)
        keep = s.v[page, 0, slot].clone()
        s.v[page, 0, slot] = 1000
        other = paged.cache_attention(s.q, *s.args())
        assert got.isfinite().all() and lse.isfinite().all() and torch.equal(got, other) and torch.equal(got[~sees], clean[~sees])
        s.v[page, 0, slot] = keep
        s.k[page, 0, slot, 0] = 0
    s.k[..., 0] = -3e38
    got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True)
    assert got.isnan().all() and (lse == -math.inf).all()


PRECISE = [([300], [130], 2, 2, 128), ([129], [100], 1, 4, 256), ([333, 20], [77, 20], 1, 1, 192), ([200, 90], [64, 3], 2, 1, 96), ([31, 32, 33, 64, 65, 1], [5, 1, 33, 2, 65, 1], 2, 3, 64),
           ([5000, 700], [40, 60], 1, 2, 32), ([1300], [1300], 1, 1, 128), ([20000, 90], [1100, 1], 1, 1, 80)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", PRECISE)
@pytest.mark.parametrize("kw", [dict(), dict(window=100)])
def test_precise_attention(case, dtype, kw):
    """Weights of fp32 precision in every form.  What is left of them after two roundings is 2^-16 (bf16) and, as long as it stays above fp16's smallest step, 2^-22; the result
    is rounded once.  A value of 2^-9 of the weighted |v| (half a step of bf16 weights) would not pass."""
    lens, new, kv_heads, group, dim = case
    s = Served(lens, new, kv_heads, group, dim, 16, dtype, seed=dim)
    got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, precise=True, **kw)
    plain, sums = paged.cache_attention(s.q, *s.args(), return_lse=True, **kw)
    assert torch.equal(lse, sums)
    for b, n in enumerate(new):
        at = int(s.cu[b])
        if n * group <= 16:
            assert torch.equal(got[at:at + n], plain[at:at + n])
        m = min(n, 6)
        for i in {0, n - m}:
            rows, length = slice(at + i, at + i + m), lens[b] - n + i + m
            want, size, _, off = R.attended(s.q[rows], s.k, s.v, s.table[b:b + 1], torch.tensor([length]), torch.tensor([0, m]), **kw)
            left = 2.0 ** -16 if dtype == BF else 2.0 ** -21
            tiny = length * 2.0 ** -25 * 2.0 ** -6 * s.v.double().nan_to_num(0, 0, 0).abs().max().item() if dtype == HF else 0.0
            tol = half(dtype) * want.abs() + (left + 2 * off[..., None] + 2.0 ** -20) * size + tiny + torch.finfo(dtype).smallest_normal
            assert ((got[rows].double().cpu() - want).abs() <= tol).all()


@pytest.mark.parametrize("new,dim", [(40, 64), (1100, 128)])
def test_precise_attention_and_what_is_not_seen(new, dim):
    """Values that are not finite, and pages outside the cache, as without it."""
    s = Served([1500], [new], 1, 1, dim, 16, BF, seed=dim)
    pos, hit = torch.arange(1500 - new, 1500, device=DEV), 1500 - new // 2
    sees = pos >= hit
    clean = paged.cache_attention(s.q, *s.args(), precise=True)
    page, slot = int(s.table[0, hit // 16]), hit % 16
    for value in (math.nan, math.inf, -math.inf):
        keep = s.v[page, 0, slot].clone()
        s.v[page, 0, slot, 3:11] = value
        got = paged.cache_attention(s.q, *s.args(), precise=True)
        want = clean[sees].clone()
        want[..., 3:11] = value
        assert torch.equal(got[~sees], clean[~sees]) and torch.equal(got[sees].nan_to_num(7, 8, 9), want.nan_to_num(7, 8, 9))
        s.v[page, 0, slot] = keep
    s.table[0, hit // 16] = -1
    got = paged.cache_attention(s.q, *s.args(), precise=True)
    sees = pos >= hit // 16 * 16
    assert torch.equal(got[~sees], clean[~sees]) and got[sees].isnan().all()


def test_attention_of_nothing():
    s = Served([50, 0, 20], [0, 0, 0], 2, 2, 64, 16, BF)
    assert paged.cache_attention(s.q, *s.args()).shape == (0, 4, 64)
    s = Served([0, 20], [0, 1], 2, 2, 64, 16, BF)
    check(s)
    # more new tokens than the length holds: those before the sequence's start see nothing
    s = Served([3, 20], [3, 1], 1, 2, 64, 16, BF)
    q = torch.randn(6, 2, 64, generator=gen(1)).to(BF).to(DEV)
    for cu in (ints([0, 5, 6]),):
        got, lse = paged.cache_attention(q, s.k, s.v, s.table, s.lens, cu, return_lse=True)
        assert (got[:2] == 0).all() and (lse[:2] == -math.inf).all()
        close_attended(got, lse, q, s.k, s.v, s.table, s.lens, cu)
    zero = ints([0, 0])                                  # lengths of zero with new tokens
    got, lse = paged.cache_attention(q, s.k, s.v, s.table, zero, ints([0, 5, 6]), return_lse=True)
    assert (got == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("new", [4, 9, 80])
def test_what_a_query_does_not_see_cannot_reach_it(new, value):
    """A key and value in the middle of the new tokens, or before the window, that are not finite: only the queries that see them notice."""
    for kw, hit in ((dict(), 150 - new // 2), (dict(window=20), 150 - new - 5), (dict(window=20), 150 - new // 2)):
        s = Served([150], [new], 1, 2, 64, 16, BF, seed=6)
        page, slot = int(s.table[0, hit // 16]), hit % 16
        for which in ("k", "v"):
            clean = paged.cache_attention(s.q, *s.args(), **kw)
            keep = getattr(s, which)[page, 0, slot].clone()
            getattr(s, which)[page, 0, slot, 3:11] = value
            got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, **kw)
            pos = torch.arange(150 - new, 150, device=DEV)
            sees = (pos >= hit) & (pos < hit + kw.get("window", 1 << 20))
            assert sees.any() or hit < 150 - new
            assert torch.equal(got[~sees], clean[~sees])
            if which == "v":
                want = R.attended(s.q, *s.args(), **kw)[0]
                for i in sees.nonzero()[:, 0].tolist():
                    assert torch.equal(got[i].double().cpu().isfinite(), want[i].isfinite())
                    assert torch.equal(got[i].isnan().cpu(), want[i].isnan())
            elif math.isnan(value):
                assert got[sees].isnan().all()
            getattr(s, which)[page, 0, slot] = keep


def test_scores_that_overflow():
    """A row whose scores are all -inf has no softmax: NaN, unlike a row without keys.  One +inf: NaN too, as exp(inf - inf)."""
    s = Served([40], [2], 1, 1, 64, 16, BF)
    q = torch.zeros(2, 1, 64, dtype=BF, device=DEV)
    s.k.nan_to_num_(0)
    s.k[:] = 3e38
    q[0], q[1] = -3e38, 1e-30
    got, lse = paged.cache_attention(q, *s.args(), return_lse=True)
    assert got[0].isnan().all() and got[1].isfinite().all()


@pytest.mark.parametrize("new", [1, 40])
def test_pages_outside_the_cache_are_not_read(new):
    """A page number out of range gives NaN to the queries that see it and to no others, and no address is formed from it."""
    for number in (-1, -2 ** 31, 1 << 20, 2 ** 31 - 1):
        s = Served([120, 90], [new, new], 2, 2, 64, 16, BF, seed=new)
        clean = paged.cache_attention(s.q, *s.args())
        s.table[0, 6] = number                           # keys 96 .. 111
        got, lse = paged.cache_attention(s.q, *s.args(), return_lse=True)
        pos = torch.arange(120 - new, 120)
        sees = torch.cat((pos >= 96, torch.zeros(new, dtype=torch.bool))).to(DEV)
        assert got[sees].isnan().all() and lse[sees].isnan().all()
        assert torch.equal(got[~sees], clean[~sees])


def test_lengths_out_of_range_are_cut():
    s = Served([64], [1], 1, 1, 64, 16, BF, spare=0)
    s.table = torch.cat((s.table[:, :4], s.table[:, :4]), 1).contiguous()      # capacity 128 tokens
    want = paged.cache_attention(s.q, s.k, s.v, s.table, ints([128]), s.cu)
    got = paged.cache_attention(s.q, s.k, s.v, s.table, ints([2 ** 31 - 1]), s.cu)
    assert torch.equal(got, want)
    got = paged.cache_attention(s.q, s.k, s.v, s.table, ints([-5]), s.cu)
    assert (got == 0).all()


def test_attention_refusals():
    s = Served([50, 20], [4, 1], 2, 2, 64, 16, BF)
    bad = [
        lambda: paged.cache_attention(s.q.half(), *s.args()), lambda: paged.cache_attention(s.q[..., :32], *s.args()),
        lambda: paged.cache_attention(s.q, s.k, s.v[:-1], s.table, s.lens, s.cu), lambda: paged.cache_attention(s.q, s.k.float(), s.v.float(), s.table, s.lens, s.cu),
        lambda: paged.cache_attention(s.q, s.k, s.v.half(), s.table, s.lens, s.cu), lambda: paged.cache_attention(s.q, s.k, s.v, s.table.long(), s.lens, s.cu),
        lambda: paged.cache_attention(s.q, s.k, s.v, s.table[:, ::2], s.lens, s.cu), lambda: paged.cache_attention(s.q, s.k, s.v, s.table, s.lens[:1], s.cu),
        lambda: paged.cache_attention(s.q, s.k, s.v, s.table, s.lens, s.cu[:2]), lambda: paged.cache_attention(s.q, *s.args(), out=s.q[:2]),
        lambda: paged.cache_attention(s.q.transpose(1, 2), *s.args()), lambda: paged.cache_attention(s.q[:, :3].contiguous(), *s.args()),
        lambda: paged.cache_attention(s.q, *s.args(), window=-1), lambda: paged.cache_attention(s.q, *s.args(), causal=False, window=3),
        lambda: paged.cache_attention(s.q, *s.args(), scale=math.inf), lambda: paged.cache_attention(s.q, s.k.cpu(), s.v, s.table, s.lens, s.cu),
        lambda: paged.cache_attention(torch.zeros(5, 4, 65, dtype=BF, device=DEV)[..., 1:], *s.args())]
    for call in bad:
        with pytest.raises((ValueError, _ffi.DiscoError)):
            call()
    with pytest.raises(NotImplementedError):
        paged.cache_attention(s.q.clone().requires_grad_(), *s.args())


# ---- append -------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", [
    # lens, new, q heads, kv heads, dim, rotated, page, interleaved
    ([1], [1], 1, 1, 8, 8, 1, False), ([300, 0, 7, 40], [1, 0, 7, 13], 8, 2, 64, 64, 16, False), ([33, 1000], [20, 1], 5, 1, 80, 32, 32, True),
    ([64, 65], [64, 1], 4, 4, 128, 50, 8, False), ([200, 5], [90, 2], 2, 2, 256, 256, 128, True), ([70], [9], 0, 3, 96, 0, 16, False), ([700], [600], 6, 2, 40, 6, 16, True)])
def test_append(case, dtype):
    lens, new, q_heads, kv_heads, dim, rotated, page, inter = case
    s = Served(lens, new, kv_heads, 1, dim, page, dtype, seed=dim)
    total = sum(new)
    qkv = torch.randn(total + 2, q_heads + 2 * kv_heads, dim, generator=gen(3)).to(dtype).to(DEV)       # two rows behind the last sequence
    q, k, v = qkv.split([q_heads, kv_heads, kv_heads], 1)
    f = paged.rotary_frequencies(rotated) if rotated else None
    kc, vc = s.k.clone(), s.v.clone()
    out = torch.full((total + 2, q_heads, dim), 5.0, dtype=dtype, device=DEV) if q_heads else None
    got = paged.cache_append(q if q_heads else None, k, v, kc, vc, s.table, s.lens, s.cu, inv_freq=f, gain=1.1, interleaved=inter, q_out=out)
    pos = torch.cat([torch.arange(n - m, n) for n, m in zip(lens, new)]).to(DEV)
    if q_heads:
        assert (got[total:] == 5).all()
        if rotated:
            close_turned(got[:total], q[:total], pos, f, 1.1, inter)
        else:
            assert torch.equal(got[:total], q[:total])
    want_k, want_v, at = s.k.clone(), s.v.clone(), 0
    there = torch.zeros(s.pool, page, dtype=torch.bool, device=DEV)
    for b, (n, m) in enumerate(zip(lens, new)):
        for p in range(n - m, n):
            pg, slot = int(s.table[b, p // page]), p % page
            there[pg, slot] = True
            if rotated:
                close_turned(kc[pg, :, slot][None], k[at:at + 1], pos[at:at + 1], f, 1.1, inter)
            else:
                assert torch.equal(kc[pg, :, slot], k[at])
            assert torch.equal(vc[pg, :, slot], v[at])
            at += 1
    for a, b in ((kc, s.k), (vc, s.v)):                   # the other slots are as they were
        assert torch.equal(a.transpose(1, 2)[~there].nan_to_num(9), b.transpose(1, 2)[~there].nan_to_num(9))


def test_append_positions_place_and_bad_pages():
    """Given positions; in place; tokens whose page is out of range, or whose place lies before the sequence, are not written anywhere."""
    s = Served([60, 30], [10, 3], 2, 1, 64, 16, BF, seed=2)
    qkv = torch.randn(13, 6, 64, generator=gen(3)).to(BF).to(DEV)
    q, k, v = qkv.clone().split([2, 2, 2], 1)
    f, pos = paged.rotary_frequencies(64), torch.randint(0, 99999, (13,), generator=gen(4)).to(DEV)
    for p in (pos, pos.int()):
        kc, vc, qq = s.k.clone(), s.v.clone(), q.clone()
        assert paged.cache_append(qq, k, v, kc, vc, s.table, s.lens, s.cu, inv_freq=f, positions=p, q_out=qq) is qq
        close_turned(qq, q, pos, f, 1.0, False)
        close_turned(kc[int(s.table[1, 1]), :, 11:14].transpose(0, 1), k[10:], pos[10:], f, 1.0, False)
    s.table[0, 3] = 1 << 30                                # places 48 .. of the first sequence
    kc, vc = s.k.clone(), s.v.clone()
    paged.cache_append(q, k, v, kc, vc, s.table, ints([60, 2]), s.cu, inv_freq=f)       # and the second has one place before its start
    same = (kc == s.k) | (kc.isnan() & s.k.isnan())
    changed = (~same).any(-1).any(1).nonzero().tolist()   # (page, slot)
    assert sorted(map(tuple, changed)) == sorted([(int(s.table[1, 0]), 0), (int(s.table[1, 0]), 1)])
    paged.cache_append(None, k[:0], v[:0], kc, vc, s.table, s.lens, ints([0, 0, 0]), inv_freq=f)


def test_rows_before_the_first_sequence_are_not_appended():
    """cu_new of some sequences of a larger batch: the rows in front of the first one belong to none, and are written nowhere."""
    s = Served([60, 30], [10, 3], 2, 1, 64, 16, BF, seed=2)
    qkv = torch.randn(18, 6, 64, generator=gen(3)).to(BF).to(DEV)
    q, k, v = qkv.split([2, 2, 2], 1)
    f = paged.rotary_frequencies(64)
    want_k, want_v, kc, vc = s.k.clone(), s.v.clone(), s.k.clone(), s.v.clone()
    want = paged.cache_append(q[5:], k[5:], v[5:], want_k, want_v, s.table, s.lens, s.cu, inv_freq=f)
    out = torch.full((18, 2, 64), 5.0, dtype=BF, device=DEV)
    paged.cache_append(q, k, v, kc, vc, s.table, s.lens, s.cu + 5, inv_freq=f, q_out=out)
    assert torch.equal(out[5:], want) and (out[:5] == 5).all()
    for a, b in ((kc, want_k), (vc, want_v)):
        assert torch.equal(a.nan_to_num(9), b.nan_to_num(9))


@pytest.mark.parametrize("captured", [False, True])
def test_append_behind_a_failed_reserve(captured):
    """Pages are missing: the step's append leaves the cache as it is, bit for bit, also pages that rows share; with enough of them it appends."""
    page, f = 16, paged.rotary_frequencies(64)
    s = Served([60, 60, 30], [0, 0, 0], 2, 1, 64, page, BF, seed=2, spare=2)
    s.table[1, :3] = s.table[0, :3]                       # a fork: three full pages shared, a last page each
    refs = torch.zeros(s.pool, dtype=torch.int32, device=DEV)
    for b, u in enumerate(s.used):
        refs[s.table[b, :u].long()] += 1
    refs[refs == 0] = -1
    free = (refs == -1).nonzero()[:3, 0]
    refs[free] = 0
    cu, qkv = ints([0, 1, 10, 20]), torch.randn(20, 6, 64, generator=gen(3)).to(BF).to(DEV)
    q, k, v = qkv.split([2, 2, 2], 1)
    table = torch.cat((s.table, torch.full((3, 2), -1, dtype=torch.int32, device=DEV)), 1).contiguous()
    kc, vc = s.k.clone(), s.v.clone()

    def step():
        t, n, r, info = paged.cache_reserve(table, s.lens, refs, cu, page)
        out = paged.cache_append(q, k, v, kc, vc, t, n, cu, inv_freq=f, info=info)
        return t, n, r, info, out, paged.cache_attention(out, kc, vc, t, n, cu)

    if captured:
        stream = torch.cuda.Stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            step()
        torch.cuda.current_stream().wait_stream(stream)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step()
    for some in (3, 0, 1, 2, 3):                          # free pages; two are needed: the second row's ten tokens and the third's
        refs[free] = -1
        refs[free[:some]] = 0
        kc.copy_(s.k)
        vc.copy_(s.v)
        if captured:
            graph.replay()
            torch.cuda.synchronize()
        else:
            outs = step()
        t, n, r, info, out, _ = outs
        assert info.tolist() == ([some - 2, 0, 0, 0] if some >= 2 else [some, 2 - some, 0, 0])
        pos = (n - (cu[1:] - cu[:-1])).repeat_interleave(cu[1:] - cu[:-1]) + torch.cat([torch.arange(int(m), device=DEV) for m in cu[1:] - cu[:-1]])
        close_turned(out, q, pos, f, 1.0, False)
        if some < 2:
            assert torch.equal(kc.nan_to_num(9), s.k.nan_to_num(9)) and torch.equal(vc.nan_to_num(9), s.v.nan_to_num(9))
        else:
            want_k, want_v = s.k.clone(), s.v.clone()
            paged.cache_append(q, k, v, want_k, want_v, t, n, cu, inv_freq=f)
            assert not torch.equal(kc.nan_to_num(9), s.k.nan_to_num(9))
            assert torch.equal(kc.nan_to_num(9), want_k.nan_to_num(9)) and torch.equal(vc.nan_to_num(9), want_v.nan_to_num(9))
    for bad in (info[:3], info.long(), torch.zeros(8, dtype=torch.int32, device=DEV)[::2]):
        with pytest.raises(ValueError, match="info"):
            paged.cache_append(q, k, v, kc, vc, t, n, cu, info=bad)


# ---- pages --------------------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("rows,pages,page,width", [(1, 3, 16, 4), (5, 40, 8, 9), (70, 3000, 1, 64), (1100, 9000, 16, 16), (3, 70000, 4, 1000), (9, 64, 16, 8), (16384, 20000, 16, 2)])
def test_reserve(rows, pages, page, width):
    g = gen(rows)
    budget = torch.randint(0, width * page + 1, (rows,), generator=g)
    lens = (budget * torch.rand(rows, generator=g)).int().tolist()
    order, table, at = torch.randperm(pages, generator=g).tolist(), [[-7] * width for _ in range(rows)], 0
    for b in range(rows):
        u = -(-lens[b] // page)
        if at + u > pages * 2 // 3:
            lens[b], u = 0, 0
        table[b][:u] = order[at:at + u]
        at += u
    refs = [0] * pages
    for p in order[:at]:
        refs[p] = 1
    new = [int(min(max(0, n - m), torch.randint(0, 3 * page + 1, (1,), generator=g))) if b % 7 else 0 for b, (n, m) in enumerate(zip(budget.tolist(), lens))]
    for scale in (0, 1, 1000):                            # no new tokens, as drawn, far too many
        n = [x * scale for x in new]
        cu = [0]
        for x in n:
            cu.append(cu[-1] + x)
        want = R.reserved(table, lens, refs, cu, page)
        got = paged.cache_reserve(ints(table), ints(lens), ints(refs), ints(cu), page)
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == want[2]
        assert got[3].tolist() == [*want[3], 0, 0]


def test_reserve_counts_what_is_out_of_range():
    got = paged.cache_reserve(ints([[0, -1], [-1, -1]]), ints([99, -4]), ints([1, 0, 0, 0]), ints([0, 0, 3]), 16)
    assert got[1].tolist() == [32, 3] and got[3].tolist() == [2, 0, 2, 0] and got[0].tolist() == [[0, -1], [1, -1]]


@pytest.mark.parametrize("row", [0, 64, 150, 1023, 1024, 1999])
def test_reserve_counts_the_rows_of_every_wave(row):
    """One row that is too long for the table, or out of range, wherever among the rows: the call fails as a whole, or counts it."""
    rows = 2000
    table, lens, refs = ints([[b, -1] for b in range(rows)]), [9] * rows, ints([1] * rows + [0] * rows)
    cu = [0]
    for b in range(rows):
        cu.append(cu[-1] + (40 if b == row else 1))       # 49 tokens: four pages, two more than the table is wide
    got = paged.cache_reserve(table, ints(lens), refs, ints(cu), 16)
    assert torch.equal(got[0], table) and got[1].tolist() == lens and torch.equal(got[2], refs) and got[3].tolist() == [rows, 2, 0, 0]
    lens[row] = -3
    got = paged.cache_reserve(table, ints(lens), refs, ints(list(range(rows + 1))), 16)
    assert got[3].tolist()[1:] == [0, 1, 0] and got[1].tolist() == [10 if b != row else 1 for b in range(rows)]


def fork_state(rows, page, seed, full=False):
    """Rows of which some share their first pages."""
    g = gen(seed)
    lens, table, count = [], [], 0
    for r in range(rows):
        if r and float(torch.rand(1, generator=g)) < 0.5:
            o = int(torch.randint(0, r, (1,), generator=g))
            n = lens[o] if full else max(lens[o] // page * page, lens[o] - int(torch.randint(0, 2 * page, (1,), generator=g)))
            shared = n // page if n < lens[o] or True else 0
            mine = list(range(count, count + -(-n // page) - shared))
            table.append(table[o][:shared] + mine)
        else:
            n = int(torch.randint(0, 9 * page, (1,), generator=g))
            mine = list(range(count, count + -(-n // page)))
            table.append(mine)
        count += len(mine)
        lens.append(n)
    return lens, table, count


@pytest.mark.parametrize("rows,page,layers,kv_heads,dim,spare", [(*a, b) for a in [(1, 16, 1, 1, 8), (6, 8, 3, 2, 64), (40, 16, 2, 1, 80), (1200, 4, 1, 1, 16)] for b in (0, 3, 2000)]
                         + [(5000, 2, 1, 1, 8, 0), (5000, 2, 1, 1, 8, 9000), (30, 16, 1, 1, 8, 70000)])      # (pools and tables beyond what one workgroup counts)
def test_select(rows, page, layers, kv_heads, dim, spare):
    g = gen(rows + spare)
    lens, table, count = fork_state(rows, page, rows)
    pages, width = count + spare + 1, max(max(map(len, table)), 1) + 1
    place = torch.randperm(pages, generator=g).tolist()
    table = [[place[p] for p in row] + [-5] * (width - len(row)) for row in table]
    k, v = (torch.randn(layers, pages, kv_heads, page, dim, generator=g).half().to(DEV) for _ in range(2))
    identity = list(range(rows))
    for parents in (identity, [-1] * rows, [0] * rows, [int(x) for x in torch.randint(-1, rows, (rows,), generator=g)], identity[::-1],
                    [p if i % 3 else max(0, i - 1) for i, p in enumerate(identity)]):
        want = R.selected([row[:] for row in table], lens, parents, page, pages)
        kk, vv = k.clone(), v.clone()
        got = paged.cache_select(ints(table), ints(lens), ints(parents), kk, vv)
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == want[2]
        free, missing, copied = want[3]
        assert got[3].tolist() == [free, missing, 0, copied]
        for src, dst, slots in want[4]:
            for new, old in ((kk, k), (vv, v)):
                assert torch.equal(new[:, dst, :, :slots], old[:, src, :, :slots])
        for new, old in ((kk, k), (vv, v)):               # nothing else
            for src, dst, slots in want[4]:
                new[:, dst, :, :slots] = old[:, dst, :, :slots]
            assert torch.equal(new, old)


@pytest.mark.parametrize("rows,page,spare", [(2, 16, 3), (7, 8, 30), (60, 4, 200), (60, 16, 2), (1200, 4, 3000), (5000, 2, 9000), (30, 16, 70000)])
def test_select_of_rows_that_were_cut_back(rows, page, spare):
    """Rows of different parents that share a page which a shortened length has made a last page that is not full, for one of them or for several: no two rows may
    end inside the same page, nor inside one that another row has full."""
    g = gen(rows + page)
    lens, table, count = fork_state(rows, page, rows)
    lens = [n if b % 3 == 0 else max(0, n - int(torch.randint(0, 2 * page + 1, (1,), generator=g))) for b, n in enumerate(lens)]
    pages, width = count + spare, max(max(map(len, table)), 1) + 1
    place = torch.randperm(pages, generator=g).tolist()
    table = [[place[p] for p in row] + [-5] * (width - len(row)) for row in table]
    k, v = (torch.randn(1, pages, 1, page, 8, generator=g).half().to(DEV) for _ in range(2))
    identity = list(range(rows))
    for parents in (identity, [int(x) for x in torch.randint(-1, rows, (rows,), generator=g)], identity[::-1], [0] * rows):
        want = R.selected_by_page([row[:] for row in table], lens, parents, page, pages)
        kk, vv = k.clone(), v.clone()
        got = paged.cache_select(ints(table), ints(lens), ints(parents), kk, vv)
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == want[2]
        free, missing, copied = want[3]
        assert got[3].tolist() == [free, missing, 0, copied]
        for new, old in ((kk, k), (vv, v)):
            old = old.cpu().clone()
            for src, dst, slots in want[4]:
                old[:, dst, :, :slots] = old[:, src, :, :slots]
            assert torch.equal(new.cpu(), old)
        if not missing:                                   # a new token of every row, and no two of them in one place
            got = paged.cache_reserve(got[0], got[1], got[2], ints(list(range(rows + 1))), page)
            info = got[3].tolist()
            assert info[3] == 0
            if info[1] == 0:
                at = [(row[(n - 1) // page], (n - 1) % page) for row, n in zip(got[0].tolist(), got[1].tolist())]
                assert len(set(at)) == rows and (got[2][[p for p, _ in at]] == 1).all()


def test_reserve_refuses_new_tokens_in_shared_pages():
    """Rows 0 and 1 share a full page and row 1 is cut back into it; rows 3 and 4 end in the same page.  Nothing is taken, the two that may not write are counted
    (of 3 and 4 only row 4 has new tokens), cache_select makes the pages their own, and the step goes through."""
    page, f = 16, paged.rotary_frequencies(8)
    table, lens = ints([[0, 1, -1], [0, -1, -1], [2, -1, -1], [3, -1, -1], [3, -1, -1]]), ints([20, 10, 5, 9, 7])
    refs = ints([2, 1, 1, 2, 0, 0, 0])
    k = torch.randn(7, 1, page, 8, generator=gen(1)).half().to(DEV)
    v, cu = -k, ints([0, 1, 2, 3, 3, 5])
    got = paged.cache_reserve(table, lens, refs, cu, page)
    assert got[3].tolist() == [3, 2, 0, 2]
    assert torch.equal(got[0], table) and torch.equal(got[1], lens) and torch.equal(got[2], refs)
    x = torch.randn(5, 1, 8, generator=gen(2)).half().to(DEV)
    kc, vc = k.clone(), v.clone()
    paged.cache_append(None, x, x, kc, vc, got[0], got[1], cu, inv_freq=f, info=got[3])
    assert torch.equal(kc, k) and torch.equal(vc, v)
    t, n, r, info = paged.cache_select(table, lens, ints([0, 1, 2, 3, 4]), k, v)
    assert info.tolist() == [1, 0, 0, 2] and t[:, 0].tolist() == [0, 4, 2, 3, 5] and torch.equal(n, lens)
    assert torch.equal(k[4, :, :10], k[0, :, :10]) and torch.equal(v[5, :, :7], v[3, :, :7])
    got = paged.cache_reserve(t, n, r, cu, page)
    assert got[3].tolist() == [1, 0, 0, 0] and got[1].tolist() == [21, 11, 6, 9, 9]
    before, s = k.clone(), n.tolist()
    paged.cache_append(None, x, x, k, v, got[0], got[1], cu, inv_freq=f, info=got[3])
    for b, row in enumerate(got[0].tolist()):             # what the rows held is still there
        for p in range(s[b]):
            assert torch.equal(k[row[p // page], 0, p % page], before[row[p // page], 0, p % page])
    assert all(torch.equal(v[row, 0, at], x[i, 0]) for i, (row, at) in enumerate([(1, 4), (4, 10), (2, 5), (5, 7), (5, 8)]))


def test_select_counts_what_is_out_of_range():
    """Parents that are no rows are empty rows; page numbers outside the cache are passed on, never followed; lengths are cut."""
    k = torch.zeros(4, 1, 16, 8, dtype=BF, device=DEV)
    got = paged.cache_select(ints([[2, 99], [1, -3], [0, 3]]), ints([20, 20, 1000]), ints([0, 0, 7]), k, k.clone())
    # (both rows share page 2; row 0 keeps its last "page" 99, row 1 gets the lowest free page, 0, as its copy of 99: nothing is copied)
    assert got[0].tolist() == [[2, 99], [2, 0], [-1, -1]] and got[1].tolist() == [20, 20, 0] and got[2].tolist() == [1, 0, 2, 0]
    assert got[3].tolist()[2] == 3 and (k == 0).all()
    got = paged.cache_select(ints([[2, 99], [1, -3], [0, 3]]), ints([20, 20, 1000]), ints([2, -1, -1]), k, k.clone())
    assert got[1].tolist() == [32, 0, 0] and got[0].tolist() == [[0, 3], [-1, -1], [-1, -1]] and got[3].tolist() == [2, 0, 1, 0]


@pytest.mark.parametrize("rows,page,layers,kv_heads,dim,spare", [(1, 16, 1, 1, 8, 0), (6, 8, 3, 2, 64, 30), (40, 16, 2, 1, 80, 200), (1, 1, 1, 1, 16, 5000), (300, 4, 1, 1, 16, 9000), (5000, 2, 1, 1, 8, 100), (20, 4, 1, 1, 8, 70000)])
@pytest.mark.parametrize("slot_major", [False, True])
def test_compact(rows, page, layers, kv_heads, dim, spare, slot_major):
    g = gen(rows + spare)
    lens, table, count = fork_state(rows, page, rows)
    pages, width = count + spare + 1, max(max(map(len, table)), 1) + 2
    place = torch.randperm(pages, generator=g).tolist()
    table = [[place[p] for p in row] + [77] * (width - len(row)) for row in table]
    shape = (layers, pages, page, kv_heads, dim) if slot_major else (layers, pages, kv_heads, page, dim)
    k, v = (torch.randn(shape, generator=g).to(BF).to(DEV) for _ in range(2))
    if slot_major:
        k, v = k.transpose(2, 3), v.transpose(2, 3)
    want_table, want_refs, (free, moved), moves = R.compacted(table, lens, page, pages)
    wk, wv = k.clone(), v.clone()
    for src, dst in moves:
        wk[:, dst], wv[:, dst] = k[:, src], v[:, src]
    got = paged.cache_compact(ints(table), ints(lens), k, v)
    assert got[0].tolist() == want_table and got[1].tolist() == want_refs and got[2].tolist() == [free, 0, 0, moved]
    assert torch.equal(k, wk) and torch.equal(v, wv)
    again = paged.cache_compact(got[0], ints(lens), k, v)
    assert torch.equal(again[0], got[0]) and torch.equal(again[1], got[1]) and again[2].tolist() == [free, 0, 0, 0] and torch.equal(k, wk)


def test_copy_pages():
    k, v = (torch.randn(2, 30, 3, 8, 40, generator=gen(s)).half().to(DEV) for s in (1, 2))
    src, dst = [0, 5, 5, 29, -1, 30, 7, 8], [1, 2, 3, 4, 9, 10, -1, 1 << 30]       # the last four have a page out of range
    wk, wv = k.clone(), v.clone()
    for a, b in zip(src[:4], dst[:4]):
        wk[:, b], wv[:, b] = k[:, a], v[:, a]
    paged.cache_copy_pages(k, v, ints(src), ints(dst))
    paged.cache_copy_pages(k, v, ints([]), ints([]))
    assert torch.equal(k, wk) and torch.equal(v, wv)
    paged.cache_copy_pages(k[0], v[0], ints([12]), ints([13]))
    assert torch.equal(k[0, 13], k[0, 12]) and not torch.equal(k[1, 13], k[1, 12])


# ---- all of them together -----------------------------------------------------------------------------------------------------------------

class Model:
    """Sequences grown step by step on a paged cache, and beside it their keys and values as plain lists."""

    def __init__(self, rows, pages, width, layers=2, kv_heads=2, group=2, dim=64, page=8, dtype=HF):
        self.table, self.lens, self.refs = ints([[-1] * width] * rows), ints([0] * rows), ints([0] * pages)
        self.k, self.v = (torch.full((layers, pages, kv_heads, page, dim), math.nan, dtype=dtype, device=DEV) for _ in range(2))
        self.f = paged.rotary_frequencies(dim)
        self.plain = [[(torch.zeros(0, kv_heads, dim, dtype=dtype), torch.zeros(0, kv_heads, dim, dtype=dtype)) for _ in range(layers)] for _ in range(rows)]
        self.rows, self.layers, self.kv_heads, self.heads, self.dim, self.page, self.dtype = rows, layers, kv_heads, group * kv_heads, dim, page, dtype

    def step(self, new, seed):
        cu = ints([sum(new[:i]) for i in range(len(new) + 1)])
        self.table, self.lens, self.refs, info = paged.cache_reserve(self.table, self.lens, self.refs, cu, self.page)
        assert info.tolist()[1:3] == [0, 0]
        for layer in range(self.layers):
            qkv = torch.randn(sum(new), self.heads + 2 * self.kv_heads, self.dim, generator=gen(seed * 10 + layer)).to(self.dtype).to(DEV)
            q, k, v = qkv.split([self.heads, self.kv_heads, self.kv_heads], 1)
            before = [len(r[layer][0]) for r in self.plain]
            pos = torch.cat([torch.arange(b, b + n) for b, n in zip(before, new)]).to(DEV)
            q = paged.cache_append(q, k, v, self.k[layer], self.v[layer], self.table, self.lens, cu, inv_freq=self.f)
            turned = paged.rotary(k, pos, self.f)
            at = 0
            for r, n in enumerate(new):
                a, b = self.plain[r][layer]
                self.plain[r][layer] = (torch.cat((a, turned[at:at + n].cpu())), torch.cat((b, v[at:at + n].cpu())))
                at += n
            got, lse = paged.cache_attention(q, self.k[layer], self.v[layer], self.table, self.lens, cu, return_lse=True)
            self.compare(got, lse, q, layer, new)

    def compare(self, got, lse, q, layer, new):
        at = 0
        for r, n in enumerate(new):
            if n:                                         # the row's own keys and values as a cache of one page
                a, b = (x.transpose(0, 1)[None] for x in self.plain[r][layer])
                close_attended(got[at:at + n], lse[at:at + n], q[at:at + n], a, b, torch.zeros(1, 1, dtype=torch.int32), torch.tensor([a.shape[2]]), torch.tensor([0, n]))
            at += n

    def select(self, parents):
        self.table, self.lens, self.refs, info = paged.cache_select(self.table, self.lens, ints(parents), self.k, self.v)
        assert info.tolist()[1:3] == [0, 0]
        layers = range(self.layers)
        empty = [tuple(x[:0] for x in self.plain[0][layer]) for layer in layers]
        self.plain = [[self.plain[p][layer] if p >= 0 else empty[layer] for layer in layers] for p in parents]


def test_a_run_of_all_operators():
    """Prompts, steps, forks, an ended sequence whose row is used again, a compaction, steps: at every step attention sees what each sequence has been told."""
    m = Model(5, 60, 12)
    m.step([13, 0, 30, 1, 8], 1)
    m.step([1, 0, 1, 1, 1], 2)
    m.select([0, 0, 2, 2, 0])
    m.step([1, 1, 1, 1, 1], 3)
    m.select([3, 1, -1, 3, 1])
    m.step([2, 1, 19, 5, 1], 4)
    live = int((m.refs > 0).sum())
    m.table, m.refs, info = paged.cache_compact(m.table, m.lens, m.k, m.v)
    assert info.tolist()[:3] == [60 - live, 0, 0] and (m.refs[:live] > 0).all() and (m.refs[live:] == 0).all()
    m.step([1, 1, 1, 1, 1], 5)
    m.select([4, 3, 2, 1, 0])
    m.step([1, 7, 0, 1, 1], 6)
    for _ in range(3):
        m.step([1] * 5, 7 + _)


def test_a_captured_step():
    """reserve, append, attention and select in one graph, replayed with other inputs in the same places, with eager work in between: every replay equals the eager result."""
    lens, new, page = [700, 33, 0, 64, 90], [1, 3, 0, 1, 20], 16
    s = Served(lens, [0] * 5, 2, 4, 64, page, BF, seed=1, spare=20)
    s.table = torch.cat((s.table, torch.full((5, 3), -1, dtype=torch.int32, device=DEV)), 1).contiguous()
    cu, refs, f = ints([0, 1, 4, 4, 5, 25]), s.refs(), paged.rotary_frequencies(64)
    parents = ints([0, 0, 3, 3, 4])
    qkv = torch.randn(25, 12, 64, generator=gen(2)).to(BF).to(DEV)
    k0, v0 = s.k.clone(), s.v.clone()

    def step():
        q, k, v = qkv.split([8, 2, 2], 1)
        table, lens, r, info = paged.cache_reserve(s.table, s.lens, refs, cu, page)
        q = paged.cache_append(q, k, v, s.k, s.v, table, lens, cu, inv_freq=f)
        out = paged.cache_attention(q, s.k, s.v, table, lens, cu)
        return (out, *paged.cache_select(table, lens, parents, s.k, s.v), info)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(4):
        qkv.copy_(torch.randn(25, 12, 64, generator=gen(10 + i)).to(BF))
        s.k.copy_(k0)
        s.v.copy_(v0)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in outs] + [s.k.clone(), s.v.clone()]
        s.k.copy_(k0)
        s.v.copy_(v0)
        want = [*step(), s.k, s.v]
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a.nan_to_num(7) if a.is_floating_point() else a, b.nan_to_num(7) if b.is_floating_point() else b)


@pytest.mark.parametrize("group", [2, 20])
def test_a_captured_token_while_its_sequences_grow(group):
    """One graph serves every length up to its table's: how the keys are cut is found on the GPU, from the lengths of the replay."""
    s = Served([9000, 6000], [1, 1], 2, group, 64, 64, BF, seed=2)
    s.k.nan_to_num_(0.5)
    s.v.nan_to_num_(0.5)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        paged.cache_attention(s.q, *s.args())
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged.cache_attention(s.q, *s.args())
    for lens in ([0, 1], [511, 512], [513, 1025], [2048, 3], [8999, 6000], [1, 0]):
        s.lens.copy_(ints(lens))
        graph.replay()
        torch.cuda.synchronize()
        got_now = got.clone()
        want, lse = paged.cache_attention(s.q, *s.args(), return_lse=True, max_new=1, max_len=max(max(lens), 1))
        assert torch.equal(got_now, want)
        close_attended(want, lse, s.q, *s.args())


@pytest.mark.parametrize("rows,pages", [(9000, 12000), (64, 40000)])
def test_captured_page_calls_over_large_pools(rows, pages):
    """Plans with more shared memory than a launch has unasked, and plans of several launches, replayed over tables that change between the replays."""
    kv = torch.randn(pages, 1, 8, 8, generator=gen(1)).to(BF).to(DEV)
    k, v = kv.clone(), -kv
    g = gen(2)
    lens = torch.randint(0, 9, (rows,), generator=g, dtype=torch.int32)
    table = torch.full((rows, 3), -1, dtype=torch.int32)
    used = torch.randperm(pages, generator=g)[:rows].int()
    table[:, 0] = torch.where(lens > 0, used, table[:, 0])
    table, lens = table.to(DEV), lens.to(DEV)
    refs = torch.zeros(pages, dtype=torch.int32, device=DEV)
    refs[table[lens > 0, 0].long()] = 1
    cu = ints(list(range(rows + 1)))
    parents = torch.arange(rows, dtype=torch.int32, device=DEV)

    def step():
        t, n, r, info = paged.cache_reserve(table, lens, refs, cu, 8)
        t, n, r, more = paged.cache_select(t, n, parents, k, v)
        return (*paged.cache_compact(t, n, k, v), n, info, more)

    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(3):
        parents.copy_(torch.arange(rows) // (i + 1) * (i + 1) % rows)
        k.copy_(kv)
        v.copy_(-kv)
        graph.replay()
        torch.cuda.synchronize()
        got = [x.clone() for x in outs] + [k.clone(), v.clone()]
        k.copy_(kv)
        v.copy_(-kv)
        want = [*step(), k, v]
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_captured_groups_of_parts_and_two_streams():
    """A call whose workgroups add parts up, replayed over lengths that change, with another such call on a second stream meanwhile."""
    rows, pages, page, g = 6000, 400, 64, gen(3)
    table = torch.stack([torch.randperm(pages, generator=g) for _ in range(40)]).int().repeat(rows // 40, 1).to(DEV)
    k, v = (torch.randn(pages, 2, page, 64, generator=g).to(BF).to(DEV) for _ in range(2))
    q, cu, lens = torch.randn(rows, 8, 64, generator=g).to(BF).to(DEV), ints(list(range(rows + 1))), ints([50] * rows)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        paged.cache_attention(q, k, v, table, lens, cu)
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = paged.cache_attention(q, k, v, table, lens, cu)
    other = ints([9000 if b % 1000 == 7 else 3 for b in range(rows)])
    want_other = paged.cache_attention(q, k, v, table, other, cu)
    for step in range(3):
        lens.copy_(ints([25000 - 4000 * step if b % 999 == 1 else 10 + step for b in range(rows)]))
        torch.cuda.synchronize()
        graph.replay()
        with torch.cuda.stream(stream):
            beside = paged.cache_attention(q, k, v, table, other, cu)
        torch.cuda.synchronize()
        now = got.clone()
        assert torch.equal(beside, want_other) and torch.equal(now, paged.cache_attention(q, k, v, table, lens, cu))


def test_other_streams_and_calls_at_once():
    """Each call runs on the current stream; calls on several streams at once have workspaces of their own."""
    s = [Served([3000 + 7 * i, 40], [1, 30], 2, 4, 64, 16, BF, seed=i) for i in range(4)]
    want = [paged.cache_attention(x.q, *x.args()) for x in s]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in s], [None] * 4
    for _ in range(3):
        for i, (x, st) in enumerate(zip(s, streams)):
            with torch.cuda.stream(st):
                got[i] = paged.cache_attention(x.q, *x.args())
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a, b)


def test_more_threads_than_an_axis_of_a_launch_has():
    """2^26 rows at a wave each are 2^32 threads: a rotation of that many, and an append and an attention in a buffer of that many, most of them of no sequence."""
    tokens, f = (1 << 26) + 5, paged.rotary_frequencies(8)
    x = torch.randn(tokens, 1, 8, device=DEV, dtype=HF)
    p = torch.arange(tokens, device=DEV, dtype=torch.int32)
    got = paged.rotary(x, p, f)
    for at in (0, 1 << 25, tokens - 1000):
        assert torch.equal(got[at:at + 1000], paged.rotary(x[at:at + 1000], p[at:at + 1000], f))
    del got, p
    s = Served([2000, 700], [3, 1], 1, 1, 8, 16, HF, seed=1)
    kc, vc, want_k, want_v = s.k.clone(), s.v.clone(), s.k.clone(), s.v.clone()
    for cu in (s.cu, s.cu + (tokens - 4)):                # the sequences' rows at the buffer's start, and at its end
        here = x[int(cu[0]):int(cu[0]) + 4]
        paged.cache_append(None, x, x, kc, vc, s.table, s.lens, cu, inv_freq=f)
        paged.cache_append(None, here, here, want_k, want_v, s.table, s.lens, s.cu, inv_freq=f)
        assert torch.equal(kc.nan_to_num(9), want_k.nan_to_num(9)) and torch.equal(vc.nan_to_num(9), want_v.nan_to_num(9))
        out = torch.full_like(x, 3.0)
        paged.cache_attention(x, kc, vc, s.table, s.lens, cu, out=out)
        want = paged.cache_attention(here.contiguous(), kc, vc, s.table, s.lens, s.cu)
        assert torch.equal(out[int(cu[0]):int(cu[0]) + 4], want) and int((out != 3).any(-1).sum()) == 4


def test_offsets_beyond_32_bits():
    """A pool of more than 4 GiB a side: the last pages are read, written and copied where they are."""
    page, kv_heads, dim = 128, 8, 256
    pages = (1 << 32) // (page * kv_heads * dim * 2) + 9
    k, v = (torch.empty(pages, kv_heads, page, dim, dtype=HF, device=DEV) for _ in range(2))
    for c, seed in ((k, 1), (v, 2)):
        c[-3:].copy_(torch.randn(3, kv_heads, page, dim, generator=gen(seed)).half())
        c[:3].zero_()
    table, lens, cu = ints([[pages - 1, pages - 3]]), ints([200]), ints([0, 2])
    q = torch.randn(2, kv_heads, dim, generator=gen(3)).half().to(DEV)
    got, lse = paged.cache_attention(q, k, v, table, lens, cu, return_lse=True)
    small = torch.stack((k[-1], k[-3])), torch.stack((v[-1], v[-3]))
    close_attended(got, lse, q, *small, torch.tensor([[0, 1]]), lens, cu)
    new_k, new_v = (torch.randn(2, kv_heads, dim, generator=gen(s)).half().to(DEV) for s in (4, 5))
    paged.cache_append(None, new_k, new_v, k, v, table, lens, cu)
    assert torch.equal(k[-3, :, 70], new_k[0]) and torch.equal(v[-3, :, 71], new_v[1])
    t, r, info = paged.cache_compact(table, lens, k, v)
    assert t.tolist() == [[1, 0]] and torch.equal(k[1], k[-1]) and torch.equal(v[0], v[-3])

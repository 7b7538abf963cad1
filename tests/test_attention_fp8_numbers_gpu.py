"""Attention over a cache of 8-bit rows where numbers end: infinite queries, bytes that are NaN, factors of the scores that are zero, negative or
large, the largest key scales, and long sums of f32 rows."""
import math

import pytest
import torch

from cache_fp8_tools import PAGE, Cache, Step, attention64
from sapient_b200 import ops
from sapient_b200._lib import check, lib

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("ty", [ops.F32, ops.BF16])


def ways(s):
    """(max_rows, sequences without rows or tokens) that send a call to each kernel: as asked, tiles of 256 rows, row tiles, tiles of 128 rows twice."""
    some = 128 * s.c.kv // s.heads
    return [(max(most, s.max_rows), empty) for most, empty in ((1, 0), (4096, 0), (1, 64), (some, 70), (some, 18))]


@BOTH
@pytest.mark.parametrize("sign", [1, -1])
@pytest.mark.parametrize("rows,dim", [(1, 128), (3, 64), (20, 128), (140, 80), (300, 128)])
def test_infinite_queries(rows, dim, sign, ty):
    """A row and head with an infinity is NaN, whatever the keys' signs there and whichever kernel it goes to; all others are as they were. One that
    sees nothing is zeros."""
    c = Cache([400], 2, dim, 1)
    c.values[:, 0, :, :, 5] &= 0x7F  # of one sign there: every score has the infinity's
    s = Step(c, [(0, rows, 400)], 4, ty, 2)
    head = slice(dim, 2 * dim)
    q = s.q.clone()
    for most, empty in ways(s):
        want = s.run(max_rows=most, empty=empty, out=torch.full_like(s.out, 7.0))
        for coordinate in (5, dim - 1):
            s.q[rows // 2, dim + coordinate] = sign * math.inf
            got = s.run(max_rows=most, empty=empty, out=torch.full_like(s.out, 7.0))
            assert got[rows // 2, head].isnan().all()
            got[rows // 2, head] = want[rows // 2, head]
            assert torch.equal(got, want)
            s.q.copy_(q)
    s.q[rows // 2, dim + 5] = sign * math.inf
    nothing = Step(c, [(0, rows, 0)], 4, ty)
    nothing.q = s.q
    for most, empty in ways(s):
        assert (nothing.run(max_rows=most, empty=empty)[:rows] == 0).all()


@BOTH
@pytest.mark.parametrize("window", [0, 40])
@pytest.mark.parametrize("rows,dim", [(1, 128), (5, 64), (20, 128), (140, 80), (300, 64)])
def test_bytes_that_are_nan(rows, dim, window, ty):
    """A value byte that is NaN beside a finite scale makes its coordinate NaN for the rows that see its token, a key's byte all of them; rows that do not
    see it are as they were, bit for bit."""
    n, heads, kv = 400, 4, 2
    c = Cache([n], kv, dim, 3)
    s = Step(c, [(0, rows, n)], heads, ty, 4)
    pos = torch.arange(n - rows, n, device="cuda")
    values = c.values.clone()
    for most, empty in ways(s):
        want = s.run(window=window, max_rows=most, empty=empty, out=torch.full_like(s.out, 7.0))
        assert not want.isnan().any()
        for token in (n - 1, n - 2, n - rows, max(0, n - rows - 1), n - rows // 2 - 17, n - 129, 130, 0):
            page, row = int(c.table[0, token // PAGE]), token % PAGE
            sees = (pos >= token) & (pos < token + (window or n))
            for which in (1, 0):
                c.values[page, which, 1, row, dim - 3] = 0xFF if token % 2 else 0x7F
                got = s.run(window=window, max_rows=most, empty=empty, out=torch.full_like(s.out, 7.0))
                y = got[:rows].view(rows, heads, dim)
                mine = y[:, 2:] if which == 0 else y[:, 2:, dim - 3]
                assert mine[sees].isnan().all(), (most, empty, token, which)
                assert torch.equal(y[~sees], want[:rows].view(rows, heads, dim)[~sees]), (most, empty, token, which)
                assert torch.equal(y[:, :2], want[:rows].view(rows, heads, dim)[:, :2]) and torch.equal(got[rows:], want[rows:])
                c.values.copy_(values)


@BOTH
@pytest.mark.parametrize("rows", [1, 20, 140])
def test_nan_on_pages_of_others(rows, ty):
    """The first page of the pool, which stands in for pages that are not there, and what lies behind a sequence's end."""
    c = Cache([500], 2, 64, 5)
    c.table[0, 3], c.table[0, 20] = -1, c.n_pages
    own = set(c.table.flatten().tolist())
    if 0 in own:  # the first page becomes nobody's
        free = next(p for p in range(1, c.n_pages) if p not in own)
        c.values[free], c.scales[free] = c.values[0], c.scales[0]
        c.table[c.table == 0] = free
    s = Step(c, [(0, rows, 490)], 4, ty, 6)
    for page in range(c.n_pages):
        if page not in set(c.table.flatten().tolist()):
            c.values[page] = 0x7F
    last = int(c.table[0, 490 // PAGE])
    c.values[last, :, :, 490 % PAGE:] = 0xFF
    s.run()
    s.check()
    assert not s.out.isnan().any()


@BOTH
@pytest.mark.parametrize("scale", [0.0, -0.0, -0.09, 2.0, -30.0, 1e-30])
@pytest.mark.parametrize("rows,dim", [(1, 128), (20, 64), (140, 128), (300, 64)])
def test_factors_of_the_scores(rows, dim, scale, ty):
    """-scale and q are scale and -q: the bounds on errors are those of the latter. 0: the mean of what a row sees."""
    c = Cache([700, 300, 300], 2, dim, 7)
    s = Step(c, [(0, rows, 700), (1, rows, rows // 2), (2, rows, 0)], 4, ty, 8)
    c.table[0, 5] = -1
    q = s.q[: s.n].reshape(s.n, 4, dim)
    for window in (0, 33):
        want, far = attention64(c, -q if scale < 0 else q, s.seqs, abs(scale), window, True)
        for most, empty in ways(s):
            got = s.run(scale=scale, window=window, max_rows=most, empty=empty, out=torch.full_like(s.out, 7.0))
            off = (got[: s.n].view(want.shape).double() - want).abs()
            assert (off <= far).all(), (most, empty, float((off / far).max()))
            assert (got[s.n:] == 7).all()
    check(lib().sp_cuda_check_kernels(0))


@pytest.mark.parametrize("rows,n,steps,keys", [(1, 300000, 12 * 32, 4), (64, 60000, 128, 128)])
def test_long_sums_of_f32_rows(rows, n, steps, keys):
    """A block for each key head of 148 sequences, whose sums run over all of the keys: what the tensor cores cut off does not grow with their number."""
    dim, seqs = 64, 148
    c = Cache([n], 1, dim, 9)
    c.values[:, 1] &= 0x7F  # of one sign, so that errors are relative to the sum itself
    s = Step(c, [(0, rows, n)] * seqs, 1, ops.F32, 10, size=0.05)
    s.q[:] = s.q[:rows].repeat(seqs, 1)
    want, _ = attention64(c, s.q[:rows].view(rows, 1, dim), [(0, rows, n)], dim**-0.5)
    got = s.run(max_rows=128 if rows > 1 else 1)[: s.n].view(seqs, rows, 1, dim)
    assert (got == got[0]).all()
    # Between two additions apart 256 keys in two planes, 16 at a time, are added up: 32 additions, each of which cuts off up to 2^-23 of the sum. The sums
    # apart and those of the weights round to nearest, n times off by 2^-24 / 3 sqrt(n) of the result (a standard deviation, the sum growing evenly), six of
    # which are allowed; rows: of the 12 warps, or 96 threads, that share a row, whose errors are added up as squares. Weights: q is small, z below 1 in size,
    # its error (formula in cache_fp8_tools.py) below 2^-21, ex2's 2^-22, in numerator and denominator; fp16 plus remainder 2^-22; last roundings 2^-23.
    flushes, adds = n / steps / (8 if rows == 1 else 2), n / steps * (keys if rows == 1 else 1) + 32
    shared = 12 if rows == 1 else 1
    six = 6 * 2.0**-24 / 3 * (math.sqrt(flushes / shared) + math.sqrt(adds / (8 * shared if rows == 1 else 1)))
    far = 32 * 2.0**-23 + six + 2 * (2.0**-21 + 2.0**-22) + 2.0**-22 + 2.0**-23
    assert far < 1.3e-5
    off = ((got[0].double() - want).abs() / want).max()
    assert off <= far, (float(off), far)


@BOTH
@pytest.mark.parametrize("rows,dim", [(1, 128), (20, 64), (140, 128), (300, 64)])
def test_the_largest_key_scales(rows, dim, ty):
    """Key scales up to 2^99 against queries that are as small as they are large: no score passes f32's range on its way."""
    c = Cache([700], 2, dim, 11)
    c.scales[:, 0] = 2.0**99 * (0.5 + 0.5 * torch.rand_like(c.scales[:, 0]))
    c.scales[int(c.table[0, 1]), 0] = 2.0**99
    s = Step(c, [(0, rows, 700)], 4, ty, 12, size=2.0**-107)
    want, far = attention64(c, s.q[: s.n].view(s.n, 4, dim), s.seqs, dim**-0.5, 0, True)
    for most, empty in ways(s):
        got = s.run(max_rows=most, empty=empty, out=torch.full_like(s.out, 7.0))
        off = (got[: s.n].view(want.shape).double() - want).abs()
        assert (off <= far).all(), (most, empty, float((off / far).max()))

"""Attention over a cache of 8-bit rows where numbers end: infinite queries and bytes that are NaN."""
import math

import pytest
import torch

from cache_fp8_tools import PAGE, Cache, Step
from sapient_b200 import ops

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

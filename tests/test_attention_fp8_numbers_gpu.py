"""Attention over a cache of 8-bit rows where numbers end: infinite queries."""
import math

import pytest
import torch

from cache_fp8_tools import Cache, Step
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

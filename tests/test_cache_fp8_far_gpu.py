"""The largest page tables that the calls on a cache of 8-bit rows take: positions up to 2^31 - 17, the same bits there as near the start."""
import pytest
import torch

from cache_fp8_tools import PAGE, TYPES, Cache, Step, ints
from sapient_b200 import ops
from sapient_b200._lib import check, lib

pytestmark = pytest.mark.gpu
MOST = (2**31 - 1) // PAGE  # pages of a slot
NEAR, FAR = 496, MOST * PAGE  # the two ends lie alike in tiles of 128 keys


@pytest.fixture(scope="module")
def table():
    return torch.full((1, MOST), -1, dtype=torch.int32, device="cuda")  # 0.5 GB


def caches(kv, dim, table, seed):
    """The same pages at the start of a short page table and at the end of the longest."""
    near = Cache([NEAR], kv, dim, seed)
    far = Cache([NEAR], kv, dim, seed)
    table[0, -(NEAR // PAGE):] = near.table[0]
    far.table, far.max_pages = table, MOST
    far.own = ops.CacheFp8(far.values.data_ptr(), far.scales.data_ptr(), table.data_ptr(), far.n_pages, 1, MOST, kv, dim)
    return near, far


@pytest.mark.parametrize("past", [0, 15])  # tokens behind the page table's end, which nobody sees
@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("rows,dim", [(1, 128), (5, 64), (20, 128), (140, 80), (300, 128)])
def test_attention(rows, dim, ty, past, table):
    assert (FAR - NEAR) % 128 == 0 and FAR + past <= 2**31 - 1
    near, far = caches(2, dim, table, 1)
    steps = [Step(c, [(0, rows, n + past)], 4, ty, 2) for c, n in ((near, NEAR), (far, FAR))]
    some = 128 * 2 // 4
    for most, empty in ((rows, 0), (4096, 0), (max(1, rows), 64), (max(some, rows), 18)):
        want, got = (s.run(window=100, max_rows=most, max_len=5000, empty=empty, out=torch.full_like(s.out, 7.0)) for s in steps)
        assert torch.equal(want, got)
    steps[0].run(window=100)
    steps[0].check(window=100)
    check(lib().sp_cuda_check_kernels(0))


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
def test_append_and_read(ty, table):
    kv, dim = 2, 64
    near, far = caches(kv, dim, table, 3)
    k, v = (torch.randn(20, kv * dim, device="cuda").to(TYPES[ty]) for _ in range(2))
    slot, out = ints([0] * 20), []
    for c, n in ((near, NEAR), (far, FAR)):
        pos = ints([min(n - 19 + i, 2**31 - 1) for i in range(20)])  # the last one lies behind the page table
        y = [torch.full((20, kv * dim), 7.0, device="cuda", dtype=TYPES[ty]) for _ in range(2)]
        ops.cache_fp8_append_dev(c.own, 20, slot.data_ptr(), pos.data_ptr(), k.data_ptr(), v.data_ptr(), dtype=ty)
        ops.cache_fp8_read_dev(c.own, 20, slot.data_ptr(), pos.data_ptr(), y[0].data_ptr(), y[1].data_ptr(), dtype=ty)
        out.append((c.values, c.scales, *y))
    assert all(torch.equal(a, b) for a, b in zip(*out))
    assert (out[1][2][19] == 7).all() and not (out[1][2][:19] == 7).all(-1).any()

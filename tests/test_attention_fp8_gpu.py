"""Attention over a paged cache of 8-bit rows against its formula in 64 bits."""
import math

import pytest
import torch

from cache_fp8_tools import PAGE, Cache, Step, ints
from sapient_b200 import ops
from sapient_b200._lib import check, lib

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("ty", [ops.F32, ops.BF16])


def run(lens, rows, heads, kv, dim, ty, window=0, seed=0, size=1.5):
    c = Cache(lens, kv, dim, seed)
    s = Step(c, [(i, r, n) for i, (r, n) in enumerate(zip(rows, lens))], heads, ty, seed + 1, size)
    s.run(window=window)
    s.check(window=window)
    check(lib().sp_cuda_check_kernels(0))


@BOTH
@pytest.mark.parametrize("dim", [16, 48, 64, 80, 112, 128])
@pytest.mark.parametrize("heads,kv", [(1, 1), (8, 2), (7, 1), (17, 1)])
def test_one_token(heads, kv, dim, ty):
    run([1, 16, 17, 100, 517], [1] * 5, heads, kv, dim, ty)


@BOTH
@pytest.mark.parametrize("n", [1, 2, 15, 31, 32, 33, 255, 256, 257, 1025, 5000, 20011])
def test_lengths(n, ty):
    run([n], [1], 8, 2, 128, ty)


@BOTH
@pytest.mark.parametrize("rows", [1, 2, 3, 4, 5, 8, 9, 16, 17, 33])
@pytest.mark.parametrize("heads,kv,dim", [(4, 1, 128), (6, 2, 64)])
def test_a_few_tokens(rows, heads, kv, dim, ty):
    run([rows, rows + 1, 300, 1040], [rows] * 4, heads, kv, dim, ty)


@BOTH
@pytest.mark.parametrize("rows", [31, 32, 64, 127, 128, 129, 255, 300])
@pytest.mark.parametrize("heads,kv,dim", [(8, 2, 128), (3, 3, 80), (14, 2, 64), (5, 1, 32)])
def test_prompts_and_chunks(rows, heads, kv, dim, ty):
    run([rows, rows + 700, rows + 13, 1], [rows, rows, rows // 2 + 1, 1], heads, kv, dim, ty)


@BOTH
def test_long_prompt(ty):
    run([2113], [2113], 4, 1, 128, ty)


@BOTH
@pytest.mark.parametrize("window", [1, 2, 16, 17, 100, 128, 1000, 5000])
@pytest.mark.parametrize("rows", [1, 5, 200])
def test_window(rows, window, ty):
    run([rows, 1300, 700], [rows] * 3, 8, 2, 128, ty, window=window)


@BOTH
def test_large_and_small_scores(ty):
    for size in (0.0, 1e-30, 1e-3, 40.0, 1e4):
        run([700, 33], [1, 1], 4, 1, 64, ty, size=size)
        run([700, 333], [150, 150], 4, 1, 64, ty, size=size)


@BOTH
@pytest.mark.parametrize("rows", [1, 4, 140])
def test_rows_that_see_nothing(rows, ty):
    """Sequences without tokens, with fewer tokens than rows, without rows, in slots that are not there."""
    c = Cache([300, 300, 300, 300], 2, 64, 3)
    s = Step(c, [(0, rows, 0), (1, rows, rows // 2), (2, 0, 40), (9, rows, 100), (-1, rows, 100), (3, rows, 290), (3, rows, -7)], 4, ty, 4)
    s.run()
    s.check()


@BOTH
@pytest.mark.parametrize("rows", [1, 4, 140])
def test_pages_that_are_not_there(rows, ty):
    """Numbers that are no page's: their tokens are not seen, and nothing is read there. Lengths past the page table as well."""
    c = Cache([600, 600, 600], 2, 128, 5)
    c.table[0, 1] = -1
    c.table[0, 7] = c.n_pages
    c.table[1, :] = 2**30
    c.table[2, 30] = -(2**31)
    s = Step(c, [(0, rows, 500), (1, rows, 500), (2, rows, 3000), (2, rows, 600)], 6, ty, 6)
    s.run()
    s.check()


@BOTH
@pytest.mark.parametrize("rows", [1, 4, 140])
def test_what_is_not_seen_does_not_matter(rows, ty):
    """NaN, infinities and garbage behind a sequence's end, and in tokens that only later rows see."""
    c = Cache([333, 333], 2, 128, 7)
    for slot in (0, 1):
        page = int(c.table[slot, 333 // PAGE])
        c.values[page, :, :, 333 % PAGE:] = 0x7F
        c.scales[page, :, :, 333 % PAGE:] = math.nan
        c.scales[page, 1, :, 333 % PAGE + 1] = math.inf
        c.scales[page, 0, :, 333 % PAGE + 2] = 3e38
    for t in range(c.n_pages):
        if t not in set(c.table.flatten().tolist()):
            c.values[t], c.scales[t] = 0x7F, math.nan
    s = Step(c, [(0, rows, 333), (1, rows, 333)], 6, ty, 8)
    s.run()
    s.check()
    if rows > 1:  # the last token's values, and another sequence's last key
        for slot, which in ((0, 1), (1, 0)):
            page = int(c.table[slot, 332 // PAGE])
            c.values[page, which, :, 332 % PAGE] = 0x7F
            c.scales[page, which, :, 332 % PAGE] = math.nan
        s.run()
        s.check()
        assert not s.out[: rows - 1].isnan().any() and s.out[rows - 1, : 6 * 128].isnan().all()


@BOTH
@pytest.mark.parametrize("rows", [1, 150])
def test_values_of_very_different_size(rows, ty):
    """Scales that grow from token to token: what was added up before stays in proportion."""
    c = Cache([900], 1, 64, 9)
    for i in range(900):
        c.scales[int(c.table[0, i // PAGE]), 1, :, i % PAGE] *= 2.0 ** (i / 30 - 15)
    s = Step(c, [(0, rows, 900)], 4, ty, 10, size=3.0)
    s.run()
    s.check()
    c.scales[:, 1] = 2.0**-100  # rows of zeros
    c.values[:, 1] = 0
    s.run()
    assert (s.out[: s.n, : 4 * 64] == 0).all()


@BOTH
def test_rows_with_nan_or_infinities_keep_to_themselves(ty):
    for rows, most in ((3, None), (140, None), (140, 4096), (3, 4096)):
        c = Cache([400], 2, 128, 11)
        s = Step(c, [(0, rows, 400)], 4, ty, 12)
        s.run(max_rows=most)
        want = s.out.clone()
        s.q[1, :128] = math.nan
        s.q[2, 130] = math.inf
        s.run(max_rows=most)
        got = s.out.clone()
        assert got[1, :128].isnan().all() and not got[0].isnan().any()
        want[1, :128] = want[2, 128:256] = got[1, :128] = got[2, 128:256] = 0
        assert torch.equal(want, got)


@BOTH
@pytest.mark.parametrize("rows", [1, 3, 200])
def test_strides_and_in_place(rows, ty):
    c = Cache([250], 2, 80, 13)
    s = Step(c, [(0, rows, 250)], 4, ty, 14, ld=4 * 80 + 24)
    s.run()
    s.check()
    q = s.q.clone()
    for most in (rows, 128, 4096):
        s.q.copy_(q)
        s.run(max_rows=max(rows, most))
        want = s.out[: s.n, : 4 * 80].clone()
        ops.attention_fp8_dev(c.own, s.q.data_ptr(), 4, s.q.data_ptr(), 1, s.start.data_ptr(), s.len.data_ptr(), max(rows, most), 250, 80**-0.5, dtype=ty, ldq=s.ld, ldo=s.ld)
        assert torch.equal(s.q[:, : 4 * 80], want)


@BOTH
def test_max_rows_and_max_len_are_bounds(ty):
    """Larger bounds give the same; rows past max_rows stay as they are."""
    c = Cache([500, 40], 2, 64, 15)
    s = Step(c, [(0, 20, 500), (1, 3, 40)], 4, ty, 16)
    for rows, length in ((20, 500), (21, 100000), (300, 500), (20, 0)):
        s.out[: s.n] = 0
        s.run(max_rows=rows, max_len=length)
        s.check()
    s.out[:] = 7
    s.run(max_rows=2)
    assert (s.out[2:20, : 4 * 64] == 7).all() and (s.out[22] == 7).all() and not (s.out[:2, : 4 * 64] == 7).any()


def test_far_into_a_large_pool():
    """Pages whose offsets pass 32 bits."""
    kv, dim, n = 8, 128, 140000  # 4.6 GB of values
    values = torch.empty(n, 2, kv, PAGE, dim, dtype=torch.uint8, device="cuda")
    scales = torch.empty(n, 2, kv, PAGE, device="cuda")
    c = Cache([100], kv, dim, 17)
    at = [n - 1 - 2 * i for i in range(7)]
    for i, p in enumerate(at):
        values[p], scales[p] = c.values[int(c.table[0, i])], c.scales[int(c.table[0, i])]
    c.values, c.scales, c.table, c.n_pages = values, scales, ints([at]), n
    c.own = ops.CacheFp8(values.data_ptr(), scales.data_ptr(), c.table.data_ptr(), n, 1, 7, kv, dim)
    for rows in (1, 64):
        s = Step(c, [(0, rows, 100)], 32, ops.BF16, 18)
        s.run()
        s.check()


@pytest.mark.parametrize("rows,n", [(1, 3000), (5, 1200), (300, 1500)])
def test_two_streams_graphs_and_repetition(rows, n):
    """The same bits every time: twice in a row, on two streams at once, in graphs."""
    a = [Step(Cache([n, n // 2], 2, 128, 20 + i), [(0, rows, n), (1, rows, n // 2)], 8, ops.BF16, 30 + i) for i in range(2)]
    want = []
    for s in a:
        want.append(s.run().clone())
        s.check()
    torch.cuda.synchronize()
    graphs = []
    for s in a:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        graphs.append(g)
        s.out.zero_()
    streams = [torch.cuda.Stream() for _ in a]
    torch.cuda.synchronize()
    for _ in range(8):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        for s, st in zip(a, streams):
            s.run(stream=st.cuda_stream)
    torch.cuda.synchronize()
    for s, w in zip(a, want):
        assert torch.equal(s.out[: s.n], w[: s.n])
    check(lib().sp_cuda_check_kernels(0))


def test_many_sequences():
    n = [(i * 37) % 90 for i in range(1000)]
    c = Cache(n, 1, 64, 40)
    s = Step(c, [(i, 1, x) for i, x in enumerate(n)], 2, ops.BF16, 41)
    s.run()
    s.check()

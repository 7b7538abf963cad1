"""Writing a paged cache of 8-bit rows, with norms and rotation, and reading it back, against the formulas in 64 bits."""
import math

import numpy as np
import pytest
import torch

from cache_fp8_tools import PAGE, STEP, TYPES, Cache, Step, ints, normed64, rotated64
from sapient_b200 import ops
from sapient_b200._lib import check, lib

pytestmark = pytest.mark.gpu
BOTH = pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
EPS = 1e-5


class Tokens:
    """q, k and v side by side, and where they go."""

    def __init__(self, c, at, heads, ty, rotary, pairs=False, norms=True, seed=0, extra=0, size=1.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        n, d, kv = len(at), c.dim, c.kv
        self.c, self.at, self.heads, self.ty, self.rotary, self.pairs, self.n = c, at, heads, ty, rotary, pairs, n
        self.wide = (heads + 2 * kv) * d + extra
        self.x = (size * torch.randn(n, self.wide, generator=g, device="cuda")).to(TYPES[ty])
        self.q_out = torch.full((n + 1, heads * d + extra), 7.0, device="cuda", dtype=TYPES[ty])
        self.slot, self.pos = ints([s for s, _ in at]), ints([p for _, p in at])
        self.w = [0.5 + torch.rand(d, generator=g, device="cuda") if norms else None for _ in range(2)]
        self.n_angles = max(1, max(p for _, p in at) + 1)
        self.angles = torch.from_numpy(ops.rope_table(self.n_angles, rotary, 10000.0)).cuda()

    def run(self, q=True, in_place=False, stream=None):
        st = torch.cuda.current_stream().cuda_stream if stream is None else stream
        d, kv, h, size = self.c.dim, self.c.kv, self.heads, self.x.element_size()
        p, w = self.x.data_ptr(), [0 if w is None else w.data_ptr() for w in self.w]
        queries = dict(q=p, n_heads=h, ldq=self.wide, q_out=p if in_place else self.q_out.data_ptr(), ldqo=self.wide if in_place else self.q_out.shape[1]) if q else {}
        ops.cache_fp8_append_dev(self.c.own, self.n, self.slot.data_ptr(), self.pos.data_ptr(), p + h * d * size, p + (h + kv) * d * size, q_w=w[0], k_w=w[1], eps=EPS,
                                 angles=self.angles.data_ptr() if self.rotary else 0, n_angles=self.n_angles, rotary_dim=self.rotary, pairs=self.pairs, dtype=self.ty,
                                 ldk=self.wide, ldv=self.wide, stream=st, **queries)

    def want(self):
        d, kv, h = self.c.dim, self.c.kv, self.heads
        x = self.x[:, : (h + 2 * kv) * d].double().reshape(self.n, h + 2 * kv, d)
        angles = self.angles[self.pos.long().clamp(0, self.n_angles - 1)]
        head = lambda y, w: rotated64(normed64(y, w, EPS), angles, self.rotary, self.pairs)  # noqa: E731
        return head(x[:, :h], self.w[0]), torch.stack([head(x[:, h: h + kv], self.w[1]), x[:, h + kv:]], 1)


def near(got, want, ty, norms):
    """f32: the norm's factor (d additions in threes: 2^-19, rsqrtf 2^-22, two products) and the rotation's three roundings, of the pair's
    length; bf16: half a step more. Without a norm the factor is none."""
    size = want.abs().amax(-1, keepdim=True)
    off = (got.double() - want).abs()
    assert (off <= size * (2.0**-19 if norms else 2.0**-22) + STEP[ty] * want.abs() * (ty == ops.BF16)).all()


def check_cells(c, t, before, live=None):
    """The tokens' cells hold what they should, all others what they held."""
    _, kv = t.want()
    values, scales = c.values.clone(), c.scales.clone()
    for i, (s, p) in enumerate(t.at):
        if live is not None and not live[i]:
            continue
        page = int(c.table[s, p // PAGE])
        y = kv[i]
        scale = scales[page, :, :, p % PAGE].double()
        most = y.abs().amax(-1) / 448
        assert ((scale - most.clamp_min(2.0**-100)).abs() <= most * 2.0**-18 + 2.0**-120).all()
        got = values[page, :, :, p % PAGE].view(torch.float8_e4m3fn).double() * scale[..., None]
        # half a step of e4m3 (2^-10 of the scale below its normal range), values of the row off by 2^-18 of its largest, quotients by 2^-22
        assert ((got - y).abs() <= torch.maximum(y.abs() * 2.0**-4, scale[..., None] * 2.0**-10) * (1 + 2.0**-16) + scale[..., None] * 448 * 2.0**-18).all()
        values[page, :, :, p % PAGE], scales[page, :, :, p % PAGE] = before[0][page, :, :, p % PAGE], before[1][page, :, :, p % PAGE]
    assert torch.equal(values, before[0]) and torch.equal(scales, before[1])


def go(at, room, heads, kv, dim, ty, rotary, pairs=False, norms=True, extra=0, seed=0, size=1.0):
    c = Cache(room, kv, dim, seed)
    t = Tokens(c, at, heads, ty, rotary, pairs, norms, seed, extra, size)
    before = c.values.clone(), c.scales.clone()
    t.run()
    near(t.q_out[: t.n, : heads * dim].reshape(t.n, heads, dim), t.want()[0], ty, norms)
    assert (t.q_out[t.n:] == 7).all() and (t.q_out[:, heads * dim:] == 7).all()
    check_cells(c, t, before)
    return c, t


@BOTH
@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dim,rotary", [(16, 16), (32, 16), (48, 0), (64, 64), (80, 32), (96, 96), (112, 48), (128, 128), (128, 64)])
@pytest.mark.parametrize("heads,kv", [(1, 1), (5, 1), (14, 2), (33, 11)])
def test_append(heads, kv, dim, rotary, pairs, ty):
    go([(0, 0), (0, 17), (1, 31), (1, 4)], [40, 32], heads, kv, dim, ty, rotary, pairs)


@BOTH
@pytest.mark.parametrize("n", [1, 2, 16, 301])
def test_append_prompt(n, ty):
    go([(1, 5 + i) for i in range(n)], [10, n + 9], 8, 2, 128, ty, 128, norms=n % 2 == 0)


@BOTH
def test_append_far_positions(ty):
    """Angles come from the table: no position is too far for them."""
    c = Cache([30], 2, 64, 3, max_pages=9000)
    c.table[0, 8100] = 1
    t = Tokens(c, [(0, 16 * 8100 + 5)], 4, ty, 64, seed=4)
    before = c.values.clone(), c.scales.clone()
    t.run()
    near(t.q_out[:1].reshape(1, 4, 64), t.want()[0], ty, True)
    check_cells(c, t, before)
    pos = 16 * 8100 + 5  # the table's own values
    f = 10000.0 ** (-np.arange(0, 64, 2) / 64)
    assert np.abs(t.angles[pos].cpu().numpy() - np.stack([np.cos(pos * f), np.sin(pos * f)], -1)).max() <= 2.0**-24


@BOTH
def test_append_strides_in_place_and_without_queries(ty):
    c, t = go([(0, i) for i in range(9)], [20], 6, 2, 80, ty, 32, extra=24)
    x, want = t.x.clone(), t.q_out[:9, : 6 * 80].clone()
    t.run(in_place=True)
    assert torch.equal(t.x[:, : 6 * 80], want) and torch.equal(t.x[:, 6 * 80:], x[:, 6 * 80:])
    values, scales = c.values.clone(), c.scales.clone()
    c.values.zero_(), c.scales.zero_()
    t.x.copy_(x)
    t.run(q=False)
    page = c.table[0, :1].long()
    assert torch.equal(c.values[page, :, :, :9], values[page, :, :, :9]) and torch.equal(c.scales[page, :, :, :9], scales[page, :, :, :9])


@BOTH
def test_append_skips_what_is_not_there(ty):
    """Slots and positions outside of the cache, and positions without angles: nothing is written; pages that are none: the query alone."""
    c = Cache([64, 64], 2, 64, 5)
    c.table[1, 2] = c.n_pages
    c.table[1, 3] = -5
    at = [(0, 3), (-1, 3), (2, 3), (0, -1), (0, 64), (2**31 - 1, 0), (0, 2**31 - 1), (1, 40), (1, 50), (1, 8), (0, 62)]
    t = Tokens(c, [(0, 3)] * len(at), 4, ty, 64, seed=6)
    t.at, t.slot, t.pos = at, ints([s for s, _ in at]), ints([p for _, p in at])
    t.n_angles = 61
    t.angles = torch.from_numpy(ops.rope_table(61, 64, 10000.0)).cuda()
    before = c.values.clone(), c.scales.clone()
    t.run()
    queries, cells = [0, 7, 8, 9], [0, 9]
    got = t.q_out[: t.n].reshape(t.n, 4, 64)
    near(got[queries], t.want()[0][queries], ty, True)
    assert (got[[i for i in range(len(at)) if i not in queries]] == 7).all()
    check_cells(c, t, before, [i in cells for i in range(len(at))])


@BOTH
def test_append_zeros_nan_and_infinities(ty):
    c = Cache([16], 2, 64, 7)
    t = Tokens(c, [(0, i) for i in range(4)], 2, ty, 64, norms=False, seed=8)
    t.x[0] = 0
    k = slice(2 * 64, 3 * 64)
    t.x[1, k.start + 5] = math.nan
    t.x[2, k.start + 7] = math.inf
    t.x[3, :] *= 1e30
    t.run()
    page = int(c.table[0, 0])
    s, v = c.scales[page], c.values[page].view(torch.float8_e4m3fn).float()
    assert (s[:, :, 0] == 2.0**-100).all() and (v[:, :, 0] == 0).all()
    assert s[0, 0, 1].isnan() and not s[0, 0, 2].isfinite() and s[0, 1, 1:3].isfinite().all() and s[1, :, :4].isfinite().all()
    assert v[0, 0, 1].isnan().all() and not v[0, 1, :4].isnan().any() and s[:, :, 3].isfinite().all()
    assert t.q_out[:4].isfinite().all()


@BOTH
@pytest.mark.parametrize("dim", [16, 80, 128])
def test_read(dim, ty):
    c = Cache([100, 37], 3, dim, 9)
    c.table[1, 1] = -1
    at = [(0, p) for p in range(100)] + [(1, 36), (1, 20), (5, 0), (-1, 0), (0, -1), (0, 500), (1, 0), (1, 0)]
    slot, pos = ints([s for s, _ in at]), ints([p for _, p in at])
    k, v = (torch.full((len(at), 3 * dim + 8), 7.0, device="cuda", dtype=TYPES[ty]) for _ in range(2))
    ops.cache_fp8_read_dev(c.own, len(at), slot.data_ptr(), pos.data_ptr(), k.data_ptr(), v.data_ptr(), dtype=ty, ldk=3 * dim + 8, ldv=3 * dim + 8)
    for which, y in ((0, k), (1, v)):
        for i, (s, p) in enumerate(at):
            if 0 <= s < 2 and 0 <= p < 16 * c.max_pages and int(c.table[s, p // PAGE]) >= 0:
                want = c.rows(s, p + 1, which)[p].reshape(-1)
                assert ((y[i, : 3 * dim].double() - want).abs() <= want.abs() * STEP[ty]).all()  # one product, rounded once
            else:
                assert (y[i] == 7).all()
        assert (y[:, 3 * dim:] == 7).all()
    one = torch.empty(1, 3 * dim, device="cuda", dtype=TYPES[ty])
    ops.cache_fp8_read_dev(c.own, 1, slot.data_ptr(), pos.data_ptr(), v=one.data_ptr(), dtype=ty)  # values alone
    assert torch.equal(one[0], v[0, : 3 * dim])


@BOTH
@pytest.mark.parametrize("rows", [1, 6, 180])
def test_append_attention_and_read_one_after_the_other(rows, ty):
    """Steps of two sequences as a layer makes them, ten in a row without a pause, and once more from graphs."""
    heads, kv, dim = 8, 2, 128
    c = Cache([10 * rows + 30, 10 * rows], kv, dim, 10)
    steps, reads = [], []
    for i in range(10):
        at = [(0, 30 + i * rows + j) for j in range(rows)] + [(1, i * rows + j) for j in range(rows)]
        t = Tokens(c, at, heads, ty, 128, seed=50 + i)
        s = Step(c, [(0, rows, 30 + (i + 1) * rows), (1, rows, (i + 1) * rows)], heads, ty)
        s.q = t.q_out
        s.ld = heads * dim
        steps.append((t, s))
        reads.append([torch.empty(2 * rows, kv * dim, device="cuda", dtype=TYPES[ty]) for _ in range(2)])

    def all_of_it():
        for (t, s), (k, v) in zip(steps, reads):
            t.run()
            s.run()
            ops.cache_fp8_read_dev(c.own, t.n, t.slot.data_ptr(), t.pos.data_ptr(), k.data_ptr(), v.data_ptr(), dtype=ty, stream=torch.cuda.current_stream().cuda_stream)

    all_of_it()
    for (t, s), (k, v) in zip(steps, reads):
        s.check()
        near(t.q_out[: t.n].reshape(t.n, heads, dim), t.want()[0], ty, True)
        for i in (0, rows, 2 * rows - 1):
            for which, y in ((0, k), (1, v)):
                want = c.rows(t.at[i][0], t.at[i][1] + 1, which)[-1].reshape(-1)
                assert ((y[i].double() - want).abs() <= want.abs() * STEP[ty]).all()
    outs = [s.out.clone() for _, s in steps]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        all_of_it()
    first = int(c.table[0, 0])
    for page in range(c.n_pages):
        if page not in (first, int(c.table[0, 1])):
            c.values[page], c.scales[page] = 0, 0
    for _, s in steps:
        s.out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    for (_, s), w in zip(steps, outs):
        assert torch.equal(s.out[: s.n], w[: s.n])
    check(lib().sp_cuda_check_kernels(0))


@BOTH
@pytest.mark.parametrize("n", [500, 5000])
@pytest.mark.parametrize("heads,kv,dim", [(32, 8, 128), (14, 2, 64)])
def test_append_long_prompt(heads, kv, dim, n, ty):
    """So many tokens that one is only four or two warps' work."""
    go([(0, 3 + i) for i in range(n)], [n + 3], heads, kv, dim, ty, dim)


@BOTH
@pytest.mark.parametrize("n", [9999, 10000, 12347])
def test_read_many(n, ty):
    """Enough tokens that a warp takes four, some of which are not there; keys and values, and either alone."""
    kv, dim = 3, 48
    c = Cache([900, 0, 333], kv, dim, 12)
    c.table[0, 5], c.table[2, 3], c.table[2, 4] = -1, c.n_pages, 2**31 - 1
    g = torch.Generator(device="cuda").manual_seed(n)
    slot = torch.randint(-1, 4, (n,), generator=g, device="cuda").int()
    pos = torch.randint(-3, 16 * c.max_pages + 3, (n,), generator=g, device="cuda").int()
    s, p = slot.long().clamp(0, 2), pos.long().clamp(0, 16 * c.max_pages - 1)
    page = c.table[s, p // PAGE].long()
    there = (slot >= 0) & (slot < 3) & (pos >= 0) & (pos < 16 * c.max_pages) & (page >= 0) & (page < c.n_pages)
    assert there.any() and not there.all()
    page = torch.where(there, page, 0)
    for both in (3, 1, 2):
        out = [torch.full((n + 1, kv * dim), 7.0, device="cuda", dtype=TYPES[ty]) for _ in range(2)]
        ops.cache_fp8_read_dev(c.own, n, slot.data_ptr(), pos.data_ptr(), *(y.data_ptr() if both >> i & 1 else 0 for i, y in enumerate(out)), dtype=ty)
        for which, y in enumerate(out):
            want = c.values[page, which, :, p % PAGE].view(torch.float8_e4m3fn).double() * c.scales[page, which, :, p % PAGE].double().unsqueeze(-1)
            off = (y[:n].double() - want.reshape(n, -1)).abs()
            if both >> which & 1:
                assert (off <= want.reshape(n, -1).abs() * STEP[ty])[there].all() and (y[:n][~there] == 7).all() and (y[n] == 7).all()
            else:
                assert (y == 7).all()

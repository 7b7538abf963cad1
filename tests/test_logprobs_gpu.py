"""Token distributions against the formulas in 64 bits.

Tolerance. exp of a difference d is off by less than 2^-21 + 2^-22 |d|, and |d| exp(d) is at most 1/e; a thread's sums have chains of at
most 16 values a chunk and a chunk in 4096, joins add 20 roundings: for up to 200000 tokens R and T are off by less than
2^-24 (50 + 8 + 20) + 2^-20 < 2^-17 of sum exp and of sum |d| exp. The last subtractions are of numbers below 2^6 (2^-18)."""
import numpy as np
import pytest
import torch

from sapient_b200 import ops

pytestmark = pytest.mark.gpu
TYPES = {ops.F32: torch.float32, ops.BF16: torch.bfloat16}
ABS = 2.0**-16


def call(z, ids, top, outputs=15, ld=0):
    rows, n = z.shape
    lp, ent = torch.full((rows + 1,), 7.0, device="cuda"), torch.full((rows + 1,), 7.0, device="cuda")
    ti, tl = torch.full((rows + 1, top), 7, device="cuda", dtype=torch.int32), torch.full((rows + 1, top), 7.0, device="cuda")
    p = [t.data_ptr() if outputs >> i & 1 else 0 for i, t in enumerate((lp, ent, ti, tl))]
    ops.logprobs_dev(z.data_ptr(), rows, n, ids.data_ptr(), p[0], p[1], top, p[2], p[3], ops.F32 if z.dtype == torch.float32 else ops.BF16, z.stride(0),
                     stream=torch.cuda.current_stream().cuda_stream)
    assert lp[rows] == 7 and ent[rows] == 7 and (ti[rows] == 7).all() and (tl[rows] == 7).all()
    return lp[:rows], ent[:rows], ti[:rows], tl[:rows]


def want(z, ids, top):
    d = z.double()
    lp = torch.log_softmax(d, -1)
    p = lp.exp()
    ent = -(torch.where(p > 0, p * lp, 0.0)).sum(-1)
    at = torch.sort(z + 0.0, dim=-1, descending=True, stable=True).indices[:, :top]
    return lp.gather(1, ids.long()[:, None])[:, 0], ent, at.int(), lp.gather(1, at)


def near(a, b, rel=2.0**-15):
    a, b = a.double(), b.double()
    ok = (a == b) | ((a - b).abs() <= ABS + rel * b.abs())
    assert ok.all(), float((a - b)[~ok].abs().max())


def check(z, ids, top):
    got, exp = call(z, ids, top), want(z, ids, top)
    assert torch.equal(got[2], exp[2])
    for a, b in zip((got[0], got[1], got[3]), (exp[0], exp[1], exp[3])):
        near(a, b)
    return got


def logits(rows, n, ty, seed, ld=None, off=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    z = 3 * torch.randn(rows * (ld or n) + off, generator=g, device="cuda")
    ids = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
    return z.to(TYPES[ty])[off:].view(rows, ld or n)[:, :n], ids


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("rows,n,top", [(1, 1, 1), (3, 2, 2), (2, 5, 0), (4, 31, 31), (1, 32, 32), (2, 100, 8), (5, 1000, 9), (1, 4095, 20), (2, 4097, 32), (3, 8193, 5),
                                        (300, 32768, 20), (1, 50257, 5), (7, 51200, 1), (1, 151936, 20), (40, 151936, 32), (75, 128256, 3), (160, 65536, 20), (1, 200003, 32)])
def test_distribution(ty, rows, n, top):
    check(*logits(rows, n, ty, rows + n), top)


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("ld,off", [(5003, 0), (5003, 1), (5001, 3), (5008, 7), (5002, 5)])
def test_rows_that_start_anywhere(ty, ld, off):
    check(*logits(9, 5000, ty, ld + off, ld, off), 20)


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("rows,n,top", [(1, 65536, 8), (1, 65537, 0), (2, 70001, 1), (9, 131072, 5), (10, 131073, 8), (1, 262147, 9), (1, 400000, 24), (3, 90000, 25), (1, 66000, 32), (16, 50257, 31)])
@pytest.mark.parametrize("off", [0, 1, 6])
def test_few_long_rows(ty, rows, n, top, off):
    z, ids = logits(rows, n, ty, rows + n, n + 3, off)
    check(z, ids, top)
    z[:, :: n // 40] = 9.0  # as many equal maxima as are asked for, in all parts
    z[0, n - 1] = 9.5
    check(z, ids, top)


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("rows,n,top", [(300, 100, 32), (301, 1500, 7), (400, 16384, 25), (310, 9001, 1), (2500, 33, 3), (330, 4097, 0), (299, 32768, 32), (700, 1, 1), (320, 6145, 24)])
def test_many_short_rows(ty, rows, n, top):
    z, ids = logits(rows, n, ty, rows + n, n + 1, 1)
    check(z, ids, top)
    if top:
        z[::3] = 1.5                                  # rows of nothing but ties
        z[1::3, : n // 2] = torch.finfo(z.dtype).min  # and half masked ones
        z[2::3] = (torch.arange(n, device="cuda") * 30 // n).to(z.dtype)
        ids[:] = n - 1
        check(z, ids, top)


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("n", [5000, 70000])
def test_orders_and_ties(ty, n):
    """Ascending rows push every value, constant ones tie everywhere, steps tie in long runs; the lowest id comes first."""
    up = torch.arange(n, device="cuda") / n * 20
    z = torch.stack([up, up.flip(0), torch.full((n,), 2.5, device="cuda"), (up * 0.7).floor(), (up.flip(0)).floor(), torch.where(torch.arange(n, device="cuda") % 7 == 3, 0.0, -0.0)]).to(TYPES[ty])
    ids = torch.tensor([0, n - 1, 5, n // 2, 3, 1], device="cuda", dtype=torch.int32)
    for top in (1, 8, 9, 32):
        check(z.contiguous(), ids, top)


@pytest.mark.parametrize("n", [100, 33000])
def test_masked_tokens(n):
    z, ids = logits(8, n, ops.F32, n)
    z = z.clone()
    z[0, 3:] = -torch.inf                       # three tokens are left
    z[1] = -torch.inf                           # none
    z[2, torch.arange(n, device="cuda") != n - 1] = -torch.inf  # one
    z[3, ::2] = -torch.inf
    z[4] = torch.finfo(torch.float32).min       # all at the type's lowest value: even
    z[5, :-5] = torch.finfo(torch.float32).min
    z[6, 7] = 3e38
    ids[2], ids[5], ids[6] = n - 1, n - 1, 7
    lp, ent, ti, tl = call(z, ids, 20)
    e = want(z, ids, 20)
    keep = [0, 2, 3, 4, 5, 6, 7]
    assert torch.equal(ti, e[2])
    for a, b in ((lp, e[0]), (ent, e[1]), (tl, e[3])):
        near(a[keep], b[keep])
    assert lp[1] == -torch.inf and ent[1] == 0 and (tl[1] == -torch.inf).all() and ti[1].tolist() == list(range(20))


def test_what_is_no_distribution_is_nan():
    z, ids = logits(6, 9000, ops.F32, 1)
    z = z.clone()
    z[1, 8000], z[3, 17], z[4, 5], z[4, 6] = torch.inf, torch.nan, torch.inf, -torch.nan
    good = [0, 2, 5]
    lp, ent, ti, tl = call(z, ids, 4)
    for a in (lp, ent, tl):
        assert torch.isfinite(a[good]).all() and torch.isnan(a[[1, 3, 4]]).all()
    assert ti[1, 0] == 8000 and ti[3, 0] == 17 and ti[4, :2].tolist() == [6, 5]


def test_a_likely_token_keeps_its_digits():
    """One token with nearly all of the mass: log p = -log1p(R) and the entropy, both about R, to a relative 2^-15."""
    n = 60000
    g = torch.Generator(device="cuda").manual_seed(3)
    z = torch.randn(4, n, generator=g, device="cuda")
    ids = torch.tensor([0, 4096, n - 1, 777], device="cuda", dtype=torch.int32)
    z[torch.arange(4), ids.long()] = torch.tensor([22.0, 26.0, 30.0, 40.0], device="cuda")
    lp, ent, _, tl = call(z, ids, 1)
    # (1 + R in 64 bits is off by 2^-53, which is 2^-12 of an R of 4e-13: R apart from the 1 here, too)
    d = z.double() - z.double().amax(-1, keepdim=True)
    d[torch.arange(4), ids.long()] = -torch.inf
    e = torch.exp(d)
    r, t = e.sum(-1), torch.where(e > 0, d * e, 0.0).sum(-1)
    for a, b in ((lp, -torch.log1p(r)), (ent, torch.log1p(r) - t / (1 + r)), (tl[:, 0], -torch.log1p(r))):
        assert ((a.double() - b).abs() <= 2.0**-15 * b.abs()).all()


def test_ids_outside_and_outputs_left_out():
    z, ids = logits(3, 500, ops.BF16, 2)
    bad = torch.tensor([500, -1, 499], device="cuda", dtype=torch.int32)
    lp, ent, _, _ = call(z, bad, 0)
    assert torch.isnan(lp[:2]).all() and torch.isfinite(lp[2]) and torch.isfinite(ent).all()
    whole = call(z, ids, 6)
    for outputs in range(16):
        part = call(z, ids, 6, outputs)
        for i in range(4):
            assert torch.equal(part[i], whole[i]) if outputs >> i & 1 else (part[i] == 7).all()


def test_the_same_bits_on_every_run_and_in_every_batch():
    z, ids = logits(200, 40000, ops.F32, 5)
    a, b = call(z, ids, 20), call(z, ids, 20)
    assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_host_form():
    z, ids = logits(3, 700, ops.F32, 6)
    lp, ent, ti, tl = ops.logprobs(z.cpu().numpy(), ids.cpu().numpy(), top=5)
    e = want(z, ids, 5)
    near(torch.from_numpy(lp).cuda(), e[0]), near(torch.from_numpy(ent).cuda(), e[1]), near(torch.from_numpy(tl).cuda(), e[3])
    assert np.array_equal(ti.astype(np.int32), e[2].cpu().numpy())
    assert ops.logprobs(z.cpu().numpy(), None)[0] is None


@pytest.mark.parametrize("n", [700, 40000, 128256])
@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
def test_rows_alone_and_among_others(ty, n):
    """Blocks and threads of a row go by how many rows there are: its bits may differ, its tokens not, nor the bounds of its numbers."""
    z, ids = logits(320, n, ty, 8)
    for at, count in [(0, 1), (199, 1), (0, 3), (40, 30), (7, 75), (0, 160), (0, 320)]:
        check(z[at : at + count], ids[at : at + count].clone(), 20)

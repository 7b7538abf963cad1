"""Products of fp8 rows with fp8 weights against sums in 64 bits.

Tolerance. Products of e4m3 values are exact in f32. A sum over k columns in any order, cut off or rounded at 2^-23 of the running sum
at every step, is off by at most (k + blocks) 2^-23 of the sum of the magnitudes; in practice columns meet in groups of 32, so that
chains are k / 32 + 32 long, and that is what is allowed, with the scales' product, its use and the last rounding."""
import numpy as np
import pytest
import torch

from sapient_b200 import ops

pytestmark = pytest.mark.gpu
TYPES = {ops.F32: torch.float32, ops.BF16: torch.bfloat16}


def inputs(m, n, k, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    e4m3 = lambda *s: (100 * torch.randn(*s, generator=g, device="cuda")).clamp(-448, 448).to(torch.float8_e4m3fn)  # noqa: E731
    xq, wq = e4m3(m, k), e4m3(n, k)
    xs = torch.rand(m, -(-k // 128), generator=g, device="cuda") * 0.02 + 1e-4
    ws = torch.rand(-(-n // 128), -(-k // 128), generator=g, device="cuda") * 0.001 + 1e-5
    return xq, xs, wq, ws


def held(q, s, height):
    return q.float().double() * s.double().repeat_interleave(height, 0)[: q.shape[0]].repeat_interleave(128, 1)[:, : q.shape[1]]


def product(xq, xs, wq, ws, ty=ops.F32, pad=0, device=0):
    m, n = xq.shape[0], wq.shape[0]
    y = torch.full((m + 1, n + pad), 77.0, device=xq.device, dtype=TYPES[ty])
    ops.matmul_fp8_dev(xq.data_ptr(), xs.data_ptr(), m, wq.data_ptr(), ws.data_ptr(), n, xq.shape[1], y.data_ptr(), ty, n + pad, device,
                       torch.cuda.current_stream(xq.device).cuda_stream)
    assert (y[m] == 77).all() and (y[:, n:] == 77).all()  # what lies behind the last row and the last column
    return y[:m, :n]


def check(y, xq, xs, wq, ws):
    x, w = held(xq, xs, 1), held(wq, ws, 128)
    k = x.shape[1]
    want, size = x @ w.T, x.abs() @ w.abs().T
    far = (y.double() - want).abs()
    allowed = (k / 32 + 32 + k / 128 + 4) * 2.0**-23 * size + (torch.finfo(y.dtype).eps / 2) * want.abs()
    assert (far <= allowed).all(), float((far / allowed).max())


# one row to many, sizes around the tiles' edges, a last block of every length, long and short sums
SIZES = [(1, 1, 16), (1, 128, 128), (1, 4096, 4096), (1, 1000, 8960), (2, 129, 144), (3, 896, 4864), (7, 300, 272), (8, 2048, 2048), (13, 1111, 2064), (16, 127, 1008),
         (17, 256, 256), (31, 515, 1040), (32, 8200, 512), (33, 640, 912), (48, 1, 4096), (64, 2560, 10240), (65, 333, 2000), (100, 4096, 400), (127, 2000, 1536),
         (128, 128, 128), (129, 257, 384), (200, 151, 8960), (256, 1024, 4096), (300, 513, 1120), (389, 1544, 2064), (512, 256, 16), (1000, 700, 640), (1025, 2049, 1168)]


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_product(ty, m, n, k):
    a = inputs(m, n, k, m + n + k)
    pad = (m % 4) if m % 2 else 8 * (n % 2)
    y = product(*a, ty, pad)
    check(y, *a)
    assert torch.equal(y, product(*a, ty, 0))  # the stride changes nothing, and twice is the same


# a size or two for every way that products take: which kernel, how its columns are shared, whether tiles come in rounds, are halved or
# leave by warps of their own
@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("m,n,k", [(8, 9000, 1536), (5, 2000, 8208), (16, 1000, 1040), (12, 4100, 2064), (3, 20000, 1024), (24, 640, 8192), (30, 3000, 512), (48, 1530, 8960),
                                   (64, 333, 4112), (96, 1536, 8960), (128, 200, 6160), (100, 32000, 896), (128, 28700, 1040), (40, 4000, 640), (128, 9400, 272), (500, 1000, 1040),
                                   (300, 8200, 1168), (512, 4100, 144), (257, 16500, 528), (2000, 8192, 512), (1500, 8200, 1296), (1300, 5000, 2064), (640, 19000, 1040), (300, 500, 12304), (513, 129, 8208), (128, 4096, 4112), (100, 2500, 8208), (60, 4090, 8192), (384, 1500, 8976), (130, 1001, 6160), (70, 2600, 14352),
                                   (40, 600, 14336), (256, 1024, 6400), (17, 28800, 1040), (41, 20000, 2064), (19, 9300, 2576)])
def test_every_way(ty, m, n, k):
    a = inputs(m, n, k, m + n)
    check(product(*a, ty, 4 * (m % 2)), *a)
    if m % 4 == 0:
        check(product(*a, ty, 3), *a)  # rows of y that start anywhere


@pytest.mark.parametrize("m", [1, 7, 8, 9, 16])
@pytest.mark.parametrize("n,k", [(1, 32), (700, 16), (2000, 48), (2300, 992), (2400, 12320), (4700, 6176), (4800, 1056), (9600, 160), (4752, 4096), (17, 5008), (12800, 2096), (30000, 48), (100, 33024)])
def test_up_to_sixteen_rows(m, n, k):
    """Every number of warps and of blocks of columns ahead, rows that start on 32 bytes and on 16, a matrix that starts on 16."""
    a = inputs(m, n, k, m + n)
    check(product(*a, ops.F32, 1), *a)
    xq, xs, wq, ws = a
    off = torch.empty(n * k + 16, device="cuda", dtype=torch.uint8)[16:]
    off.copy_(wq.view(torch.uint8).reshape(-1))
    check(product(xq, xs, off.view(n, k).view(torch.float8_e4m3fn), ws, ops.BF16), *a)


@pytest.mark.parametrize("m,n,k", [(1, 14336, 4096), (5, 26000, 4096), (8, 8200, 4112), (24, 28672, 4096), (2048, 4096, 2048), (700, 16400, 1040)])
def test_large(m, n, k):
    a = inputs(m, n, k, 3)
    check(product(*a), *a)


@pytest.mark.parametrize("m,n,k", [(70000, 16, 16), (17, 200000, 16), (16, 100003, 16), (33, 65537, 128), (200001, 7, 32), (1000, 3, 16400), (2, 5, 60000), (129, 1, 16), (40000, 130, 48)])
def test_long_in_one_direction(m, n, k):
    a = inputs(m, n, k, 11)
    check(product(*a, ops.BF16, 1), *a)


def test_each_row_is_its_own_whatever_the_others():
    """Rows of a batch, of a prompt and alone: within the tolerance of each other, since all are of the formula; a NaN or an infinite
    scale in one row leaves the others."""
    for m in (5, 40, 300):
        xq, xs, wq, ws = inputs(m, 384, 528, 9)
        y = product(xq, xs, wq, ws)
        xs2 = xs.clone()
        xs2[2, 1] = float("nan")
        xs2[4, 0] = float("inf")
        z = product(xq, xs2, wq, ws)
        keep = [i for i in range(m) if i not in (2, 4)]
        assert torch.equal(z[keep], y[keep]) and torch.isnan(z[2]).all() and not torch.isfinite(z[4]).any()
        wq2 = wq.clone().view(torch.uint8)
        wq2[200, 527] = 0x7F  # e4m3's NaN
        z = product(xq, xs, wq2.view(torch.float8_e4m3fn), ws)
        cols = [i for i in range(384) if i != 200]
        assert torch.equal(z[:, cols], y[:, cols]) and torch.isnan(z[:, 200]).all()


def test_what_lies_behind_a_matrix_is_not_multiplied():
    """Rows and columns behind the last ones, in tiles and blocks that hang over, hold NaN here."""
    for m, n, k in [(3, 130, 144), (140, 200, 272)]:
        xq, xs, wq, ws = inputs(m, n, k, 4)
        big = lambda q: torch.cat([q.view(torch.uint8).reshape(-1), torch.full((1 << 16,), 0x7F, device="cuda", dtype=torch.uint8)])  # noqa: E731
        bx, bw = big(xq), big(wq)
        y = torch.empty(m, n, device="cuda")
        ops.matmul_fp8_dev(bx.data_ptr(), xs.data_ptr(), m, bw.data_ptr(), ws.data_ptr(), n, k, y.data_ptr())
        torch.cuda.synchronize()
        check(y, xq, xs, wq, ws)


def test_weights_on_the_device():
    rng = np.random.default_rng(2)
    for n, k, ms in [(200, 272, (1, 3, 40)), (129, 4096, (2, 300, 5))]:
        _, _, wq, ws = inputs(1, n, k, 8)
        w = ops.Weight.from_fp8(wq.view(torch.uint8).cpu().numpy(), ws.cpu().numpy())
        assert (w.n, w.k, w.dtype) == (n, k, ops.F8_E4M3)
        want = held(wq, ws, 128)
        assert np.array_equal(w.dequant(), want.float().cpu().numpy())  # one rounding of an exact product
        for m in ms:
            x = rng.standard_normal((m, k)).astype(np.float32)
            xq, xs = ops.quant_fp8(x)
            y = w.matmul_nt(x)
            assert np.array_equal(y, ops.matmul_fp8(xq, xs, wq.view(torch.uint8).cpu().numpy(), ws.cpu().numpy()))
            check(torch.from_numpy(y).cuda(), torch.from_numpy(xq).cuda().view(torch.float8_e4m3fn), torch.from_numpy(xs).cuda(), wq, ws)
        from sapient_b200._lib import SP_ERR_DTYPE, SapientCudaError

        with pytest.raises(SapientCudaError) as e:
            w.embed([0])
        assert e.value.status == SP_ERR_DTYPE
        w.free()


def test_results_that_start_inside_a_value():
    from sapient_b200._lib import SP_ERR_ARG, SapientCudaError

    w = ops.Weight.from_fp8(np.ones((4, 32), np.uint8), np.ones((1, 1)))
    x, y = torch.ones(2, 32, device="cuda"), torch.zeros(16, device="cuda")
    for off in (1, 2, 3):
        with pytest.raises(SapientCudaError) as e:
            w.matmul_nt_dev(x.data_ptr(), 2, y.data_ptr() + off, torch.cuda.current_stream().cuda_stream)
        assert e.value.status == SP_ERR_ARG
    w.matmul_nt_dev(x.data_ptr(), 2, y.data_ptr() + 4, torch.cuda.current_stream().cuda_stream)
    assert (y[1:9] != 0).all() and (y[9:] == 0).all() and y[0] == 0


@pytest.mark.parametrize("n,k", [(384, 528), (4100, 2064), (2000, 8208)])
def test_rows_alone_and_among_others(n, k):
    """Which kernel a row goes through depends on how many there are, and so do its bits; the bounds of the formula do not."""
    xq, xs, wq, ws = inputs(600, n, k, 12)
    for at, m in [(0, 1), (599, 1), (5, 7), (64, 16), (10, 40), (100, 128), (0, 300), (0, 600)]:
        a = (xq[at : at + m], xs[at : at + m], wq, ws)
        check(product(*a), *a)

"""Norm, SwiGLU and plain rows to fp8 against the formulas in 64 bits.

Tolerances. y: of a norm the sum of squares has at most 32 + 5 + 32 roundings in a chain of positive terms, half of which the root
leaves, and the root, two products, the addition and the mean add 8: 2^-24 x 43 < 2^-18. SwiGLU: exp and the division are off by
less than 2^-21 + |g| 2^-23 where the result matters (|g| <= 20 here): below 2^-17. A scale adds one rounding. q is off by half a step:
2^-4 of a normal value, 2^-10 of the scale below that."""
import numpy as np
import pytest
import torch

from sapient_b200 import ops

pytestmark = pytest.mark.gpu
TYPES = {ops.F32: torch.float32, ops.BF16: torch.bfloat16}
REL = 2.0**-17


def held(q, scale):
    """What fp8 rows stand for, in 64 bits."""
    v = q.view(torch.float8_e4m3fn).float().double()
    return v * scale.double().repeat_interleave(128, 1)[:, : q.shape[1]]


def scales_of(y):
    p = torch.nn.functional.pad(y.abs(), (0, -y.shape[1] % 128)).view(y.shape[0], -1, 128)
    return (p.amax(-1) / 448).clamp_min(2.0**-100)


def check(q, scale, y):
    want = scales_of(y)
    assert ((scale.double() - want).abs() <= REL * want).all()
    far = (held(q, scale) - y).abs()
    s = want.repeat_interleave(128, 1)[:, : y.shape[1]]
    assert (far <= torch.maximum(2.0**-4 * y.abs(), 2.0**-10 * s) * (1 + 2 * REL) + 2 * REL * y.abs()).all()


def rows(g, n, dim, ld, ty, scale=1.0):
    """[n, dim] inside rows of ld values."""
    return (torch.randn(n, ld, generator=g, device="cuda") * scale).to(TYPES[ty])[:, :dim]


def norm(x, r, w, eps=1e-5, total=None):
    n, dim = x.shape
    q, s = torch.full((n + 1, dim), 7, device="cuda", dtype=torch.uint8), torch.full((n + 1, -(-dim // 128)), -1.0, device="cuda")
    at = lambda t: 0 if t is None else t.data_ptr()  # noqa: E731
    ld = lambda t: 0 if t is None else t.stride(0)  # noqa: E731
    ops.rms_norm_fp8_dev(at(x), n, dim, at(w), eps, at(q), at(s), dtype=ops.F32 if x.dtype == torch.float32 else ops.BF16, residual=at(r), sum_out=at(total),
                         ldx=ld(x), ldr=ld(r), lds=ld(total), stream=torch.cuda.current_stream().cuda_stream)
    assert (q[n] == 7).all() and (s[n] == -1).all()  # the row behind the last one
    return q[:n], s[:n]


def norm64(x, r, w, eps=1e-5):
    h = x.double() if r is None else x.double() + r.double()
    y = h / (h.square().mean(-1, keepdim=True) + eps).sqrt()
    return h, y if w is None else y * w.double()


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("n,dim,pad", [(1, 16, 0), (3, 112, 0), (2, 128, 8), (5, 144, 0), (33, 896, 0), (7, 1536, 8), (300, 2048, 0), (2, 2064, 16), (9, 4096, 0), (4, 4112, 0),
                                       (3, 8192, 0), (2, 8208, 8), (2, 14336, 0), (1, 32768, 0), (1200, 64, 0), (2500, 256, 0)])
def test_norm(ty, n, dim, pad):
    g = torch.Generator(device="cuda").manual_seed(n * dim + ty)
    x, r = rows(g, n, dim, dim + pad, ty), rows(g, n, dim, dim + 2 * pad, ty, 3.0)
    w = 0.5 + torch.rand(dim, generator=g, device="cuda")
    total = torch.zeros(n, dim + pad, device="cuda", dtype=TYPES[ty])[:, :dim]
    q, s = norm(x, r, w, total=total)
    h, y = norm64(x, r, w)
    check(q, s, y)
    assert torch.equal(total, (x.float() + r.float()).to(TYPES[ty]))
    again = norm(x, r, w)  # without the sum
    assert torch.equal(q, again[0]) and torch.equal(s, again[1])
    q, s = norm(x, None, None)
    check(q, s, norm64(x, None, None)[1])


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
def test_the_sum_may_take_the_place_of_either_input(ty):
    g = torch.Generator(device="cuda").manual_seed(5)
    x, r = rows(g, 700, 512, 520, ty), rows(g, 700, 512, 512, ty)
    w = torch.rand(512, generator=g, device="cuda")
    want = (x.float() + r.float()).to(TYPES[ty])
    q0, s0 = norm(x, r, w)
    for k in (0, 1):
        a = [x.clone(memory_format=torch.preserve_format), r.clone()]
        q, s = norm(a[0], a[1], w, total=a[k])
        assert torch.equal(a[k], want) and torch.equal(q, q0) and torch.equal(s, s0)
    y = x.clone()
    norm(y, y, w, total=y)  # the same rows twice
    assert torch.equal(y, (x.float() * 2).to(TYPES[ty]))


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("n,dim", [(1, 16), (2, 208), (3, 4096), (901, 1040), (5, 8208), (2001, 144), (3, 20000)])
def test_norm_without_a_residual(ty, n, dim):
    """Rows in twos, odd numbers of them; the sum is a copy, elsewhere or in place."""
    g = torch.Generator(device="cuda").manual_seed(n + dim)
    x, w = rows(g, n, dim, dim + 8, ty), 0.5 + torch.rand(dim, generator=g, device="cuda")
    want = norm64(x, None, w)[1]
    total = torch.zeros(n + 1, dim, device="cuda", dtype=TYPES[ty])
    q, s = norm(x, None, w, total=total[:n])
    check(q, s, want)
    assert torch.equal(total[:n], x) and (total[n] == 0).all()
    y = x.clone(memory_format=torch.preserve_format)
    assert torch.equal(norm(y, None, w, total=y)[0], q) and torch.equal(x, y)
    x[n // 2] = 0  # a row of zeros beside others
    q, s = norm(x, None, w)
    assert (q[n // 2] & 0x7F == 0).all() and torch.isfinite(s).all()
    check(q, s, norm64(x, None, w)[1])


@pytest.mark.parametrize("gated", [False, True])
@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("n,dim,pad", [(1, 16, 0), (3, 112, 8), (2, 1040, 0), (7, 4864, 0), (64, 2560, 16), (3, 14336, 0), (70000, 16, 0)])
def test_rows(gated, ty, n, dim, pad):
    g = torch.Generator(device="cuda").manual_seed(n + dim)
    x = rows(g, n, dim * (2 if gated else 1), dim * (2 if gated else 1) + pad, ty, 3.0)
    q, s = torch.empty(n, dim, device="cuda", dtype=torch.uint8), torch.empty(n, -(-dim // 128), device="cuda")
    f = ops.swiglu_fp8_dev if gated else ops.quant_fp8_dev
    f(x.data_ptr(), n, dim, q.data_ptr(), s.data_ptr(), ty, x.stride(0), stream=torch.cuda.current_stream().cuda_stream)
    y = x.double()
    if gated:
        y = y[:, :dim] / (1 + torch.exp(-y[:, :dim])) * y[:, dim:]
    check(q, s, y)


def test_zeros_and_small_and_large_rows():
    x = torch.zeros(6, 256, device="cuda")
    x[1] = 1e-38
    x[2] = 3e38
    x[3, 5] = 2.0**-90
    x[4] = torch.linspace(-1, 1, 256)
    x[5, 128] = -448.0
    q, s = torch.empty(6, 256, device="cuda", dtype=torch.uint8), torch.empty(6, 2, device="cuda")
    ops.quant_fp8_dev(x.data_ptr(), 6, 256, q.data_ptr(), s.data_ptr())
    check(q, s, x.double())
    assert (s[0] == 2.0**-100).all() and (q[0] & 0x7F == 0).all() and s[5, 1] == 1 and s[3, 1] == 2.0**-100
    q, s = norm(x[:1], None, None)
    assert (q & 0x7F == 0).all() and torch.isfinite(s).all()


def test_a_nan_or_an_infinity_reaches_whoever_reads_its_block():
    for bad in (float("nan"), float("inf"), -float("inf")):
        x = torch.ones(3, 400, device="cuda")
        x[1, 130] = bad
        q, s = torch.empty(3, 400, device="cuda", dtype=torch.uint8), torch.empty(3, 4, device="cuda")
        ops.quant_fp8_dev(x.data_ptr(), 3, 400, q.data_ptr(), s.data_ptr())
        assert not torch.isfinite(s[1, 1]) and torch.isfinite(s[[0, 2]]).all() and torch.isfinite(s[1, [0, 2, 3]]).all()
        assert torch.isnan(held(q, s)[1, 128:256]).all()
        q, s = norm(x, None, None)  # the norm takes it to the whole row
        assert torch.isfinite(held(q, s)[[0, 2]]).all() and torch.isnan(held(q, s)[1, 130])


def test_host_forms_and_another_stream():
    rng = np.random.default_rng(1)
    x, r, w = (rng.standard_normal(s).astype(np.float32) for s in ((5, 272), (5, 272), (272,)))
    q, s, h = ops.rms_norm_fp8(x, w, 1e-6, residual=r)
    t = lambda a: torch.from_numpy(a).cuda()  # noqa: E731
    check(t(q), t(s), norm64(t(x), t(r), t(w), 1e-6)[1])
    assert np.array_equal(h, x + r)
    y = x[:, :256]
    q, s = ops.swiglu_fp8(y)
    y = t(y).double()
    check(t(q), t(s), y[:, :128] / (1 + torch.exp(-y[:, :128])) * y[:, 128:])
    q, s = ops.quant_fp8(x)
    check(t(q), t(s), t(x).double())
    st = torch.cuda.Stream()
    a, ww = t(x), t(w)
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        q, s = norm(a, None, ww)
    st.synchronize()
    check(q, s, norm64(a, None, ww)[1])


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("dim", [272, 4096, 8208, 20000])
@pytest.mark.parametrize("with_sum", [False, True])
def test_norms_of_zeros_and_of_very_small_rows(ty, dim, with_sum):
    """1 / sqrt(mean(h^2) + eps) and 1 / scale are both large here, their product past the largest f32: a block of zeros is zeros all the
    same, and small values keep their digits. Of h and w only values whose sums and products f32 holds without a rounding of their own
    below 2^-126: eight bits of a sum of two equal rows, w a power of two."""
    g = torch.Generator(device="cuda").manual_seed(dim + ty)
    w = torch.full((dim,), 2.0, device="cuda")
    for size, eps in [(0.0, 1e-18), (0.0, 1e-20), (0.0, 1e-30), (1e-10, 0.0), (1e-17, 0.0), (1e-37, 1e-30), (1e-37, 1e-37), (1e-41, 1e-37)]:
        x = (torch.randn(5, dim, generator=g, device="cuda").bfloat16().float() * size).to(TYPES[ty])
        x[:, 128:256] = 0
        if size:
            x[:, 0] = size  # bf16 has few of the smallest
        if with_sum and size == 0:
            x = rows(g, 5, dim, dim, ty)
        r = None if not with_sum else -x if size == 0 else x.clone()
        q, s = norm(x, r, w, eps)
        check(q, s, norm64(x, r, w, eps)[1])
        assert (q[:, 128:256] & 0x7F == 0).all() and (s[:, 1] == 2.0**-100).all()


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("u_size", [1.0, 1e4, 1e30])
def test_gates_far_from_zero(ty, u_size):
    """The sigmoid is taken for zero below 2^-126, and off by 2^-21 + |g| 2^-23 of itself above (|g| 2^-24 and half as much again from the
    exponent's product, exp and reciprocal 2^-22 each); products, the scale and its reciprocal add less than 2^-21."""
    g = torch.Generator(device="cuda").manual_seed(3)
    gates = torch.tensor([-1e30, -200.0, -89.0, -88.5, -87.5, -87.25, -87.0, -80.0, -40.0, -0.0, 0.0, 40.0, 80.0, 87.5, 89.0, 200.0, 1e4], device="cuda").repeat_interleave(128)
    dim = gates.numel()
    x = torch.empty(3, 2 * dim, device="cuda")
    x[:, :dim], x[:, dim:] = gates, u_size * torch.randn(3, dim, generator=g, device="cuda")
    x = x.to(TYPES[ty])
    q, s = torch.empty(3, dim, device="cuda", dtype=torch.uint8), torch.empty(3, dim // 128, device="cuda")
    ops.swiglu_fp8_dev(x.data_ptr(), 3, dim, q.data_ptr(), s.data_ptr(), ty, stream=torch.cuda.current_stream().cuda_stream)
    gd, u = x.double().chunk(2, 1)
    y = gd / (1 + torch.exp(-gd)) * u
    off = (2.0**-20 + gd.abs().clamp_max(200) * 2.0**-23) * y.abs() + torch.where(gd < -87, gd.abs().clamp_max(200) * u.abs() * 2.0**-126, 0.0)
    off[:, :128] = 0  # (at -1e30 nothing is left of it, in 64 bits either)
    most = torch.nn.functional.max_pool1d((y.abs() + off)[:, None], 128)[:, 0] / 448
    least = torch.nn.functional.max_pool1d((y.abs() - off).clamp_min(0)[:, None], 128)[:, 0] / 448
    assert (s <= most.clamp_min(2.0**-100) * (1 + 2.0**-21)).all() and (s >= least.clamp_min(2.0**-100) * (1 - 2.0**-21)).all()
    step = torch.maximum(2.0**-4 * (y.abs() + off), 2.0**-10 * s.double().repeat_interleave(128, 1)) * (1 + 2.0**-20)
    assert ((held(q, s) - y).abs() <= step + off).all()


@pytest.mark.parametrize("gate,up", [("inf", 1.0), ("-inf", 1.0), ("nan", 1.0), ("inf", 0.0), (0.0, "inf"), (-200.0, "inf"), (3.0, "-inf"), (3.0, "nan"), (100.0, 3e38)])
def test_swiglu_of_what_is_not_finite_reaches_its_block(gate, up):
    x = torch.ones(3, 800, device="cuda")
    x[1, 130], x[1, 530] = float(gate), float(up)
    q, s = torch.empty(3, 400, device="cuda", dtype=torch.uint8), torch.empty(3, 4, device="cuda")
    ops.swiglu_fp8_dev(x.data_ptr(), 3, 400, q.data_ptr(), s.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
    assert not torch.isfinite(s[1, 1]) and torch.isnan(held(q, s)[1, 128:256]).all()
    s[1, 1] = 1.0
    v = held(q, s)
    v[1, 128:256] = 1 / (1 + np.exp(-1.0))
    assert ((v - 1 / (1 + np.exp(-1.0))).abs() <= 2.0**-4).all()

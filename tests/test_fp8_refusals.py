"""What the operators on fp8 rows and token distributions refuse before any device work (checked without a GPU)."""
import ctypes as C

import numpy as np
import pytest

from sapient_b200 import _lib, ops

OK, SHAPE, DTYPE, ARG, VOCAB = _lib.SP_OK, _lib.SP_ERR_SHAPE, _lib.SP_ERR_DTYPE, _lib.SP_ERR_ARG, _lib.SP_ERR_VOCAB
F32, BF16 = ops.F32, ops.BF16
P = 1 << 20  # an address that nothing is read from: every call below ends before


def _norm(x=P, ldx=256, res=0, ldr=256, total=0, lds=256, w=P, rows=2, dim=256, q=P, scale=P, dtype=F32):
    return _lib.lib().sp_cuda_rms_norm_fp8_dev(0, dtype, x, ldx, res, ldr, total, lds, w, 1e-5, rows, dim, q, scale, None)


@pytest.mark.parametrize("status,kw", [
    (ARG, {"x": 0}), (ARG, {"q": 0}), (ARG, {"scale": 0}), (ARG, {"x": P + 8}), (ARG, {"q": P + 8}), (ARG, {"w": P + 4}), (ARG, {"scale": P + 2}),
    (ARG, {"res": P + 8}), (ARG, {"total": P + 8}), (ARG, {"total": P, "lds": 512}), (ARG, {"res": 2 * P, "total": 2 * P, "ldr": 512}),
    (SHAPE, {"dim": 0}), (SHAPE, {"dim": -16}), (SHAPE, {"dim": 24}), (SHAPE, {"dim": 32784, "ldx": 32784}), (SHAPE, {"rows": -1}), (SHAPE, {"ldx": 240}),
    (SHAPE, {"ldx": 258}), (SHAPE, {"res": P, "ldr": 255}), (SHAPE, {"total": 2 * P, "lds": 16}), (SHAPE, {"dtype": BF16, "ldx": 260}),
    (DTYPE, {"dtype": ops.F16}), (DTYPE, {"dtype": 99}), (OK, {"rows": 0}), (OK, {"rows": 0, "w": 0, "dtype": BF16})])
def test_rms_norm_fp8(status, kw):
    assert _norm(**kw) == status


@pytest.mark.parametrize("fn,wide", [("sp_cuda_swiglu_fp8_dev", 2), ("sp_cuda_quant_fp8_dev", 1)])
def test_rows_to_fp8(fn, wide):
    f = getattr(_lib.lib(), fn)
    call = lambda x=P, ld=wide * 64, rows=3, dim=64, q=P, s=P, dtype=F32: f(0, dtype, x, ld, rows, dim, q, s, None)  # noqa: E731
    assert [call(x=0), call(q=0), call(s=0), call(x=P + 4), call(q=P + 8)] == [ARG] * 5
    assert [call(dim=8), call(dim=0), call(rows=-1), call(ld=wide * 64 - 4), call(ld=wide * 64 + 2), call(ld=wide * 64 + 4, dtype=BF16)] == [SHAPE] * 6
    assert call(dtype=ops.Q8_0) == DTYPE and call(rows=0) == OK


def test_matmul_fp8():
    f = _lib.lib().sp_cuda_matmul_fp8_dev
    call = lambda xq=P, xs=P, m=4, wq=P, ws=P, n=8, k=32, y=P, dtype=F32, ldy=8: f(0, xq, xs, m, wq, ws, n, k, y, dtype, ldy, None)  # noqa: E731
    assert [call(**{a: 0}) for a in ("xq", "xs", "wq", "ws", "y")] == [ARG] * 5
    assert [call(xq=P + 8), call(wq=P + 4), call(xs=P + 2), call(ws=P + 1), call(y=P + 2), call(y=P + 1, dtype=BF16)] == [ARG] * 6
    assert [call(k=0), call(k=40), call(m=-1), call(n=-1), call(ldy=7), call(m=1 << 31), call(n=1 << 31, ldy=1 << 31), call(k=1 << 31)] == [SHAPE] * 8
    assert call(dtype=ops.F16) == DTYPE and call(m=0) == OK and call(n=0, ldy=0) == OK


def test_logprobs_dev():
    f = _lib.lib().sp_cuda_logprobs_dev
    call = lambda z=P, ld=100, rows=2, n=100, ids=P, top=3, lp=P, dtype=F32: f(0, dtype, z, ld, rows, n, ids, top, lp, P, P, P, None)  # noqa: E731
    assert [call(z=0), call(ids=0), call(top=-1), call(top=33), call(n=2, top=3), call(z=P + 2), call(z=P + 1, dtype=BF16)] == [ARG] * 7
    assert [call(n=0), call(rows=-1), call(ld=99), call(n=(1 << 30) + 1, ld=1 << 31)] == [SHAPE] * 4
    assert call(dtype=ops.F16) == DTYPE and call(rows=0) == OK


def test_host_forms():
    x = np.zeros((2, 64), np.float32)
    q, xs = np.zeros((2, 64), np.uint8), np.ones((2, 1), np.float32)
    w, ws = np.zeros((130, 64), np.uint8), np.ones((2, 1), np.float32)
    refused = [(SHAPE, lambda: ops.rms_norm_fp8(x[:, :24], None, 1e-5)), (SHAPE, lambda: ops.rms_norm_fp8(x[0], None, 1e-5)),
               (SHAPE, lambda: ops.rms_norm_fp8(x, np.ones(32), 1e-5)), (SHAPE, lambda: ops.rms_norm_fp8(x, None, 1e-5, residual=x[:1])),
               (SHAPE, lambda: ops.swiglu_fp8(x[:, :63])), (SHAPE, lambda: ops.swiglu_fp8(x[:, :48])), (SHAPE, lambda: ops.quant_fp8(x[:, :40])),
               (SHAPE, lambda: ops.matmul_fp8(q, xs, w, ws[:1])), (SHAPE, lambda: ops.matmul_fp8(q, xs[:1], w, ws)), (SHAPE, lambda: ops.matmul_fp8(q[:, :32], xs, w, ws)),
               (SHAPE, lambda: ops.matmul_fp8(q[:, :40], xs, w[:, :40], ws)), (SHAPE, lambda: ops.Weight.from_fp8(w, ws[:1])),
               (SHAPE, lambda: ops.Weight.from_fp8(w[:, :40], ws)), (SHAPE, lambda: ops.Weight.from_fp8(w[0], ws)),
               (SHAPE, lambda: ops.logprobs(x, [1])), (SHAPE, lambda: ops.logprobs(x[0], [1])), (ARG, lambda: ops.logprobs(x, [0, 1], top=33)),
               (ARG, lambda: ops.logprobs(x, [0, 1], top=-1)), (ARG, lambda: ops.logprobs(x[:, :4], [0, 1], top=5)), (VOCAB, lambda: ops.logprobs(x, [0, 64]))]
    for status, call in refused:
        with pytest.raises(_lib.SapientCudaError) as e:
            call()
        assert e.value.status == status
    h = C.c_void_p()
    p = x.ctypes.data_as(C.c_void_p)
    assert _lib.lib().sp_cuda_upload_weight_fp8(0, 4, 64, None, p, C.byref(h)) == ARG
    assert _lib.lib().sp_cuda_upload_weight_fp8(0, 0, 64, p, p, C.byref(h)) == SHAPE
    # no block of raw ggml bytes has this type
    assert _lib.lib().sp_cuda_upload_weight(0, ops.F8_E4M3, 4, 64, p, 256, C.byref(h)) == DTYPE


def test_nothing_to_do_needs_no_device():
    q, s, h = ops.rms_norm_fp8(np.zeros((0, 64), np.float32), None, 1e-5)
    assert q.shape == (0, 64) and s.shape == (0, 1) and h.shape == (0, 64)
    assert ops.swiglu_fp8(np.zeros((0, 64), np.float32))[0].shape == (0, 32)
    assert ops.matmul_fp8(np.zeros((0, 64), np.uint8), np.zeros((0, 1)), np.zeros((5, 64), np.uint8), np.zeros((1, 1))).shape == (0, 5)
    assert [a.shape for a in ops.logprobs(np.zeros((0, 9)), [], top=2)] == [(0,), (0,), (0, 2), (0, 2)]


def test_values_that_are_not_bytes():
    """A float8 array of any package has items of one byte; floats and integers are not silently taken for bits."""
    x, xs, ws = np.zeros((2, 64), np.uint8), np.ones((2, 1), np.float32), np.ones((1, 1), np.float32)
    for bad in (np.float32, np.int32, np.float16, bool):
        for call in (lambda: ops.matmul_fp8(x.astype(bad), xs, x, ws), lambda: ops.matmul_fp8(x, xs, x.astype(bad), ws), lambda: ops.Weight.from_fp8(x.astype(bad), ws)):
            with pytest.raises(_lib.SapientCudaError) as e:
                call()
            assert e.value.status == DTYPE


def test_arguments_reach_the_library_as_ctypes_would_pass_them():
    """The module between Python and the library: the same statuses as ctypes, integers of any package, None for no address; what is no
    number, does not fit or is one too few raises."""
    c, L = _lib.calls(), _lib.lib()
    norm = [0, F32, P, 256, 0, 256, 0, 256, P, 1e-5, 2, 256, P, P, 0]
    for at, value in [(1, 99), (2, 0), (2, P + 8), (3, 240), (6, P), (10, -1), (11, 24), (11, 1 << 40), (12, None), (10, 0), (10, np.int64(0)), (3, np.int32(255))]:
        a = list(norm)
        a[at] = value
        if a[10] == 2 and at == 6:
            a[7] = 512
        assert c.rms_norm_fp8(*a) == L.sp_cuda_rms_norm_fp8_dev(*[None if v is None else v if isinstance(v, float) else int(v) for v in a])
        assert a[10] == 0 or c.rms_norm_fp8(*a) != OK
    assert c.matmul_fp8(0, P, P, 0, P, P, 8, 32, P, F32, 8, None) == OK and c.matmul_fp8(0, P, P, 4, P, P, 8, 32, P, F32, 7, 0) == SHAPE
    assert c.swiglu_fp8(0, F32, P, 128, 0, 64, P, P, 0) == OK and c.quant_fp8(0, F32, P, 64, 0, 64, P, P, 0) == OK
    assert c.logprobs(0, F32, P, 100, 2, 100, 0, 33, 0, P, P, P, 0) == ARG
    if hasattr(c, "bind"):  # (ctypes takes a number modulo 2^32)
        for bad, error in [((0, 1 << 40, P, 64, 0, 64, P, P, 0), OverflowError), ((0, F32, "x", 64, 0, 64, P, P, 0), TypeError), ((0, F32, P, 64.0, 0, 64, P, P, 0), TypeError),
                           ((0, F32, P, 64, 0, 64, P, P), TypeError), ((0, F32, P, 1 << 80, 0, 64, P, P, 0), OverflowError)]:
            with pytest.raises(error):
                c.quant_fp8(*bad)


def test_addresses_of_distributions():
    """Of each array the call writes or reads: addresses inside a value would fault."""
    f = _lib.lib().sp_cuda_logprobs_dev
    call = lambda ids=P, lp=P, ent=P, ti=P, tl=P: f(0, F32, P, 100, 2, 100, ids, 3, lp, ent, ti, tl, None)  # noqa: E731
    for name in ("ids", "lp", "ent", "ti", "tl"):
        assert [call(**{name: P + off}) for off in (1, 2, 3)] == [ARG] * 3


def test_more_rows_than_bytes_can_be_counted():
    """Host forms multiply sizes before they allocate: products past 64 bits are refused, not taken modulo them."""
    x = np.zeros((2, 64), np.float32)
    p, L = x.ctypes.data_as(C.c_void_p), _lib.lib()
    for rows, dim in [(1 << 60, 16), ((1 << 62) + 1, 64), ((1 << 63) - 1, 32768)]:
        assert L.sp_cuda_rms_norm_fp8(0, p, None, None, rows, dim, 1e-5, p, p, p) == SHAPE
        assert L.sp_cuda_quant_fp8(0, p, rows, dim, p, p) == SHAPE and L.sp_cuda_swiglu_fp8(0, p, rows, dim, p, p) == SHAPE
    for m, n, k in [(1 << 60, 2, 16), (2, 1 << 60, 16), (1 << 31, 2, 16), (2, 1 << 31, 16), ((1 << 62) + 1, (1 << 62) + 1, 64)]:
        assert L.sp_cuda_matmul_fp8(0, p, p, m, p, p, n, k, p) == SHAPE


def test_ids_that_are_none():
    """A token id is a whole number of 32 bits: others are not cut down to one."""
    x = np.zeros((2, 64), np.float32)
    for status, ids in [(VOCAB, [-1, 0]), (VOCAB, np.array([0, (1 << 32) + 5])), (VOCAB, np.array([0, -(1 << 32)])), (VOCAB, np.array([1 << 63, 0], np.uint64)),
                        (DTYPE, [0.0, 1.5]), (DTYPE, np.array([True, False])), (DTYPE, ["1", "2"]), (DTYPE, [1 << 70, 0])]:
        with pytest.raises(_lib.SapientCudaError) as e:
            ops.logprobs(x, ids)
        assert e.value.status == status

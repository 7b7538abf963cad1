"""Per-op interface of the CUDA backend on host (numpy) buffers, mirroring the
reference's `LlmBackend` trait (crates/sapient-models/src/forward/backend.rs:57-115)
and the resident-weight kernel API of its GPU context
(crates/sapient-backends/wgpu/src/quant.rs:94-480). Every call goes through the C ABI.
"""
from __future__ import annotations

import ctypes as C

import numpy as np

from . import _lib
from ._lib import SapientCudaError, check, lib

F32, F16, Q4_0, Q8_0, Q4_K, Q5_K, Q6_K, BF16 = 0, 1, 2, 8, 12, 13, 14, 30
F8_E4M3 = 128      # Weight.from_fp8
FP8_BLOCK = 128    # columns of an fp8 row, rows and columns of an fp8 weight, that share a scale
LOGPROBS_MAX_TOP = 32


def _p(a: np.ndarray):
    return a.ctypes.data_as(C.c_void_p)


def _blocks(k: int) -> int:
    return -(-k // FP8_BLOCK)


def _bits8(a, what: str) -> np.ndarray:
    """Values of one byte as they are: a number of another type would not be converted but taken for bits."""
    a = np.asarray(a)
    if a.dtype.itemsize != 1 or a.dtype.kind == "b":
        raise SapientCudaError(_lib.SP_ERR_DTYPE, f"{what}: e4m3 values are given as bytes (uint8), not {a.dtype}")
    return np.ascontiguousarray(a).view(np.uint8)


def _ids32(a, what: str) -> np.ndarray:
    """Token ids as they are: a number that is none is not cut down to one."""
    a = np.asarray(a).reshape(-1)
    if a.size and a.dtype.kind not in "iu":
        raise SapientCudaError(_lib.SP_ERR_DTYPE, f"{what}: ids are whole numbers, not {a.dtype}")
    if a.size and (a.min() < 0 or a.max() > 0xFFFFFFFF):
        raise SapientCudaError(_lib.SP_ERR_VOCAB, f"{what}: token id out of vocab range")
    return np.ascontiguousarray(a, dtype=np.uint32)


def _f32(a) -> np.ndarray:
    return np.ascontiguousarray(a, dtype=np.float32)


class Weight:
    """A [n, k] matrix of raw ggml blocks resident on the device (upload_q8_0 / upload_q4_k / upload_q6_k)."""

    def __init__(self, dtype: int, n: int, k: int, blocks, device: int = 0):
        raw = np.ascontiguousarray(blocks, dtype=np.uint8).reshape(-1)
        h = C.c_void_p()
        check(lib().sp_cuda_upload_weight(device, dtype, n, k, _p(raw), raw.size, C.byref(h)))
        self.h, self.dtype, self.n, self.k, self.device, self.nbytes = h, dtype, n, k, device, raw.size

    @classmethod
    def from_fp8(cls, values, scales, device: int = 0) -> "Weight":
        """An [n, k] matrix of e4m3 values (uint8: their bits) with an f32 scale for every 128 x 128 block. matmul_nt quantises the
        rows of x likewise, a scale for every 128 columns."""
        v, s = _bits8(values, "fp8 weight"), _f32(scales)
        if v.ndim != 2 or s.shape != (_blocks(v.shape[0]), _blocks(v.shape[1])):
            raise SapientCudaError(_lib.SP_ERR_SHAPE, "fp8 weight: values [n, k] and scales [ceil(n / 128), ceil(k / 128)] expected")
        h = C.c_void_p()
        check(lib().sp_cuda_upload_weight_fp8(device, *v.shape, _p(v), _p(s), C.byref(h)))
        w = cls.__new__(cls)
        w.h, w.dtype, (w.n, w.k), w.device, w.nbytes = h, F8_E4M3, v.shape, device, v.size
        return w

    def dequant(self) -> np.ndarray:
        """Tensor::to_f32_vec — bit-exact f32 values, shape [n, k]."""
        out = np.empty((self.n, self.k), np.float32)
        check(lib().sp_cuda_dequant(self.h, _p(out)))
        return out

    def matmul_nt(self, x) -> np.ndarray:
        """Y[m, n] = X[m, k] · Wᵀ (kernels::matmul::matmul_nt) with host buffers."""
        x = _f32(x)
        if x.ndim != 2:
            raise SapientCudaError(_lib.SP_ERR_SHAPE, "matmul_nt expects 2-D tensors")
        if x.shape[1] != self.k:
            raise SapientCudaError(_lib.SP_ERR_SHAPE, f"shape mismatch: expected [{x.shape[0]}, {x.shape[1]}] got [{self.n}, {self.k}]")
        y = np.empty((x.shape[0], self.n), np.float32)
        check(lib().sp_cuda_matmul_nt(self.h, _p(x), x.shape[0], _p(y)))
        return y

    def matmul_nt_dev(self, x_ptr: int, m: int, y_ptr: int, stream: int = 0) -> None:
        """Device-pointer variant (no copies, no synchronisation)."""
        check(lib().sp_cuda_matmul_nt_dev(self.h, C.c_void_p(x_ptr), m, C.c_void_p(y_ptr), C.c_void_p(stream)))

    def embed(self, ids) -> np.ndarray:
        ids = np.ascontiguousarray(ids, dtype=np.uint32).reshape(-1)
        out = np.empty((ids.size, self.k), np.float32)
        check(lib().sp_cuda_embed(self.h, _p(ids), ids.size, _p(out)))
        return out

    def free(self) -> None:
        if getattr(self, "h", None):
            lib().sp_cuda_free_weight(self.h)
            self.h = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass


def matmul_nt(x, blocks, dtype: int, n: int, device: int = 0) -> np.ndarray:
    x = _f32(x)
    if x.ndim != 2:
        raise SapientCudaError(_lib.SP_ERR_SHAPE, "matmul_nt expects 2-D tensors")
    w = Weight(dtype, n, x.shape[1], blocks, device)
    try:
        return w.matmul_nt(x)
    finally:
        w.free()


def rms_norm(x, w, eps: float, device: int = 0) -> np.ndarray:
    x = _f32(x)
    rows, dim = int(np.prod(x.shape[:-1])), x.shape[-1]
    y = np.empty_like(x)
    wv = _f32(w) if w is not None else None
    check(lib().sp_cuda_rms_norm(device, _p(x), _p(wv) if wv is not None else None, rows, dim, eps, _p(y)))
    return y


def layer_norm(x, w, b, eps: float, device: int = 0) -> np.ndarray:
    x = _f32(x)
    rows, dim = int(np.prod(x.shape[:-1])), x.shape[-1]
    y = np.empty_like(x)
    wv = _f32(w) if w is not None else None
    bv = _f32(b) if b is not None else None
    check(lib().sp_cuda_layer_norm(device, _p(x), _p(wv) if wv is not None else None, _p(bv) if bv is not None else None,
                                   rows, dim, eps, _p(y)))
    return y


def rope(x, positions, base: float, rotary_dim: int | None = None, device: int = 0) -> np.ndarray:
    """apply_rope_positions / apply_rope_partial on x [n_heads, seq, head_dim]."""
    x = _f32(x)
    H, S, D = x.shape
    pos = np.ascontiguousarray(positions, dtype=np.int64)
    if pos.size != S:
        raise SapientCudaError(_lib.SP_ERR_SHAPE, "positions length must match seq_len")
    y = np.empty_like(x)
    check(lib().sp_cuda_rope(device, _p(x), H, S, D, _p(pos), base, D if rotary_dim is None else rotary_dim, _p(y)))
    return y


def gqa_attention(q, k, v, device: int = 0) -> np.ndarray:
    """Causal GQA attention: q [H, sq, hd], k/v [Hkv, sk, hd] -> [H, sq, hd]. K/V are held as fp16 on the device."""
    q, k, v = _f32(q), _f32(k), _f32(v)
    H, sq, hd = q.shape
    Hkv, sk, _ = k.shape
    out = np.empty_like(q)
    check(lib().sp_cuda_attention(device, _p(q), _p(k), _p(v), H, Hkv, sq, sk, hd, _p(out)))
    return out


def _unary(fn, x, device):
    x = _f32(x)
    y = np.empty_like(x)
    check(fn(device, _p(x), x.size, _p(y)))
    return y


def silu(x, device: int = 0):
    return _unary(lib().sp_cuda_silu, x, device)


def gelu(x, device: int = 0):
    return _unary(lib().sp_cuda_gelu, x, device)


def add(a, b, device: int = 0):
    a, b = _f32(a), _f32(b)
    y = np.empty_like(a)
    check(lib().sp_cuda_add(device, _p(a), _p(b), a.size, _p(y)))
    return y


def mul(a, b, device: int = 0):
    a, b = _f32(a), _f32(b)
    y = np.empty_like(a)
    check(lib().sp_cuda_mul(device, _p(a), _p(b), a.size, _p(y)))
    return y


def argmax(logits, device: int = 0) -> np.ndarray:
    """Row-wise argmax; ties resolve to the last maximum (Sampler's greedy rule)."""
    x = _f32(logits)
    x2 = x.reshape(-1, x.shape[-1])
    out = np.empty(x2.shape[0], np.uint32)
    check(lib().sp_cuda_argmax(device, _p(x2), x2.shape[0], x2.shape[1], _p(out)))
    return out


# ── 8-bit floating-point rows and token distributions (no counterpart in the reference; formats in include/sapient_cuda.h) ──
def _rows2(x, what: str) -> np.ndarray:
    x = _f32(x)
    if x.ndim != 2:
        raise SapientCudaError(_lib.SP_ERR_SHAPE, f"{what} expects 2-D arrays")
    return x


def _fp8_out(rows: int, dim: int):
    return np.empty((rows, dim), np.uint8), np.empty((rows, _blocks(dim)), np.float32)


def rms_norm_fp8(x, w, eps: float, residual=None, device: int = 0):
    """RMS norm of h = x + residual as fp8 rows: (q [rows, dim] uint8, scale [rows, ceil(dim / 128)], h)."""
    x = _rows2(x, "rms_norm_fp8")
    r, wv = None if residual is None else _f32(residual), None if w is None else _f32(w)
    if (r is not None and r.shape != x.shape) or (wv is not None and wv.shape != x.shape[1:]):
        raise SapientCudaError(_lib.SP_ERR_SHAPE, "rms_norm_fp8: residual like x and w [dim] expected")
    (q, s), h = _fp8_out(*x.shape), np.empty_like(x)
    check(lib().sp_cuda_rms_norm_fp8(device, _p(x), None if r is None else _p(r), None if wv is None else _p(wv), *x.shape, eps, _p(q), _p(s), _p(h)))
    return q, s, h


def swiglu_fp8(gu, device: int = 0):
    """silu(gate) * up of rows gate | up as fp8 rows: (q, scale)."""
    gu = _rows2(gu, "swiglu_fp8")
    if gu.shape[1] % 2:
        raise SapientCudaError(_lib.SP_ERR_SHAPE, "swiglu_fp8: gate and up side by side expected")
    q, s = _fp8_out(gu.shape[0], gu.shape[1] // 2)
    check(lib().sp_cuda_swiglu_fp8(device, _p(gu), *q.shape, _p(q), _p(s)))
    return q, s


def quant_fp8(x, device: int = 0):
    """x as fp8 rows: (q, scale)."""
    x = _rows2(x, "quant_fp8")
    q, s = _fp8_out(*x.shape)
    check(lib().sp_cuda_quant_fp8(device, _p(x), *x.shape, _p(q), _p(s)))
    return q, s


def matmul_fp8(xq, xs, wq, ws, device: int = 0) -> np.ndarray:
    """Y[m, n] = X Wᵀ of fp8 rows (xq [m, k] uint8, xs [m, ceil(k / 128)]) and fp8 weights (wq [n, k], ws for 128 x 128 blocks)."""
    xq, wq = _bits8(xq, "matmul_fp8"), _bits8(wq, "matmul_fp8")
    xs, ws = _f32(xs), _f32(ws)
    if xq.ndim != 2 or wq.ndim != 2 or xq.shape[1] != wq.shape[1]:
        raise SapientCudaError(_lib.SP_ERR_SHAPE, "matmul_fp8 expects xq [m, k] and wq [n, k]")
    (m, k), n = xq.shape, wq.shape[0]
    if xs.shape != (m, _blocks(k)) or ws.shape != (_blocks(n), _blocks(k)):
        raise SapientCudaError(_lib.SP_ERR_SHAPE, "matmul_fp8: a scale for every 128 columns of a row and 128 x 128 block of the weights expected")
    y = np.empty((m, n), np.float32)
    check(lib().sp_cuda_matmul_fp8(device, _p(xq), _p(xs), m, _p(wq), _p(ws), n, k, _p(y)))
    return y


def logprobs(logits, ids, top: int = 0, device: int = 0):
    """(log probability of ids[row], entropy, top_ids [rows, top], top_logprobs [rows, top]) of rows of logits; among equal logits the
    lowest id comes first. ids may be None, the first of the four is then, too."""
    z = _rows2(logits, "logprobs")
    rows = z.shape[0]
    i = None if ids is None else _ids32(ids, "logprobs")
    if i is not None and i.size != rows:
        raise SapientCudaError(_lib.SP_ERR_SHAPE, "logprobs: one id per row expected")
    if not 0 <= top <= LOGPROBS_MAX_TOP:
        raise SapientCudaError(_lib.SP_ERR_ARG, "logprobs: top must be 0 to 32 and at most the vocabulary")
    lp, ent = np.empty(rows, np.float32), np.empty(rows, np.float32)
    ti, tl = np.empty((rows, top), np.uint32), np.empty((rows, top), np.float32)
    check(lib().sp_cuda_logprobs(device, _p(z), *z.shape, None if i is None else _p(i), top, None if i is None else _p(lp), _p(ent), _p(ti), _p(tl)))
    return None if i is None else lp, ent, ti, tl


# The same on device pointers (integers; 0: not given), without copies or synchronisation. dtype: F32 or BF16. Row strides in values, 0: dense.
def rms_norm_fp8_dev(x: int, rows: int, dim: int, w: int, eps: float, q: int, scale: int, dtype: int = F32, residual: int = 0, sum_out: int = 0,
                     ldx: int = 0, ldr: int = 0, lds: int = 0, device: int = 0, stream: int = 0) -> None:
    status = (_lib._calls or _lib.calls()).rms_norm_fp8(device, dtype, x, ldx or dim, residual, ldr or dim, sum_out, lds or dim, w, eps, rows, dim, q, scale, stream)
    if status:
        check(status)


def swiglu_fp8_dev(gu: int, rows: int, ffn: int, q: int, scale: int, dtype: int = F32, ld: int = 0, device: int = 0, stream: int = 0) -> None:
    status = (_lib._calls or _lib.calls()).swiglu_fp8(device, dtype, gu, ld or 2 * ffn, rows, ffn, q, scale, stream)
    if status:
        check(status)


def quant_fp8_dev(x: int, rows: int, dim: int, q: int, scale: int, dtype: int = F32, ldx: int = 0, device: int = 0, stream: int = 0) -> None:
    status = (_lib._calls or _lib.calls()).quant_fp8(device, dtype, x, ldx or dim, rows, dim, q, scale, stream)
    if status:
        check(status)


def matmul_fp8_dev(xq: int, xs: int, m: int, wq: int, ws: int, n: int, k: int, y: int, dtype: int = F32, ldy: int = 0, device: int = 0,
                   stream: int = 0) -> None:
    status = (_lib._calls or _lib.calls()).matmul_fp8(device, xq, xs, m, wq, ws, n, k, y, dtype, ldy or n, stream)
    if status:
        check(status)


def logprobs_dev(logits: int, rows: int, vocab: int, ids: int, logprob: int, entropy: int, top: int = 0, top_ids: int = 0, top_logprobs: int = 0,
                 dtype: int = F32, ld: int = 0, device: int = 0, stream: int = 0) -> None:
    status = (_lib._calls or _lib.calls()).logprobs(device, dtype, logits, ld or vocab, rows, vocab, ids, top, logprob, entropy, top_ids, top_logprobs, stream)
    if status:
        check(status)


def set_gemv_path(path: int) -> None:
    """0: tensor-core GEMV on tile-repacked weights (default); 1: CUDA-core GEMV on raw blocks; 3: per-warp streaming
    variant; 4: bulk-copy ring GEMV for calls of 1-5 rows."""
    check(lib().sp_cuda_set_gemv_path(path))


LARGE_M_DEFAULT = 2


def set_large_m_gemm(on) -> None:
    """Op-level matmuls with m >= 17 and k % 256 == 0: 2 (default) the tcgen05 / TMEM dequant GEMM with exact-class operands
    (activations as leading part + remainder, weights unrounded); 1 / True the one with operands rounded to fp16; 0 / False exact integer-digit passes
    on the mma.sync kernels."""
    check(lib().sp_cuda_set_large_m_gemm(int(on)))


def launch_count() -> int:
    return int(lib().sp_cuda_launch_count())

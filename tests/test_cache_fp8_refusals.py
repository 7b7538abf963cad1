"""What the calls on a paged cache of 8-bit rows refuse, before any device work, and the table of angles."""
import ctypes as C

import numpy as np
import pytest

from sapient_b200 import _lib, ops
from sapient_b200._lib import SP_ERR_ARG, SP_ERR_CUDA, SP_ERR_DTYPE, SP_ERR_SHAPE, SapientCudaError

A = 1 << 20  # an address that starts on 16 bytes; no call here looks at it


def cache(**kw):
    d = dict(values=A, scales=A, page_table=A, n_pages=4, n_slots=2, max_pages=3, n_kv_heads=2, head_dim=64)
    return ops.CacheFp8(**(d | kw))


def refused(status, fn, *args, **kw):
    with pytest.raises(SapientCudaError) as e:
        fn(*args, **kw)
    assert e.value.status == status, e.value


def append(c=None, **kw):
    d = dict(n_tok=1, slots=A, positions=A, k=A, v=A, q=A, n_heads=4, q_out=A + 4096, angles=A, n_angles=10, rotary_dim=64)
    ops.cache_fp8_append_dev(c or cache(), **(d | kw))


def read(c=None, **kw):
    ops.cache_fp8_read_dev(c or cache(), **(dict(n_tok=1, slots=A, positions=A, k=A, v=A) | kw))


def attention(c=None, **kw):
    d = dict(q=A, n_heads=4, out=A + 4096, n_seqs=1, row_start=A, seq_len=A, max_rows=1, max_len=10, scale=0.1)
    ops.attention_fp8_dev(c or cache(), **(d | kw))


@pytest.mark.parametrize("call", [append, read, attention])
def test_caches(call):
    for kw in (dict(values=0), dict(scales=0), dict(page_table=0), dict(values=A + 8), dict(scales=A + 4), dict(page_table=A + 2)):
        refused(SP_ERR_ARG, call, cache(**kw))
    for kw in (dict(head_dim=0), dict(head_dim=40), dict(head_dim=144), dict(head_dim=-16), dict(n_pages=0), dict(n_slots=0), dict(max_pages=0), dict(n_kv_heads=0),
               dict(max_pages=2**31 - 1), dict(n_kv_heads=70000)):
        refused(SP_ERR_SHAPE, call, cache(**kw))
    for kw in (dict(n_pages=2**26, n_kv_heads=1), dict(n_pages=1025, n_kv_heads=65535)):  # n_pages x 2 x n_kv_heads x 16 >= 2^31
        refused(SP_ERR_SHAPE, call, cache(**kw))
    for ty in (ops.F16, 99, -1):
        refused(SP_ERR_DTYPE, call, dtype=ty)
    assert _lib.lib().sp_cuda_cache_fp8_read_dev(None, 0, 1, A, A, A, 128, A, 128, None) == SP_ERR_ARG


def test_append():
    for kw in (dict(slots=0), dict(positions=0), dict(k=0), dict(v=0), dict(q_out=0), dict(slots=A + 1), dict(k=A + 8), dict(v=A + 4), dict(q=A + 2), dict(q_out=A + 8),
               dict(angles=A + 8), dict(q_w=A + 4), dict(k_w=A + 8), dict(angles=0), dict(n_angles=0), dict(q=0), dict(q=0, n_heads=0), dict(q_out=A, ldqo=264)):
        refused(SP_ERR_ARG, append, **kw)
    for kw in (dict(n_tok=-1), dict(n_tok=2**31), dict(n_heads=3), dict(n_heads=0), dict(n_heads=-2), dict(ldk=64), dict(ldv=130), dict(ldq=255), dict(ldqo=100),
               dict(rotary_dim=8), dict(rotary_dim=80), dict(rotary_dim=-16)):
        refused(SP_ERR_SHAPE, append, **kw)
    refused(SP_ERR_SHAPE, append, dtype=ops.BF16, ldk=132)
    st = _lib.lib().sp_cuda_cache_fp8_append_dev(cache().at, 0, 1, A, A, A, 256, 4, A + 4096, 256, A, 128, A, 128, None, None, 0.0, A, 10, 64, 2, None)
    assert st == SP_ERR_ARG


def test_read():
    for kw in (dict(slots=0), dict(positions=0), dict(positions=A + 3), dict(k=A + 8), dict(v=A + 1)):
        refused(SP_ERR_ARG, read, **kw)
    for kw in (dict(n_tok=-1), dict(n_tok=2**31), dict(ldk=120), dict(ldv=129)):
        refused(SP_ERR_SHAPE, read, **kw)


def test_attention():
    for kw in (dict(q=0), dict(out=0), dict(row_start=0), dict(seq_len=0), dict(q=A + 8), dict(out=A + 8), dict(row_start=A + 2), dict(seq_len=A + 1), dict(seq_slot=A + 2),
               dict(window=-1), dict(scale=float("nan")), dict(scale=float("inf")), dict(out=A, ldo=260)):
        refused(SP_ERR_ARG, attention, **kw)
    for kw in (dict(n_heads=3), dict(n_heads=0), dict(n_heads=-4), dict(ldq=128), dict(ldo=258), dict(n_seqs=-1), dict(n_seqs=65536), dict(max_rows=-1), dict(max_len=-1),
               dict(max_rows=2**29)):
        refused(SP_ERR_SHAPE, attention, **kw)


def test_calls_that_do_nothing_need_no_device():
    append(n_tok=0)
    read(n_tok=0)
    read(k=0, v=0)
    attention(n_seqs=0)
    attention(max_rows=0)


def test_without_a_device_they_fail():
    if _lib.lib().sp_cuda_device_count() == 0:
        for call in (append, read, attention):
            refused(SP_ERR_CUDA, call)


def test_struct_layout_matches_header():
    assert C.sizeof(_lib.SpCacheFp8) == 3 * 8 + 6 * 4
    assert ops.cache_fp8_bytes(3, 2, 80) == (3 * 2 * 2 * 16 * 80, 3 * 2 * 2 * 16 * 4)


def test_angles():
    t = ops.rope_table(5000, 64, 10000.0)
    assert t.shape == (5000, 32, 2) and t.dtype == np.float32
    i, p = np.arange(32), np.arange(5000)[:, None]
    f = 10000.0 ** (-i / 32)
    assert np.abs(t[..., 0] - np.cos(p * f)).max() <= 2.0**-24 and np.abs(t[..., 1] - np.sin(p * f)).max() <= 2.0**-24
    assert np.abs(ops.rope_table(100, 64, 10000.0, factor=4.0) - ops.rope_table(25, 64, 10000.0).repeat(4, 0))[::4].max() <= 2.0**-23  # every frequency divided
    s = ops.rope_table(2, 64, 10000.0, factor=8.0, original=4096)
    turns = 4096 * f / (2 * np.pi)
    got = np.arctan2(s[1, :, 1], s[1, :, 0])
    want = np.where(turns >= 1, f, np.where(turns <= 0.25, f / 8, f * (turns - 0.25) / 0.75 + f / 8 * (1 - (turns - 0.25) / 0.75)))
    assert np.abs(got - want).max() <= 2.0**-22
    assert ((turns > 0.25) & (turns < 1)).any()  # some lie between
    assert ops.rope_table(3, 0, 10000.0).shape == (3, 0, 2) and ops.rope_table(0, 4, 10.0).shape == (0, 2, 2)
    refused(SP_ERR_SHAPE, ops.rope_table, 3, 5, 10.0)
    refused(SP_ERR_SHAPE, ops.rope_table, -1, 4, 10.0)
    refused(SP_ERR_ARG, ops.rope_table, 3, 4, 10.0, factor=0.0)
    refused(SP_ERR_ARG, ops.rope_table, 3, 4, 10.0, original=10, low=1.0, high=1.0)

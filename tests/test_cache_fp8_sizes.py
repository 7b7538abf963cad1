"""Sizes and addresses of a cache of 8-bit rows that its description cannot hold are refused, not cut down to those it can."""
import pytest

from sapient_b200 import ops
from sapient_b200._lib import SP_ERR_ARG, SP_ERR_SHAPE, SapientCudaError

GOOD = dict(values=1 << 20, scales=1 << 20, page_table=1 << 20, n_pages=4, n_slots=2, max_pages=3, n_kv_heads=2, head_dim=64, device=0)


@pytest.mark.parametrize("name", ["n_pages", "n_slots", "max_pages", "n_kv_heads", "head_dim", "device"])
def test_sizes(name):
    for n in (2**31, 2**32 + GOOD[name], 2**63, -(2**31) - 1, -(2**32) + GOOD[name]):
        with pytest.raises(SapientCudaError) as e:
            ops.CacheFp8(**(GOOD | {name: n}))
        assert e.value.status == SP_ERR_SHAPE
    assert getattr(ops.CacheFp8(**GOOD).desc, name) == GOOD[name]


@pytest.mark.parametrize("name", ["values", "scales", "page_table"])
def test_addresses(name):
    for at in (2**64 + (1 << 20), -16):
        with pytest.raises(SapientCudaError) as e:
            ops.CacheFp8(**(GOOD | {name: at}))
        assert e.value.status == SP_ERR_ARG

"""Appending heads at the ends of the norm's range: zeros, which are 0 / 0 without eps, and the smallest and largest that the header names."""
import math

import pytest
import torch

from cache_fp8_tools import STEP, TYPES, Cache, ints, normed64
from sapient_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("dim", [16, 80, 128])
def test_ends_of_the_range(dim, ty):
    c = Cache([16], 1, dim, 1)
    x = torch.randn(4, 3 * dim, device="cuda").clamp(-4, 4)
    x[:, :2 * dim] *= torch.tensor([0.0, 1.0, 2.0**-61, 2.0**60 / math.sqrt(dim)], device="cuda")[:, None]
    x[2, :2 * dim] += torch.copysign(torch.tensor(2.0**-62, device="cuda"), x[2, :2 * dim])  # mean(x^2) above 2^-126
    x = x.to(TYPES[ty])
    w = 0.5 + torch.rand(dim, device="cuda")
    q_out = torch.empty(4, dim, device="cuda", dtype=TYPES[ty])
    slot, pos, size = ints([0] * 4), ints(range(4)), x.element_size()
    for eps in (0.0, 1e-5):
        ops.cache_fp8_append_dev(c.own, 4, slot.data_ptr(), pos.data_ptr(), x.data_ptr() + dim * size, x.data_ptr() + 2 * dim * size, q=x.data_ptr(), n_heads=1, q_out=q_out.data_ptr(),
                                 q_w=w.data_ptr(), k_w=w.data_ptr(), eps=eps, dtype=ty, ldq=3 * dim, ldk=3 * dim, ldv=3 * dim)
        k = c.rows(0, 4, 0)[:, 0]
        want_q, want_k = (normed64(x[:, i * dim: (i + 1) * dim].double(), w, eps) for i in (0, 1))
        some = slice(1, 4) if eps == 0 else slice(0, 4)
        # the norm's factor: 2^-19 (its sum, rsqrtf, products), q rounded to its type; k off by half a step of e4m3 as well, 2^-4 of the value or 2^-10 of the scale
        assert ((q_out.double() - want_q).abs() <= (2.0**-19 + STEP[ty]) * want_q.abs())[some].all()
        scale = want_k.abs().amax(-1, keepdim=True) / 448
        assert ((k - want_k).abs() <= torch.maximum(want_k.abs() * 2.0**-4, scale * 2.0**-10) + scale * 448 * 2.0**-18)[some].all()
        if eps == 0:
            assert q_out[0].isnan().all() and k[0].isnan().all()
        else:
            assert (q_out[0] == 0).all() and (k[0] == 0).all()
        assert c.rows(0, 4, 1).isfinite().all()

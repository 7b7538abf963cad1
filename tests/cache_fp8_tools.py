"""A paged cache of 8-bit rows for tests, the same computations in 64 bits, and how far the calls may be off."""
import math

import torch

from sapient_b200 import ops

PAGE = 16
TYPES = {ops.F32: torch.float32, ops.BF16: torch.bfloat16}
STEP = {ops.F32: 2.0**-24, ops.BF16: 2.0**-8}  # half a step, relative


def ints(v, device="cuda"):
    return torch.tensor(v, dtype=torch.int32, device=device)


class Cache:
    """Slots with room for `room` tokens each, on pages in no order; three pages belong to nobody."""

    def __init__(self, room, kv, dim, seed=0, max_pages=None, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        held = [-(-n // PAGE) for n in room]
        self.kv, self.dim, self.n_slots = kv, dim, len(room)
        self.max_pages = max_pages or max(1, max(held))
        self.n_pages = sum(held) + 3
        order = torch.randperm(self.n_pages, generator=g, device=device).int()
        self.table = torch.full((self.n_slots, self.max_pages), -1, dtype=torch.int32, device=device)
        at = 0
        for i, h in enumerate(held):
            self.table[i, :h] = order[at: at + h]
            at += h
        y = torch.randn(self.n_pages, 2, kv, PAGE, dim, generator=g, device=device)
        y[:, 1] *= torch.exp(torch.randn(self.n_pages, kv, PAGE, 1, generator=g, device=device))
        self.scales = y.abs().amax(-1) / 448
        self.values = (y / self.scales.unsqueeze(-1)).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
        self.own = ops.CacheFp8(self.values.data_ptr(), self.scales.data_ptr(), self.table.data_ptr(), self.n_pages, self.n_slots, self.max_pages, kv, dim)

    def rows(self, slot, n, which):
        """Keys (0) or values (1) of a slot's first n tokens in 64 bits, [n, kv, dim]; NaN where there is no page."""
        page = self.table[slot].long().repeat_interleave(PAGE)[:n]
        there = (page >= 0) & (page < self.n_pages)
        token = torch.arange(page.numel(), device=page.device) % PAGE
        at = torch.where(there, page, 0)
        y = self.values[at, which, :, token].view(torch.float8_e4m3fn).double() * self.scales[at, which, :, token].double().unsqueeze(-1)
        y[~there] = math.nan
        return y


def attention64(c, q, seqs, scale, window=0, digits=False):
    """seqs: (slot, rows, length) of each sequence; q [rows, heads, dim]. Outputs in 64 bits and how far a call's may be off. digits: with what
    bf16 queries as two e4m3 digits add, which counts where a few coordinates are much larger than the others."""
    heads, dim = q.shape[1:]
    group = heads // c.kv
    out, far = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    f32, at = q.dtype == torch.float32, 0
    for slot, r, n in seqs:
        held = min(n, c.max_pages * PAGE)
        if r and held > 0 and 0 <= slot < c.n_slots:
            k, v = c.rows(slot, held, 0), c.rows(slot, held, 1)
            page = c.table[slot].long().repeat_interleave(PAGE)[:held]
            pos = torch.arange(n - r, n, device=q.device)[:, None]
            key = torch.arange(held, device=q.device)[None]
            seen = (key <= pos) & (page >= 0) & (page < c.n_pages)
            if window:
                seen &= key > pos - window
            for h in range(heads):
                x = q[at: at + r, h].double()
                z = (x @ k[:, h // group].nan_to_num().T) * scale
                z = torch.where(seen & k[:, h // group].isnan().any(-1), math.nan, z)  # (a key that is no number, seen)
                p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
                p[~seen.any(-1)] = 0
                bad = seen & v[:, h // group].isnan().any(-1)
                u = v[:, h // group].nan_to_num()
                y = p @ u
                y[bad.any(-1)] = math.nan
                y[z.isnan().any(-1)] = math.nan
                out[at: at + r, h] = y
                # Scores: q rounded to 22 bits (bf16: exact), dim / 16 additions of the tensor cores (a plane), which cut off up to 2^-23 of the
                # terms' sum each, and four roundings in f32 of z, its scale and its distance to m (in units of log 2: 1.45 |z| 2^-24 each).
                # Weights: that, ex2's 2^-22 and two roundings. Sums: an addition for 16 keys and a plane, the accumulators' and the parts' factors (2^-22
                # each, of which 64 at most). All of it in numerator and denominator, hence twice; relative to sums of absolute values. In the
                # numerator alone: f32: weights as fp16 + fp16 of the remainder (2^-22). bf16: fp16 of the weight, of the value's
                # factor and of their product with the value, which is exact before: half a step of fp16 is 2^-11 of the value, so (1 + 2^-11)^3 - 1.
                planes = 2 if f32 else 1
                size = (x.abs() @ k[:, h // group].nan_to_num().abs().T * scale).masked_fill(~seen, 0).amax(-1, keepdim=True)
                dz = size * (2.0**-22 * f32 + planes * dim / 16 * 2.0**-23 + 6 * 2.0**-23) + 2.0**-21
                if digits:  # the lowest digit's step is 2^-9 where the row's largest value is 2^7 or more: each coordinate is off by 2^-17 of that
                    dz = dz + 1.45 * scale * 2.0**-17 * x.abs().amax(-1, keepdim=True) * (k[:, h // group].nan_to_num().abs().sum(-1) * seen).amax(-1, keepdim=True)
                w = 2 * (dz + planes * (held / 16 + 2) * 2.0**-23 + 64 * 2.0**-22) + (2.0**-22 if f32 else (1 + 2.0**-11) ** 3 - 1)
                far[at: at + r, h] = w * (p @ u.abs()) + (2 * STEP[ops.F32] if f32 else 1.01 * STEP[ops.BF16]) * y.abs() + 2.0**-100
        at += r
    return out, far


class Step:
    """New tokens of sequences: q, out and what describes them."""

    def __init__(self, c, seqs, heads, ty, seed=0, size=1.5, ld=None):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.c, self.seqs, self.heads, self.ty = c, seqs, heads, ty
        n, wide = sum(r for _, r, _ in seqs), heads * c.dim
        self.ld = ld or wide
        self.q = (size * torch.randn(max(n, 1), self.ld, generator=g, device="cuda")).to(TYPES[ty])
        self.out = torch.full((n + 2, self.ld), 7.0, device="cuda", dtype=TYPES[ty])  # two rows behind the last
        start = [0]
        for _, r, _ in seqs:
            start.append(start[-1] + r)
        self.n, self.start, self.len, self.slot = n, ints(start), ints([x for _, _, x in seqs]), ints([s for s, _, _ in seqs])
        self.max_rows, self.max_len = max(r for _, r, _ in seqs), max(0, max(x for _, _, x in seqs))

    def run(self, scale=None, window=0, max_rows=None, max_len=None, stream=None, empty=0, out=None):
        """empty: sequences without rows or tokens behind the others."""
        st = torch.cuda.current_stream().cuda_stream if stream is None else stream
        start, length, slot = self.start, self.len, self.slot
        if empty:
            start, length, slot = (torch.cat([x, last.expand(empty)]) for x, last in ((start, start[-1:]), (length, ints([0])), (slot, ints([0]))))
        out = self.out if out is None else out
        ops.attention_fp8_dev(self.c.own, self.q.data_ptr(), self.heads, out.data_ptr(), len(self.seqs) + empty, start.data_ptr(), length.data_ptr(),
                              self.max_rows if max_rows is None else max_rows, self.max_len if max_len is None else max_len,
                              self.c.dim**-0.5 if scale is None else scale, window=window, seq_slot=slot.data_ptr(), dtype=self.ty, ldq=self.ld, ldo=self.ld, stream=st)
        return out

    def check(self, scale=None, window=0, digits=False):
        """What is in out, and what the call leaves where large bounds, or sequences with nothing to do, make it share the work out otherwise."""
        wide = self.heads * self.c.dim
        q = self.q[: self.n, :wide].reshape(self.n, self.heads, self.c.dim)
        want, far = attention64(self.c, q, self.seqs, self.c.dim**-0.5 if scale is None else scale, window, digits)
        outs = {"as asked": self.out}
        some = 128 * self.c.kv // self.heads  # tokens with which a key head has 128 rows
        for name, most, empty in (("many rows", 4096, 0), ("many sequences", 1, 64), ("some rows of many", some, 70), ("some rows of some", some, 18)):
            outs[name] = self.run(scale, window, max(most, self.max_rows), empty=empty, out=torch.full_like(self.out, 7.0))
        for name, out in outs.items():
            got = out[: self.n, :wide].reshape(want.shape).double()
            assert torch.equal(got.isnan(), want.isnan()), name
            off = (got - want).abs().nan_to_num()
            assert (off <= far.nan_to_num(nan=1.0)).all(), f"{name}: off by {float((off / far.nan_to_num(nan=1.0)).max())} of what it may be"
            assert (out[self.n:] == 7).all() and (out[:, wide:] == 7).all(), name  # what is behind the last row and beside the heads


def rotated64(x, angles, rotary, pairs):
    """x [n, heads, dim] with angles [n, rotary / 2, 2]."""
    a, b = (slice(0, rotary, 2), slice(1, rotary, 2)) if pairs else (slice(0, rotary // 2), slice(rotary // 2, rotary))
    c, s = angles[:, None, :, 0].double(), angles[:, None, :, 1].double()
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def normed64(x, w, eps):
    return x if w is None else x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()

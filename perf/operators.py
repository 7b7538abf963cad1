"""What the operators around 8-bit rows cost: RMS norm (with the residual's addition) and SwiGLU that leave e4m3 rows with a
scale for every 128 columns, the matrix product of such rows with e4m3 weights that carry a scale for every 128 x 128 block,
and log probabilities of given tokens with entropy and top alternatives. Cases, inputs, the plain forms, the framework's
calls, what a pass cannot do without, and the same in 64 bits.
"""
import math

import torch

own = False  # set by the tool that measures: the framework's kernels, or the plain forms

BLOCK = 128            # columns that share a scale
E4M3_MAX = 448.0       # largest value of the format
SCALE_MIN = 2.0**-100  # a block of zeros keeps this scale
EPS = 1e-5
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}


def listed():
    return [
        # a decoded token between two layers of an 8B-shaped model, stream in f32
        {"name": "norm 1x4096 f32", "kind": "norm", "rows": 1, "dim": 4096, "type": "f32", "residual": True},
        # a ragged prompt ahead of a 2560-wide model's first layer: nothing to add
        {"name": "norm 301x2560 bf16", "kind": "norm", "rows": 301, "dim": 2560, "type": "bf16", "residual": False},
        # prompts of several sequences in one step
        {"name": "norm 8192x4096 bf16", "kind": "norm", "rows": 8192, "dim": 4096, "type": "bf16", "residual": True},
        # a few sequences decoded together, 0.5B shape
        {"name": "swiglu 7x4864 f32", "kind": "swiglu", "rows": 7, "dim": 4864, "type": "f32"},
        # a prompt chunk of the 8B shape
        {"name": "swiglu 4096x14336 bf16", "kind": "swiglu", "rows": 4096, "dim": 14336, "type": "bf16"},
        # one decoded token: attention output projection of the 8B shape
        {"name": "matmul 1x4096x4096 f32", "kind": "matmul", "rows": 1, "n": 4096, "k": 4096, "type": "f32"},
        # decoded tokens of 13 sequences: gate and up of the 8B shape in one matrix
        {"name": "matmul 13x28672x4096 bf16", "kind": "matmul", "rows": 13, "n": 28672, "k": 4096, "type": "bf16"},
        # a ragged prompt, rows and columns that end inside tiles and a last block of 16 columns
        {"name": "matmul 389x8968x2064 f32", "kind": "matmul", "rows": 389, "n": 8968, "k": 2064, "type": "f32"},
        # prompts of several sequences in one step: a projection of the 8B shape
        {"name": "matmul 4096x14336x4096 bf16", "kind": "matmul", "rows": 4096, "n": 14336, "k": 4096, "type": "bf16"},
        # one sampled token of the 1.5B shape's vocabulary, five alternatives
        {"name": "logprobs 1x151936 f32", "kind": "logprobs", "rows": 1, "n": 151936, "type": "f32", "top": 5, "masked": 0.0},
        # a batch whose grammar leaves a tenth of the vocabulary
        {"name": "logprobs 32x128256 bf16", "kind": "logprobs", "rows": 32, "n": 128256, "type": "bf16", "top": 20, "masked": 0.9},
        # scoring a prompt: every position
        {"name": "logprobs 1024x128256 f32", "kind": "logprobs", "rows": 1024, "n": 128256, "type": "f32", "top": 1, "masked": 0.0},
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind, ty = rng.choice(["norm", "swiglu", "matmul", "matmul", "logprobs"]), rng.choice(["f32", "bf16"])
    if kind in ("norm", "swiglu"):
        dim = 16 * _spread(rng, 4, 1024 if kind == "norm" else 1792)
        rows = _spread(rng, 1, max(1, min(16384, (8192 * 4096 if kind == "norm" else 4096 * 14336) * 2 // SIZE[ty] // dim)))
        return {"kind": kind, "rows": rows, "dim": dim, "type": ty} | ({"residual": rng.random() < 0.5} if kind == "norm" else {})
    if kind == "matmul":
        n, k = _spread(rng, 100, 32000), 16 * _spread(rng, 16, 896)
        most = min(8192, 4096 * 14336 * 4096 // (n * k), 4096 * 14336 * 2 // (n * SIZE[ty]))
        return {"kind": kind, "rows": _spread(rng, 1, max(1, most)), "n": n, "k": k, "type": ty}
    n = _spread(rng, 1000, 200000)
    rows = _spread(rng, 1, max(1, min(4096, 1024 * 128256 // n)))
    return {"kind": kind, "rows": rows, "n": n, "type": ty, "top": rng.randint(0, 20), "masked": rng.choice([0.0, 0.0, 0.5, 0.95])}


# ── inputs ──────────────────────────────────────────────────────────────────
def _blocks(y):
    """[rows, blocks, 128], the last block filled up with zeros."""
    rows, dim = y.shape
    return torch.nn.functional.pad(y, (0, -dim % BLOCK)).view(rows, -1, BLOCK)


def _scales(y):
    return (_blocks(y).abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)


def _over_scales(y, s):
    return (_blocks(y) / s.unsqueeze(-1)).reshape(y.shape[0], -1)[:, : y.shape[1]]


def _e4m3_rows(y):
    s = _scales(y)
    return _over_scales(y, s).to(torch.float8_e4m3fn).contiguous(), s


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, rows, ty = case["kind"], case["rows"], TYPES[case["type"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    s = {"kind": kind, "rows": rows, "type": case["type"], "stream": torch.cuda.current_stream().cuda_stream}
    if kind in ("norm", "swiglu"):
        dim = case["dim"]
        s |= {"dim": dim, "q": torch.empty(rows, dim, device="cuda", dtype=torch.float8_e4m3fn), "scale": torch.empty(rows, -(-dim // BLOCK), device="cuda")}
    if kind == "norm":
        # a stream whose columns have scales of their own, one in a hundred much larger
        col = 0.5 + torch.rand(dim, generator=g, device="cuda") + 20 * (torch.rand(dim, generator=g, device="cuda") < 0.01)
        s["w"] = 0.5 + torch.rand(dim, generator=g, device="cuda")
        s["x"] = (normal(rows, dim) * (0.3 if case["residual"] else col)).to(ty)
        s["residual"] = (normal(rows, dim) * col).to(ty) if case["residual"] else None
        s["sum"] = torch.empty_like(s["x"]) if case["residual"] else None
    elif kind == "swiglu":
        s["x"] = (2 * normal(rows, 2 * dim)).to(ty)
    elif kind == "matmul":
        n, k = case["n"], case["k"]
        s |= {"n": n, "k": k}
        s["xq"], s["xs"] = _e4m3_rows(normal(rows, k))
        # weights as they are kept: e4m3 values that fill the format's range, and the blocks' scales
        s["wq"] = (120 * normal(n, k)).clamp(-E4M3_MAX, E4M3_MAX).to(torch.float8_e4m3fn)
        s["ws"] = (0.5 + torch.rand(-(-n // BLOCK), -(-k // BLOCK), generator=g, device="cuda")) * (0.02 / 120)
        s["y"] = torch.empty(rows, n, device="cuda", dtype=ty)
    else:
        n, top = case["n"], case["top"]
        z = 3 * normal(rows, n)
        z[:, : min(64, n)] += 6 * torch.rand(rows, min(64, n), generator=g, device="cuda")
        ids = torch.randint(0, n, (rows,), generator=g, device="cuda")
        if case["masked"]:
            out = torch.rand(rows, n, generator=g, device="cuda") < case["masked"]
            out.scatter_(1, ids[:, None], False)  # the given token is one that the mask allows
            z.masked_fill_(out, -math.inf)
        s |= {"n": n, "top": top, "z": z.to(ty), "ids": ids.int(), "logprob": torch.empty(rows, device="cuda"), "entropy": torch.empty(rows, device="cuda"),
              "top_ids": torch.empty(rows, top, device="cuda", dtype=torch.int32), "top_logprobs": torch.empty(rows, top, device="cuda")}
    return s


# ── one pass ────────────────────────────────────────────────────────────────
def run(s):
    return _calls(s) if own else _plain(s)


def _calls(s):
    from sapient_b200 import ops

    kind, ty = s["kind"], ops.F32 if s["type"] == "f32" else ops.BF16
    if kind == "norm":
        res, total = s["residual"], s["sum"]
        ops.rms_norm_fp8_dev(s["x"].data_ptr(), s["rows"], s["dim"], s["w"].data_ptr(), EPS, s["q"].data_ptr(), s["scale"].data_ptr(), dtype=ty,
                             residual=0 if res is None else res.data_ptr(), sum_out=0 if total is None else total.data_ptr(), stream=s["stream"])
        return {"q": s["q"], "scale": s["scale"]} | ({} if total is None else {"sum": total})
    if kind == "swiglu":
        ops.swiglu_fp8_dev(s["x"].data_ptr(), s["rows"], s["dim"], s["q"].data_ptr(), s["scale"].data_ptr(), dtype=ty, stream=s["stream"])
        return {"q": s["q"], "scale": s["scale"]}
    if kind == "matmul":
        ops.matmul_fp8_dev(s["xq"].data_ptr(), s["xs"].data_ptr(), s["rows"], s["wq"].data_ptr(), s["ws"].data_ptr(), s["n"], s["k"], s["y"].data_ptr(),
                           dtype=ty, stream=s["stream"])
        return s["y"]
    ops.logprobs_dev(s["z"].data_ptr(), s["rows"], s["n"], s["ids"].data_ptr(), s["logprob"].data_ptr(), s["entropy"].data_ptr(), top=s["top"],
                     top_ids=s["top_ids"].data_ptr(), top_logprobs=s["top_logprobs"].data_ptr(), dtype=ty, stream=s["stream"])
    return {k: s[k] for k in ("logprob", "entropy") + (("top_ids", "top_logprobs") if s["top"] else ())}


def _plain(s):
    kind = s["kind"]
    if kind == "norm":
        h = s["x"].float() if s["residual"] is None else s["x"].float() + s["residual"].float()
        q, scale = _e4m3_rows(h * torch.rsqrt(h.square().mean(-1, keepdim=True) + EPS) * s["w"])
        return {"q": q, "scale": scale} | ({} if s["residual"] is None else {"sum": h.to(s["x"].dtype)})
    if kind == "swiglu":
        g, u = s["x"].float().chunk(2, -1)
        q, scale = _e4m3_rows(g / (1 + torch.exp(-g)) * u)
        return {"q": q, "scale": scale}
    if kind == "matmul":
        x, w = _held(s["xq"], s["xs"], 1, torch.float32), _held(s["wq"], s["ws"], BLOCK, torch.float32)
        return (x @ w.T).to(TYPES[s["type"]])
    return _distribution(s["z"], s["ids"], s["top"])


def _held(q, scale, height, ty):
    """The values that 8-bit blocks of `height` rows x 128 columns stand for."""
    each = scale.to(ty).repeat_interleave(height, 0)[: q.shape[0]].repeat_interleave(BLOCK, 1)[:, : q.shape[1]]
    return q.to(ty) * each


def _distribution(z, ids, top):
    """In 64 bits: a likely token's log probability is the difference of nearly equal numbers. Among equal logits the lowest
    index comes first."""
    d = z.double()
    m = d.amax(-1, keepdim=True)
    e = torch.exp(d - m)
    total = e.sum(-1, keepdim=True)
    lp = d - m - torch.log(total)
    out = {"logprob": lp.gather(1, ids.long()[:, None])[:, 0].float(), "entropy": -(e / total * torch.where(e > 0, lp, 0.0)).sum(-1).float()}
    if top:
        at = torch.sort(z, dim=-1, descending=True, stable=True).indices[:, :top]
        out |= {"top_ids": at.int(), "top_logprobs": lp.gather(1, at).float()}
    return out


# ── what a pass cannot do without ───────────────────────────────────────────
def work(case):
    kind, rows, size = case["kind"], case["rows"], SIZE[case["type"]]
    if kind in ("norm", "swiglu"):
        dim = case["dim"]
        out = rows * (dim + 4 * -(-dim // BLOCK))
        if kind == "norm":
            return {"bytes": rows * dim * size * (3 if case["residual"] else 1) + 4 * dim + out, "flops": 6 * rows * dim}
        return {"bytes": 2 * rows * dim * size + out, "flops": 6 * rows * dim}
    n = case["n"]
    if kind == "matmul":
        k = case["k"]
        nb = -(-k // BLOCK)
        return {"bytes": (rows + n) * k + 4 * nb * (rows + -(-n // BLOCK)) + rows * n * size, "flops": 2 * rows * n * k}
    return {"bytes": rows * (n * size + 12 + 8 * case["top"]), "flops": 4 * rows * n}


# ── the same in 64 bits ─────────────────────────────────────────────────────
def exact(case, seed):
    """From the definitions. 8-bit values: what they would be before the rounding to e4m3, so that a side's distance is that of
    the format and a value next to a border of its grid, which 32 bits put on either side of it, changes nothing."""
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("norm", "swiglu"):
        x, dim = s["x"].double(), case["dim"]
        if kind == "norm":
            h = x if s["residual"] is None else x + s["residual"].double()
            y = h / ((h * h).sum(-1, keepdim=True) / dim + EPS).sqrt() * s["w"].double()
        else:
            y = x[:, :dim] * x[:, dim:] / (1 + (-x[:, :dim]).exp())
        q, scale = torch.empty_like(y), torch.empty(y.shape[0], -(-dim // BLOCK), device=y.device, dtype=torch.float64)
        for b in range(scale.shape[1]):
            part = y[:, BLOCK * b: BLOCK * (b + 1)]
            scale[:, b] = (part.abs().max(-1).values / E4M3_MAX).clamp(min=SCALE_MIN)
            q[:, BLOCK * b: BLOCK * (b + 1)] = part / scale[:, b: b + 1]
        return {"q": q, "scale": scale} | ({"sum": h} if kind == "norm" and case["residual"] else {})
    if kind == "matmul":
        y = torch.zeros(case["rows"], case["n"], device="cuda", dtype=torch.float64)
        rows_of = torch.arange(case["n"], device="cuda") // BLOCK
        for b in range(s["xs"].shape[1]):
            cols = slice(BLOCK * b, BLOCK * (b + 1))
            y += (s["xq"][:, cols].double() @ s["wq"][:, cols].double().T) * s["xs"][:, b: b + 1].double() * s["ws"][rows_of, b].double()
        return y
    out = {k: [] for k in ("logprob", "entropy") + (("top_ids", "top_logprobs") if case["top"] else ())}
    for z, i in zip(s["z"], s["ids"].tolist()):
        z = z.double()
        lse = torch.logsumexp(z, 0)
        p = torch.exp(z - lse)
        out["logprob"].append(z[i] - lse)
        out["entropy"].append(-(p * (z - lse))[p > 0].sum())
        if case["top"]:
            best = torch.topk(z, min(case["n"], case["top"])).values
            out["top_logprobs"].append(best - lse)
            out["top_ids"].append(None)
    return {k: None if k == "top_ids" else torch.stack(v) for k, v in out.items()}

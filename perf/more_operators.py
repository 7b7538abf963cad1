"""What the operators around a paged cache of 8-bit rows cost: norms of queries and keys for each head and the position rotation in the
pass that writes keys and values into the cache, attention of new tokens (one, a few, a chunk, a whole prompt) over that cache, and
reading it back. Cases, inputs, the plain forms, the framework's calls, what a pass cannot do without, and the same in 64 bits.

The cache: pages of 16 tokens, values[page][key | value][head][token][head_dim] in e4m3, scales[page][key | value][head][token] in f32:
a token's head is a row of 8-bit values with one scale, max |y| / 448. page_table[slot][i] is the page of a slot's tokens 16 i to 16 i + 15.
"""
import math
import random

import torch

own = False  # set by the tool that measures: the framework's kernels, or the plain forms

PAGE = 16              # tokens of a page
E4M3_MAX = 448.0       # largest value of the format
SCALE_MIN = 2.0**-100  # a row of zeros keeps this scale
EPS = 1e-6
BASE = 500000.0
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "bf16": 2}
MOST_PAIRS = 8192 * 8192 * 32  # padded scores of a pass: the largest listed case


def listed():
    big = {"heads": 32, "kv": 8, "dim": 128}    # the 8B shape
    mid = {"heads": 12, "kv": 2, "dim": 128}    # the 1.5B shape
    small = {"heads": 14, "kv": 2, "dim": 64}   # the 0.5B shape
    equal = {"heads": 32, "kv": 32, "dim": 80}  # a 2.7B shape without shared heads
    return [
        # a decoded token between projections and attention
        {"name": "append 1 8B bf16", "kind": "append", **big, "seqs": 1, "rows": 1, "len": 518, "mix": 0, "type": "bf16", "rotary": 128, "pairs": False, "norms": False, "stretch": 1},
        # a ragged prompt of a small model with norms of queries and keys, neighbours rotated
        {"name": "append 301 0.5B f32", "kind": "append", **small, "seqs": 1, "rows": 301, "len": 301, "mix": 0, "type": "f32", "rotary": 64, "pairs": True, "norms": True, "stretch": 1},
        # prompts of several sequences in one step, far positions of a stretched context
        {"name": "append 8192 8B bf16", "kind": "append", **big, "seqs": 6, "rows": 1365, "len": 120000, "mix": 0, "type": "bf16", "rotary": 128, "pairs": False, "norms": True, "stretch": 8},
        # one decoded token of a short conversation, rows in f32 as the engine keeps them
        {"name": "decode 1x518 8B f32", "kind": "attention", **big, "seqs": 1, "rows": 1, "len": 518, "mix": 0, "type": "f32", "window": 0},
        # a decoded token for each of 32 conversations of different lengths
        {"name": "decode 32x8192 8B bf16", "kind": "attention", **big, "seqs": 32, "rows": 1, "len": 8192, "mix": 1, "type": "bf16", "window": 0},
        # a decoded token behind a very long document
        {"name": "decode 1x131072 8B bf16", "kind": "attention", **big, "seqs": 1, "rows": 1, "len": 131072, "mix": 0, "type": "bf16", "window": 0},
        # drafted tokens of several sequences verified together, a model with a window
        {"name": "verify 13x5 1.5B f32", "kind": "attention", **mid, "seqs": 13, "rows": 5, "len": 2001, "mix": 2, "type": "f32", "window": 1024},
        # a chunk of a prompt behind what is in the cache already
        {"name": "chunk 512 at 8704 8B bf16", "kind": "attention", **big, "seqs": 1, "rows": 512, "len": 8704, "mix": 0, "type": "bf16", "window": 0},
        # packed prompts of different lengths, a head width that is no power of two
        {"name": "prompts 9x1500 2.7B bf16", "kind": "attention", **equal, "seqs": 9, "rows": 1500, "len": 0, "mix": 3, "type": "bf16", "window": 0},
        # a long prompt
        {"name": "prompt 8192 8B bf16", "kind": "attention", **big, "seqs": 1, "rows": 8192, "len": 0, "mix": 0, "type": "bf16", "window": 0},
        # a page of a small model, for a shared prefix that moves to another engine
        {"name": "read 16 0.5B f32", "kind": "read", **small, "seqs": 1, "rows": 16, "len": 301, "mix": 0, "type": "f32"},
        # conversations that leave the cache for host memory
        {"name": "read 65536 8B bf16", "kind": "read", **big, "seqs": 8, "rows": 8192, "len": 8192, "mix": 0, "type": "bf16"},
    ]


def _spread(rng, low, high):
    """A whole number, even over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind, ty = rng.choice(["append", "attention", "attention", "attention", "read"]), rng.choice(["f32", "bf16"])
    dim, kv = rng.choice([64, 128, 128, 16 * rng.randint(2, 8)]), rng.choice([1, 2, 4, 8, rng.randint(1, 16)])
    heads = kv * rng.choice([1, 2, 4, 8, rng.randint(1, 16)])
    c = {"kind": kind, "heads": heads, "kv": kv, "dim": dim, "mix": rng.randint(1, 10**6), "type": ty}
    width = (heads + 2 * kv) * dim
    if kind == "append":
        total = _spread(rng, 1, max(1, min(16384, 8190 * 48 * 128 * 2 // (width * SIZE[ty]))))
        seqs = rng.randint(1, min(total, 64))
        c |= {"seqs": seqs, "rows": total // seqs, "len": total // seqs + _spread(rng, 1, 100000), "rotary": rng.choice([dim, dim, 16 * rng.randint(0, dim // 16)]),
              "pairs": rng.random() < 0.4, "norms": rng.random() < 0.5, "stretch": rng.choice([1, 1, 4, 8])}
        return c
    if kind == "read":
        total = _spread(rng, 1, max(1, min(131072, 65536 * 8 * 128 * 2 // (kv * dim * SIZE[ty]))))
        seqs = rng.randint(1, min(total, 64))
        return c | {"seqs": seqs, "rows": total // seqs, "len": total // seqs + _spread(rng, 1, 2000)}
    c["window"] = rng.choice([0, 0, 0, _spread(rng, 1, 4096)])
    form = rng.choice(["decode", "decode", "verify", "chunk", "prompt"])
    if form in ("decode", "verify"):
        c |= {"seqs": _spread(rng, 1, 64), "rows": 1 if form == "decode" else rng.randint(2, 16)}
        most = min(131072, 2 * 131072 * 8 * 128 // (c["seqs"] * kv * dim), MOST_PAIRS // (c["seqs"] * heads * c["rows"]))
        c["len"] = max(c["rows"], _spread(rng, 1, max(1, most)))
        return c
    if form == "prompt":
        seqs = _spread(rng, 1, 16)
        rows = _spread(rng, 1, max(1, min(8192, 65536 * 32 * 128 // (seqs * heads * dim), int(math.sqrt(MOST_PAIRS / (seqs * heads) * min(1, 128 / dim))))))
        return c | {"seqs": seqs, "rows": rows, "len": 0}
    seqs, rows = _spread(rng, 1, 8), _spread(rng, 16, 1024)
    most = min(65536, MOST_PAIRS // 2 // (seqs * rows * heads), 2 * 131072 * 8 * 128 // (seqs * kv * dim))
    return c | {"seqs": seqs, "rows": rows, "len": max(rows, _spread(rng, rows, max(rows, most)))}


def _shape(case):
    """(new tokens, length with them) of each sequence, from the case alone. mix 0: all alike, as stated; else ragged, the stated
    figures the largest, and in a batch of four or more one sequence that has nothing new."""
    n, rows, length, mix = case["seqs"], case["rows"], case["len"], case["mix"]
    if not mix:
        return [(rows, length or rows)] * n
    rng, out = random.Random(mix), []
    for i in range(n):
        r = rows if i == 0 or rows <= 16 else rng.randint(max(1, rows // 8), rows)
        out.append((r, r if not length else max(r, length if i == 0 else rng.randint(max(1, length // 8), length))))
    if n >= 4 and case["kind"] == "attention" and mix % 3 == 1:
        out[2] = (0, out[2][1])
    return out


def _freqs(case):
    """Angles of a position, in 64 bits; for a stretched context those of more than a turn in the original 8192 tokens stay, those of
    less than a quarter are divided, between them it goes over."""
    d = case["rotary"]
    f = BASE ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / max(d, 1))
    if case["stretch"] == 1:
        return f
    turns = 8192 * f / (2 * math.pi)
    keep = ((turns - 0.25) / 0.75).clamp(0, 1)
    return f * keep + f / case["stretch"] * (1 - keep)


# ── inputs ──────────────────────────────────────────────────────────────────
def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, heads, kv, dim, ty = case["kind"], case["heads"], case["kv"], case["dim"], TYPES[case["type"]]
    normal = lambda *shape: torch.randn(*shape, generator=g, device="cuda")  # noqa: E731
    ints = lambda v: torch.tensor(v, device="cuda", dtype=torch.int32)  # noqa: E731
    shape = _shape(case)
    first = [0 if kind == "read" else length - rows for rows, length in shape]
    # a slot's tokens lie on pages anywhere in the pool; slots that only write have no pages for what is far behind them
    low = [p // PAGE if kind == "append" else 0 for p in first]
    held = [-(-length // PAGE) - lo for (_, length), lo in zip(shape, low)]
    max_pages = max(1, max(lo + h for lo, h in zip(low, held)))
    pages = torch.randperm(max(1, sum(held)) + 3, generator=g, device="cuda").int()
    table = torch.zeros(len(shape), max_pages, device="cuda", dtype=torch.int32)
    at = 0
    for i, (lo, h) in enumerate(zip(low, held)):
        table[i, lo: lo + h] = pages[at: at + h]
        at += h
    n_pages, rows = pages.numel(), sum(r for r, _ in shape)
    values = normal(n_pages, 2, kv, PAGE, dim)
    # a head's keys have columns of their own size and some that stand out; values differ in size from token to token
    values[:, 0] *= 0.5 + torch.rand(kv, 1, dim, generator=g, device="cuda") + 4 * (torch.rand(kv, 1, dim, generator=g, device="cuda") < 0.02)
    values[:, 1] *= torch.exp(0.5 * normal(n_pages, kv, PAGE, 1))
    scales = _scales(values)
    values = torch.div(values, scales.unsqueeze(-1)).to(torch.float8_e4m3fn)
    s = {"kind": kind, "heads": heads, "kv": kv, "dim": dim, "type": case["type"], "rows": rows, "seqs": len(shape), "values": values, "scales": scales, "table": table,
         "stream": torch.cuda.current_stream().cuda_stream}
    if kind == "attention":
        start = [0]
        for r, _ in shape:
            start.append(start[-1] + r)
        q = 1.5 * normal(max(1, rows), heads * dim)[:rows]
        s |= {"q": q.to(ty), "out": torch.empty(rows, heads * dim, device="cuda", dtype=ty), "row_start": ints(start), "seq_len": ints([n for _, n in shape]),
              "most_rows": max(r for r, _ in shape), "most_len": max(n for _, n in shape), "window": case["window"], "scale": dim**-0.5}
        return s
    slot = torch.arange(len(shape), device="cuda", dtype=torch.int32).repeat_interleave(ints([r for r, _ in shape]))
    pos = torch.cat([torch.arange(p, p + r, device="cuda", dtype=torch.int32) for p, (r, _) in zip(first, shape)])
    s |= {"slot": slot, "pos": pos}
    if kind == "read":
        return s | {"k": torch.empty(rows, kv * dim, device="cuda", dtype=ty), "v": torch.empty(rows, kv * dim, device="cuda", dtype=ty)}
    # queries, keys and values side by side as a projection leaves them
    col = 0.5 + torch.rand((heads + 2 * kv) * dim, generator=g, device="cuda")
    s |= {"qkv": (normal(rows, (heads + 2 * kv) * dim) * col).to(ty), "q_out": torch.empty(rows, heads * dim, device="cuda", dtype=ty)}
    s |= {"q_w": 0.5 + torch.rand(dim, generator=g, device="cuda"), "k_w": 0.5 + torch.rand(dim, generator=g, device="cuda")} if case["norms"] else {"q_w": None, "k_w": None}
    freqs = _freqs(case)
    # cosines and sines of every position, which a program makes once for a model
    angle = torch.arange(max(n for _, n in shape), device="cuda", dtype=torch.float64)[:, None] * freqs
    s |= {"rotary": case["rotary"], "pairs": case["pairs"], "freqs": freqs, "angles": torch.stack([angle.cos(), angle.sin()], -1).float().contiguous()}
    return s


def _scales(y):
    return (y.abs().amax(-1) / E4M3_MAX).clamp_min(SCALE_MIN)


# ── one pass ────────────────────────────────────────────────────────────────
def run(s):
    if own:
        return _calls(s)
    return {"append": _append, "attention": _attention, "read": _read}[s["kind"]](s)


def _calls(s):
    from sapient_b200 import ops

    cache = s.get("cache")
    if cache is None:  # addresses and sizes, which a program writes down once
        cache = s["cache"] = ops.CacheFp8(s["values"].data_ptr(), s["scales"].data_ptr(), s["table"].data_ptr(), n_pages=s["values"].shape[0], n_slots=s["table"].shape[0],
                                          max_pages=s["table"].shape[1], n_kv_heads=s["kv"], head_dim=s["dim"])
    ty, rows = ops.F32 if s["type"] == "f32" else ops.BF16, s["rows"]
    if s["kind"] == "attention":
        ops.attention_fp8_dev(cache, s["q"].data_ptr(), s["heads"], s["out"].data_ptr(), s["seqs"], s["row_start"].data_ptr(), s["seq_len"].data_ptr(), s["most_rows"],
                              s["most_len"], s["scale"], window=s["window"], dtype=ty, stream=s["stream"])
        return s["out"]
    if s["kind"] == "read":
        ops.cache_fp8_read_dev(cache, rows, s["slot"].data_ptr(), s["pos"].data_ptr(), s["k"].data_ptr(), s["v"].data_ptr(), dtype=ty, stream=s["stream"])
        return {"k": s["k"], "v": s["v"]}
    qkv, wide = s["qkv"], s["qkv"].shape[1]
    at = lambda cols: qkv.data_ptr() + cols * qkv.element_size()  # noqa: E731
    ops.cache_fp8_append_dev(cache, rows, s["slot"].data_ptr(), s["pos"].data_ptr(), at(s["heads"] * s["dim"]), at((s["heads"] + s["kv"]) * s["dim"]), q=at(0),
                             n_heads=s["heads"], q_out=s["q_out"].data_ptr(), q_w=0 if s["q_w"] is None else s["q_w"].data_ptr(),
                             k_w=0 if s["k_w"] is None else s["k_w"].data_ptr(), eps=EPS, angles=s["angles"].data_ptr(), n_angles=s["angles"].shape[0],
                             rotary_dim=s["rotary"], pairs=s["pairs"], dtype=ty, ldq=wide, ldk=wide, ldv=wide, stream=s["stream"])
    return {"q": s["q_out"], "values": s["values"], "scales": s["scales"]}


def _cells(s):
    """Page and token within it of every row."""
    return s["table"][s["slot"].long(), (s["pos"] // PAGE).long()].long(), (s["pos"] % PAGE).long()


def _rotated(x, s):
    """x[rows][heads][dim]; angles in 64 bits."""
    d = s["rotary"]
    if not d:
        return x
    angle = s["pos"].double()[:, None] * s["freqs"]
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if s["pairs"]:
        a, b = x[..., 0:d:2], x[..., 1:d:2]
        return torch.cat([torch.stack([a * c - b * n, b * c + a * n], -1).flatten(-2), x[..., d:]], -1)
    a, b = x[..., : d // 2], x[..., d // 2: d]
    return torch.cat([a * c - b * n, b * c + a * n, x[..., d:]], -1)


def _normed(x, w):
    return x if w is None else x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * w


def _append(s):
    rows, heads, kv, dim = s["rows"], s["heads"], s["kv"], s["dim"]
    q, k, v = s["qkv"].float().view(rows, heads + 2 * kv, dim).split([heads, kv, kv], 1)
    s["q_out"].copy_(_rotated(_normed(q, s["q_w"]), s).reshape(rows, -1))
    y = torch.stack([_rotated(_normed(k, s["k_w"]), s), v], 1)
    scale = _scales(y)
    page, token = _cells(s)
    s["values"].view(torch.uint8)[page, :, :, token] = (y / scale.unsqueeze(-1)).to(torch.float8_e4m3fn).view(torch.uint8)
    s["scales"][page, :, :, token] = scale
    return {"q": s["q_out"], "values": s["values"], "scales": s["scales"]}


def _read(s):
    page, token = _cells(s)
    y = s["values"].view(torch.uint8)[page, :, :, token].view(torch.float8_e4m3fn).float() * s["scales"][page, :, :, token].unsqueeze(-1)
    return {name: y[:, i].reshape(s["rows"], -1).to(TYPES[s["type"]]) for i, name in enumerate(("k", "v"))}


def _attention(s):
    """All sequences side by side, filled up to the longest."""
    heads, kv, dim, seqs, rows, most, length = s["heads"], s["kv"], s["dim"], s["seqs"], s["rows"], s["most_rows"], s["most_len"]
    here = torch.arange(rows, device="cuda")
    start = s["row_start"].long()
    seq = torch.searchsorted(start[1:], here, right=True)
    q = torch.zeros(seqs, most, heads * dim, device="cuda")
    q[seq, here - start[seq]] = s["q"].float()
    q = q.view(seqs, most, kv, heads // kv, dim).permute(0, 2, 3, 1, 4)  # [sequence][key head][its queries][row][dim]
    pages = s["table"][:, : -(-length // PAGE)].long()
    cells = s["values"].view(torch.uint8)[pages].view(torch.float8_e4m3fn).float() * s["scales"][pages].unsqueeze(-1)
    k, v = cells.permute(2, 0, 3, 1, 4, 5).reshape(2, seqs, kv, 1, -1, dim)[..., :length, :]  # [sequence][key head][1][token][dim]
    new = (start[1:] - start[:-1])[:, None]
    pos = (s["seq_len"][:, None] - new + torch.arange(most, device="cuda"))[:, :, None]
    key = torch.arange(length, device="cuda")
    seen = key <= pos
    if s["window"]:
        seen &= key > pos - s["window"]
    z = q @ k.transpose(-1, -2)
    z *= s["scale"]
    z.masked_fill_(~seen[:, None, None], -math.inf)
    m = z.amax(-1, keepdim=True).clamp_min(-1e30)  # (a row that sees nothing: zeros)
    z.sub_(m).exp_()
    total = z.sum(-1, keepdim=True)
    y = z @ v / torch.where(total > 0, total, 1.0)
    y = y.permute(0, 3, 1, 2, 4).reshape(seqs, most, heads * dim)
    return y[seq, here - start[seq]].to(TYPES[s["type"]])


# ── what a pass cannot do without ───────────────────────────────────────────
def work(case):
    heads, kv, dim, size, shape = case["heads"], case["kv"], case["dim"], SIZE[case["type"]], _shape(case)
    rows = sum(r for r, _ in shape)
    cell = 2 * kv * (dim + 4)
    if case["kind"] == "read":
        return {"bytes": rows * (cell + 2 * kv * dim * size + 8), "flops": rows * 2 * kv * dim}
    if case["kind"] == "append":
        angles = len({p for r, n in shape for p in range(n - r, n)}) * case["rotary"] * 4
        return {"bytes": rows * ((2 * heads + 2 * kv) * dim * size + cell + 8) + angles, "flops": rows * (heads + 2 * kv) * dim * 8}
    w = case["window"]
    pairs = keys = 0
    for r, n in shape:
        if r:
            pairs += sum(min(p + 1, w) if w else p + 1 for p in range(n - r, n))
            keys += min(n, w + r - 1) if w else n
    return {"bytes": 2 * rows * heads * dim * size + keys * cell + 12 * len(shape), "flops": 4 * heads * dim * pairs}


# ── the same in 64 bits ─────────────────────────────────────────────────────
def exact(case, seed):
    """From the definitions. 8-bit values: what they would be before the rounding to e4m3, so that a side's distance is that of the
    format and a value next to a border of its grid, which 32 bits put on either side of it, changes nothing."""
    s = prepare(case, seed)
    kind, heads, kv, dim, rows = s["kind"], s["heads"], s["kv"], s["dim"], s["rows"]
    if kind == "attention":
        out = torch.zeros(rows, heads, dim, device="cuda", dtype=torch.float64)
        at = 0
        for i, (r, n) in enumerate(_shape(case)):
            page = s["table"][i, : -(-n // PAGE)].long()
            both = [(s["values"][page, j].double() * s["scales"][page, j].double()[..., None]).transpose(0, 1).reshape(kv, -1, dim)[:, :n] for j in (0, 1)]
            for a in range(0, r, 512):
                b = min(r, a + 512)
                pos = torch.arange(n - r + a, n - r + b, device="cuda")[:, None]
                key = torch.arange(n, device="cuda")[None]
                hidden = (key > pos) | (key <= pos - s["window"] if s["window"] else False)
                for h in range(heads):
                    z = s["q"][at + a: at + b, h * dim: (h + 1) * dim].double() @ both[0][h // (heads // kv)].T * s["scale"]
                    out[at + a: at + b, h] = torch.softmax(z.masked_fill(hidden, -math.inf), -1) @ both[1][h // (heads // kv)]
            at += r
        return out.reshape(rows, -1)
    if kind == "read":
        k, v = (torch.empty(rows, kv, dim, device="cuda", dtype=torch.float64) for _ in range(2))
        for y, j in ((k, 0), (v, 1)):
            for h in range(kv):
                at = s["table"][s["slot"].long(), s["pos"].long() // PAGE].long(), s["pos"].long() % PAGE
                y[:, h] = s["values"][:, j, h].double()[at] * s["scales"][:, j, h].double()[at][:, None]
        return {"k": k.reshape(rows, -1), "v": v.reshape(rows, -1)}
    x = s["qkv"].double().view(rows, -1, dim)
    turn = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), s["pos"].double()[:, None] * s["freqs"])

    def head(y, w):
        if w is not None:
            y = y / ((y * y).sum(-1, keepdim=True) / dim + EPS).sqrt() * w.double()
        d = s["rotary"]
        first, second = (slice(0, d, 2), slice(1, d, 2)) if s["pairs"] else (slice(0, d // 2), slice(d // 2, d))
        z = torch.complex(y[:, first], y[:, second]) * turn
        y = y.clone()
        y[:, first], y[:, second] = z.real, z.imag
        return y

    q = torch.stack([head(x[:, h], s["q_w"]) for h in range(heads)], 1).reshape(rows, -1)
    values, scales = s["values"].double(), s["scales"].double()
    page, token = s["table"][s["slot"].long(), s["pos"].long() // PAGE].long(), s["pos"].long() % PAGE
    for h in range(kv):
        for j, y in ((0, head(x[:, heads + h], s["k_w"])), (1, x[:, heads + kv + h])):
            scale = (y.abs().max(-1).values / E4M3_MAX).clamp(min=SCALE_MIN)
            values[page, j, h, token], scales[page, j, h, token] = y / scale[:, None], scale
    return {"q": q, "values": values, "scales": scales}

"""Attention over a cache of 8-bit rows: queries with outliers, ragged batches at random, first calls inside a capture and on several threads,
sequences much shorter than max_len, a reported wait."""
import random
import subprocess
import sys

import pytest
import torch

from cache_fp8_tools import Cache, Step
from sapient_b200 import ops
from sapient_b200._lib import SapientCudaError, check, lib

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("rows", [1, 3, 20, 90])
@pytest.mark.parametrize("large", [40.0, 4000.0])
def test_queries_with_outliers(large, rows, ty):
    """One coordinate much larger than the others, against keys that are small there."""
    c = Cache([700], 2, 128, 50)
    s = Step(c, [(0, rows, 700)], 8, ty, 51, size=0.5)
    q = s.q[: s.n].view(s.n, 8, 128)
    q[:, :, 5] = large
    c.values.view(torch.float8_e4m3fn)[:, 0, :, :, 5] = (c.values.view(torch.float8_e4m3fn)[:, 0, :, :, 5].float() / 64).to(torch.float8_e4m3fn)
    s.run()
    s.check(digits=True)


@pytest.mark.parametrize("seed", range(24))
def test_ragged_batches(seed):
    """Sequences of any length beside each other, some without rows or without tokens, in slots in any order, with and without a window."""
    r = random.Random(seed)
    kv, group, dim = r.choice([(1, 1), (2, 4), (3, 2), (1, 7), (8, 4)]) + (r.choice([16, 64, 96, 128]),)
    most = r.choice([2, 6, 40, 150, 400])
    seqs = []
    for slot in r.sample(range(9), r.randint(2, 9)):
        n = r.choice([0, 1, 5, 127, 128, 129, 300, 1111, r.randint(0, 2500)])
        seqs.append((slot, min(r.choice([0, 1, most, r.randint(0, most)]), n), n))
    room = [0] * 9
    for slot, _, n in seqs:
        room[slot] = n
    if not any(x[1] for x in seqs):
        seqs[0] = (seqs[0][0], 1, 0)
    c = Cache(room, kv, dim, seed)
    s = Step(c, seqs, kv * group, r.choice([ops.F32, ops.BF16]), seed + 100)
    for window in (0, r.choice([1, 15, 64, 130, 900])):
        s.out.fill_(7)
        s.run(window=window)
        s.check(window=window)


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("rows", [1, 8, 64])
def test_much_shorter_than_max_len(rows, ty):
    """max_len spreads a sequence over many blocks, most of which find nothing to do."""
    c = Cache([70, 200, 0], 1, 64, 60)
    s = Step(c, [(0, rows, 70), (1, rows, 200), (2, 1, 0)], 4, ty, 61)
    s.run(max_len=200000)
    s.check()


FIRST = """
import sys, threading
sys.path[:0] = {path!r}
import torch
from cache_fp8_tools import Cache, Step
from sapient_b200 import ops
torch.cuda.init()
steps = [Step(Cache([900], 2, dim, i), [(0, rows, 900)], 8, ty, 10 + i) for i, (rows, dim, ty) in enumerate(
    [(1, 128, ops.BF16), (3, 64, ops.BF16), (9, 128, ops.BF16), (80, 128, ops.BF16), (1, 128, ops.F32), (30, 64, ops.F32)])]
torch.cuda.synchronize()
if {captured}:
    for s in steps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            s.run()
        g.replay()
else:
    errors = []
    def work(s, stream):
        try:
            torch.cuda.set_device(0)
            for _ in range(20):
                s.run(stream=stream.cuda_stream)
        except Exception as e:
            errors.append(e)
    threads = [threading.Thread(target=work, args=(s, torch.cuda.Stream())) for s in steps for _ in range(2)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not errors, errors
torch.cuda.synchronize()
for s in steps:
    s.check()
print("all right")
"""


@pytest.mark.parametrize("captured", [True, False])
def test_first_calls(captured):
    """A process whose first calls are captured, and one whose first calls come from several threads at once."""
    path = [p for p in sys.path if p]
    r = subprocess.run([sys.executable, "-c", FIRST.format(path=path, captured=captured)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "all right" in r.stdout, r.stdout + r.stderr


def test_a_wait_that_ran_out():
    check(lib().sp_cuda_report_wait(None, 0, 4))
    torch.cuda.synchronize()
    with pytest.raises(SapientCudaError, match="attention"):
        check(lib().sp_cuda_check_kernels(0))
    check(lib().sp_cuda_check_kernels(0))


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("rows", [1, 5, 140])
@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("scale", [float("inf"), float("nan")])
def test_scales_that_are_no_numbers(scale, which, rows, ty):
    """Rows that see a key or value with such a scale are NaN, whatever the sign of its score; earlier ones are not."""
    c = Cache([300], 2, 64, 70)
    s = Step(c, [(0, rows, 300)], 4, ty, 71)
    for back in (0, min(rows - 1, 3)):  # tokens behind the one
        old = c.scales.clone()
        at = 299 - back
        page = int(c.table[0, at // 16])
        c.values.view(torch.float8_e4m3fn)[page, which, :, at % 16] = 2.0
        c.scales[page, which, :, at % 16] = scale
        for most, empty in ((rows, 0), (32, 70), (4096, 0)):
            for sign in (1, -1):
                q = s.q.clone()
                s.q.copy_(sign * s.q.abs())
                s.run(max_rows=max(most, rows), empty=empty)
                s.q.copy_(q)
                sees = torch.arange(rows, device="cuda") >= rows - 1 - back
                assert s.out[: s.n].isnan().all(-1)[sees].all() and not s.out[: s.n].isnan().any(-1)[~sees].any()
        c.scales.copy_(old)

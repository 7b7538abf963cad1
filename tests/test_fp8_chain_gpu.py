"""Norm, products, SwiGLU and log probabilities one after the other, as a feed-forward block and the head use them: in a stream, in
captured graphs, on several streams at once; rows far apart in memory; a wait that ran out; a device that is not there.

Each step is held against its formula in 64 bits on the inputs that it was given, with the tolerances of its own tests."""
import ctypes as C

import numpy as np
import pytest
import torch

import test_fp8_matmul_gpu as mat
import test_fp8_rows_gpu as rows
import test_logprobs_gpu as lp
from sapient_b200 import ops
from sapient_b200._lib import SP_ERR_CUDA, SP_ERR_OOM, SP_ERR_STATE, SapientCudaError, check, lib

pytestmark = pytest.mark.gpu
TYPES = {ops.F32: torch.float32, ops.BF16: torch.bfloat16}
HIDDEN, FFN, VOCAB, TOP, EPS = 528, 1040, 5003, 5, 1e-5


def weight(n, k, g):
    w = torch.randn(n, k, generator=g, device="cuda") / k**0.5
    s = torch.nn.functional.pad(w.abs(), (0, -k % 128, 0, -n % 128)).view(-(-n // 128), 128, -(-k // 128), 128).amax((1, 3)) / 448
    q = (w / s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)[:, :k]).clamp(-448, 448).to(torch.float8_e4m3fn)
    return q, s.contiguous()


class Block:
    """x, residual -> norm -> gate | up -> SwiGLU -> down -> norm with the sum -> head -> distribution."""

    def __init__(self, m, ty, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.m, self.ty = m, ty
        new = lambda n, t=None: torch.zeros(m, n, device="cuda", dtype=t or TYPES[ty])  # noqa: E731
        self.x = torch.randn(m, HIDDEN, generator=g, device="cuda").to(TYPES[ty])
        self.norms = [0.5 + torch.rand(HIDDEN, generator=g, device="cuda") for _ in range(2)]
        self.w = [weight(2 * FFN, HIDDEN, g), weight(HIDDEN, FFN, g), weight(VOCAB, HIDDEN, g)]
        self.ids = torch.randint(0, VOCAB, (m,), generator=g, device="cuda", dtype=torch.int32)
        self.q = [new(n, torch.uint8) for n in (HIDDEN, FFN, HIDDEN)]
        self.s = [new(-(-n // 128), torch.float32) for n in (HIDDEN, FFN, HIDDEN)]
        self.gu, self.down, self.total, self.z = new(2 * FFN), new(HIDDEN), new(HIDDEN), new(VOCAB)
        self.out = [torch.zeros(m, device="cuda") for _ in range(2)] + [torch.zeros(m, TOP, device="cuda", dtype=torch.int32), torch.zeros(m, TOP, device="cuda")]

    def product(self, i, y, st):
        q, s = self.w[i]
        ops.matmul_fp8_dev(self.q[i].data_ptr(), self.s[i].data_ptr(), self.m, q.data_ptr(), s.data_ptr(), *q.shape, y.data_ptr(), self.ty, stream=st)

    def run(self):
        st = torch.cuda.current_stream().cuda_stream
        p = lambda t: t.data_ptr()  # noqa: E731
        ops.rms_norm_fp8_dev(p(self.x), self.m, HIDDEN, p(self.norms[0]), EPS, p(self.q[0]), p(self.s[0]), self.ty, stream=st)
        self.product(0, self.gu, st)
        ops.swiglu_fp8_dev(p(self.gu), self.m, FFN, p(self.q[1]), p(self.s[1]), self.ty, stream=st)
        self.product(1, self.down, st)
        ops.rms_norm_fp8_dev(p(self.down), self.m, HIDDEN, p(self.norms[1]), EPS, p(self.q[2]), p(self.s[2]), self.ty, residual=p(self.x), sum_out=p(self.total), stream=st)
        self.product(2, self.z, st)
        o = self.out
        ops.logprobs_dev(p(self.z), self.m, VOCAB, p(self.ids), p(o[0]), p(o[1]), TOP, p(o[2]), p(o[3]), self.ty, stream=st)

    def results(self):
        return [*self.q, *self.s, self.gu, self.down, self.total, self.z, *self.out]

    def check(self):
        rows.check(self.q[0], self.s[0], rows.norm64(self.x, None, self.norms[0], EPS)[1])
        e4m3 = [q.view(torch.float8_e4m3fn) for q in self.q]
        for i, y in enumerate((self.gu, self.down, self.z)):
            mat.check(y, e4m3[i], self.s[i], *self.w[i])
        gu = self.gu.double()
        rows.check(self.q[1], self.s[1], gu[:, :FFN] / (1 + torch.exp(-gu[:, :FFN])) * gu[:, FFN:])
        assert torch.equal(self.total, (self.x.float() + self.down.float()).to(TYPES[self.ty]))
        rows.check(self.q[2], self.s[2], rows.norm64(self.down, self.x, self.norms[1], EPS)[1])
        e = lp.want(self.z, self.ids, TOP)
        assert torch.equal(self.out[2], e[2])
        for a, b in ((self.out[0], e[0]), (self.out[1], e[1]), (self.out[3], e[3])):
            lp.near(a, b)


@pytest.mark.parametrize("ty", [ops.F32, ops.BF16])
@pytest.mark.parametrize("m", [1, 5, 24, 160, 700])
def test_one_after_the_other(m, ty):
    """Ten times without a pause, over new inputs: a call that started before the one ahead of it was done would show."""
    b = Block(m, ty, m)
    for i in range(10):
        b.x.copy_(torch.randn(m, HIDDEN, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)))
        b.run()
    b.check()


@pytest.mark.parametrize("m", [1, 24, 700])
def test_captured_replayed_and_side_by_side(m):
    a, b = Block(m, ops.BF16, 1), Block(m, ops.BF16, 2)
    graphs, want = [], []
    for c in (a, b):
        c.run()
        want.append([t.clone() for t in c.results()])
    torch.cuda.synchronize()
    for c in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            c.run()
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for c in (a, b):
        for t in c.results():
            t.zero_()
    torch.cuda.synchronize()
    for _ in range(5):  # two graphs at once, and the same calls outside of graphs between
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
        with torch.cuda.stream(streams[0]):
            a.run()
    torch.cuda.synchronize()
    for c, w in zip((a, b), want):
        assert all(torch.equal(t, u) for t, u in zip(c.results(), w))


@pytest.mark.parametrize("m,n,k", [(3, 9000, 4096), (64, 4000, 8192), (128, 4096, 8208), (384, 500, 12304), (200, 2000, 2064), (900, 16400, 1168), (2048, 8192, 2064)])
def test_products_on_two_streams_at_once(m, n, k):
    a = [mat.inputs(m, n, k, s) for s in (1, 2)]
    want = [mat.product(*x, ops.BF16) for x in a]
    ys = [torch.empty_like(w) for w in want]
    streams = [torch.cuda.Stream() for _ in a]
    torch.cuda.synchronize()
    for _ in range(20):
        for (xq, xs, wq, ws), y, st in zip(a, ys, streams):
            ops.matmul_fp8_dev(xq.data_ptr(), xs.data_ptr(), m, wq.data_ptr(), ws.data_ptr(), n, k, y.data_ptr(), ops.BF16, stream=st.cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for y, w in zip(ys, want)) and lib().sp_cuda_check_kernels(0) == 0


def test_a_weight_in_captured_graphs():
    """The first call with more rows than before allocates and is not captured; what was captured before keeps its workspace."""
    g = torch.Generator(device="cuda").manual_seed(3)
    q, s = weight(300, HIDDEN, g)
    w = ops.Weight.from_fp8(q.view(torch.uint8).cpu().numpy(), s.cpu().numpy())
    xs = [torch.randn(m, HIDDEN, generator=g, device="cuda") for m in (3, 500)]
    ys = [torch.zeros(x.shape[0], 300, device="cuda") for x in xs]
    call = lambda i: check(lib().sp_cuda_matmul_nt_dev(w.h, xs[i].data_ptr(), xs[i].shape[0], ys[i].data_ptr(), torch.cuda.current_stream().cuda_stream))  # noqa: E731
    graphs = [torch.cuda.CUDAGraph() for _ in xs]
    for i in range(2):
        torch.cuda.synchronize()
        with torch.cuda.graph(graphs[i]):
            with pytest.raises(SapientCudaError) as e:
                call(i)
        assert e.value.status == SP_ERR_STATE
        call(i)
        torch.cuda.synchronize()
        graphs[i] = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graphs[i]):
            call(i)
    want = [y.clone() for y in ys]
    for _ in range(2):
        for i in (0, 1):
            ys[i].zero_()
            graphs[i].replay()
    torch.cuda.synchronize()
    assert torch.equal(ys[0], want[0]) and torch.equal(ys[1], want[1])
    for x, y in zip(xs, ys):
        xq, sx = (torch.from_numpy(t).cuda() for t in ops.quant_fp8(x.cpu().numpy()))
        mat.check(y, xq.view(torch.float8_e4m3fn), sx, q, s)
    del graphs
    w.free()


def test_rows_more_than_two_to_the_31_values_apart():
    """Offsets that pass 32 bits: outputs of the products of every height, inputs of the other calls."""
    big = torch.zeros(10 << 30, device="cuda", dtype=torch.uint8)
    half, full = big.view(torch.bfloat16), big.view(torch.float32)
    for m, n, k in [(3, 500, 144), (40, 500, 1040), (130, 300, 272), (300, 40000, 144), (700, 40000, 144)]:
        a, ld = mat.inputs(m, n, k, m), (half.numel() // m) // 8 * 8
        y = half[: m * ld].view(m, ld)[:, :n]
        xq, xs, wq, ws = a
        ops.matmul_fp8_dev(xq.data_ptr(), xs.data_ptr(), m, wq.data_ptr(), ws.data_ptr(), n, k, y.data_ptr(), ops.BF16, ld, stream=torch.cuda.current_stream().cuda_stream)
        mat.check(y, *a)
    g = torch.Generator(device="cuda").manual_seed(7)
    ld = half.numel() // 3 // 8 * 8
    x = half[: 3 * ld].view(3, ld)
    x[:, :5000] = torch.randn(3, 5000, generator=g, device="cuda")
    lp.check(x[:, :5000], torch.tensor([0, 4999, 17], device="cuda", dtype=torch.int32), 5)
    q, s = rows.norm(x[:, :528], x[:, 1000:1528], None, total=x[:, 2000:2528])
    rows.check(q, s, rows.norm64(x[:, :528], x[:, 1000:1528], None)[1])
    assert torch.equal(x[:, 2000:2528], (x[:, :528].float() + x[:, 1000:1528].float()).bfloat16())
    q, s = torch.empty(3, 512, device="cuda", dtype=torch.uint8), torch.empty(3, 4, device="cuda")
    ops.quant_fp8_dev(x.data_ptr(), 3, 512, q.data_ptr(), s.data_ptr(), ops.BF16, ld, stream=torch.cuda.current_stream().cuda_stream)
    rows.check(q, s, x[:, :512].double())
    z = full[: 12 * (full.numel() // 12)].view(12, -1)
    z[:, :700] = torch.randn(12, 700, generator=g, device="cuda")
    lp.check(z[:, :700], torch.arange(12, device="cuda", dtype=torch.int32), 3)


def test_more_than_two_to_the_31_values():
    n, dim = 140000, 16384
    x = torch.zeros(n, dim, device="cuda", dtype=torch.bfloat16)
    x[-3:] = torch.randn(3, dim, generator=torch.Generator(device="cuda").manual_seed(7), device="cuda")
    q, s = torch.zeros(n, dim, device="cuda", dtype=torch.uint8), torch.zeros(n, 128, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    ops.quant_fp8_dev(x.data_ptr(), n, dim, q.data_ptr(), s.data_ptr(), ops.BF16, stream=st)
    rows.check(q[-4:], s[-4:], x[-4:].double())
    ops.rms_norm_fp8_dev(x.data_ptr(), n, dim, 0, 1e-5, q.data_ptr(), s.data_ptr(), ops.BF16, stream=st)
    rows.check(q[-4:], s[-4:], rows.norm64(x[-4:], None, None)[1])
    ops.swiglu_fp8_dev(x.data_ptr(), n, dim // 2, q.data_ptr(), s.data_ptr(), ops.BF16, stream=st)
    y = x[-4:].double()
    y = y[:, : dim // 2] / (1 + torch.exp(-y[:, : dim // 2])) * y[:, dim // 2 :]
    rows.check(q.view(-1)[: n * dim // 2].view(n, -1)[-4:], s.view(-1)[: n * 64].view(n, -1)[-4:], y)


def test_a_wait_that_ran_out_is_reported_once():
    rng = np.random.default_rng(0)
    xq, xs = ops.quant_fp8(rng.standard_normal((20, 256)).astype(np.float32))
    wq, ws = xq.copy(), np.ones((1, 2), np.float32)
    want = ops.matmul_fp8(xq, xs, wq, ws)
    check(lib().sp_cuda_report_wait(None, 0, 3))
    with pytest.raises(SapientCudaError, match="wait expired"):
        ops.matmul_fp8(xq, xs, wq, ws)
    assert np.array_equal(ops.matmul_fp8(xq, xs, wq, ws), want)


def test_a_device_that_is_not_there():
    x = torch.ones(2, 256, device="cuda")
    q, s = torch.empty(2, 256, device="cuda", dtype=torch.uint8), torch.empty(2, 2, device="cuda")
    for device in (-1, 63):
        with pytest.raises(SapientCudaError) as e:
            ops.quant_fp8_dev(x.data_ptr(), 2, 256, q.data_ptr(), s.data_ptr(), device=device)
        assert e.value.status == SP_ERR_CUDA
    ops.quant_fp8_dev(x.data_ptr(), 2, 256, q.data_ptr(), s.data_ptr())
    torch.cuda.synchronize()
    rows.check(q, s, x.double())


def test_a_refused_call_leaves_no_error_for_the_next_one():
    """Each call that fails says so itself; the launch that follows it on the same thread is not the one to answer for it."""
    x = torch.ones(2, 256, device="cuda")
    q, s = torch.empty(2, 256, device="cuda", dtype=torch.uint8), torch.empty(2, 2, device="cuda")
    host, bytes_, ones = np.ones((2, 256), np.float32), np.ones((2, 256), np.uint8), np.ones((1, 2), np.float32)
    h, some = C.c_void_p(), host.ctypes.data_as(C.c_void_p)

    def more_than_there_is():  # (2^56 bytes: refused before anything is read)
        check(lib().sp_cuda_upload_weight_fp8(0, 1 << 28, 1 << 28, some, some, C.byref(h)))

    fails = [(SP_ERR_CUDA, lambda: ops.quant_fp8(host, device=63)), (SP_ERR_CUDA, lambda: ops.swiglu_fp8(host, device=63)),
             (SP_ERR_CUDA, lambda: ops.rms_norm_fp8(host, None, EPS, device=63)), (SP_ERR_CUDA, lambda: ops.logprobs(host, [0, 1], device=63)),
             (SP_ERR_CUDA, lambda: ops.matmul_fp8(bytes_, np.ones((2, 2)), bytes_, ones, device=63)), (SP_ERR_CUDA, lambda: ops.Weight.from_fp8(bytes_, ones, device=63)),
             (SP_ERR_CUDA, lambda: ops.silu(host, device=63)), (SP_ERR_CUDA, lambda: ops.Weight(ops.F32, 2, 256, host.view(np.uint8), device=63)),
             (SP_ERR_OOM, more_than_there_is)]
    wrong = []
    for i, (status, call) in enumerate(fails):
        with pytest.raises(SapientCudaError) as e:
            call()
        assert e.value.status == status
        q.zero_()
        try:
            ops.quant_fp8_dev(x.data_ptr(), 2, 256, q.data_ptr(), s.data_ptr(), stream=torch.cuda.current_stream().cuda_stream)
            rows.check(q, s, x.double())
        except SapientCudaError:
            wrong.append(i)
    assert not wrong


def test_a_weight_is_there_when_its_upload_returns():
    """The first product may be on any stream, one that does not wait for the default stream among them."""
    g = torch.Generator(device="cuda").manual_seed(4)
    st = torch.cuda.Stream()
    for n, k in [(16, 64), (130, 272), (1000, 1040), (4096, 4096)]:
        q, s = weight(n, k, g)
        values, scales = q.view(torch.uint8).cpu().numpy(), s.cpu().numpy()
        x = torch.randn(3, k, generator=g, device="cuda")
        y = torch.zeros(20, 3, n, device="cuda")
        torch.cuda.synchronize()
        for i in range(20):
            w = ops.Weight.from_fp8(values, scales)
            w.matmul_nt_dev(x.data_ptr(), 3, y[i].data_ptr(), st.cuda_stream)
            st.synchronize()
            w.free()
        xq, sx = (torch.from_numpy(t).cuda() for t in ops.quant_fp8(x.cpu().numpy()))
        mat.check(y[0], xq.view(torch.float8_e4m3fn), sx, q, s)
        assert (y == y[0]).all()


def test_a_weight_grows_beside_a_capture_of_another_thread():
    """The workspace's allocation is none of a capture that goes on elsewhere, and does not end it."""
    import threading

    g = torch.Generator(device="cuda").manual_seed(5)
    q, s = weight(300, HIDDEN, g)
    w = ops.Weight.from_fp8(q.view(torch.uint8).cpu().numpy(), s.cpu().numpy())
    x, y = torch.randn(40, HIDDEN, generator=g, device="cuda"), torch.zeros(40, 300, device="cuda")
    a, b = torch.ones(1000, device="cuda"), torch.zeros(1000, device="cuda")
    ops.quant_fp8(np.ones((1, 16), np.float32))  # (the library is there)
    st, graph, said = torch.cuda.Stream(), torch.cuda.CUDAGraph(), []

    def grow():
        try:
            w.matmul_nt_dev(x.data_ptr(), 40, y.data_ptr(), st.cuda_stream)
        except SapientCudaError as e:
            said.append(e)

    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        b.copy_(a)
        t = threading.Thread(target=grow)
        t.start()
        t.join()
        b.mul_(2)
    assert not said
    graph.replay()
    torch.cuda.synchronize()
    assert (b == 2).all()
    xq, sx = (torch.from_numpy(t).cuda() for t in ops.quant_fp8(x.cpu().numpy()))
    mat.check(y, xq.view(torch.float8_e4m3fn), sx, q, s)


@pytest.mark.parametrize("m", [3, 160, 700])
def test_the_first_calls_of_a_process_may_be_captured(m):
    """What a first call sets up (attributes, flags, addresses of the driver) needs no call before."""
    import os
    import subprocess
    import sys

    here = os.path.dirname(os.path.abspath(__file__))
    code = f"""import torch
import test_fp8_chain_gpu as c
b = c.Block({m}, c.ops.BF16, 1)
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.cuda.graph(g):
    b.run()
for t in b.results():
    t.zero_()
g.replay()
torch.cuda.synchronize()
b.check()
print("held")
"""
    r = subprocess.run([sys.executable, "-c", code], cwd=here, env=os.environ | {"PYTHONPATH": os.pathsep.join([os.path.dirname(here), here])}, capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and "held" in r.stdout, r.stderr[-2000:]


class Hopping(Block):
    """The steps by turns on two streams, each after the one before by an event; what `run` asks for is the stream of a step."""

    def __init__(self, *a):
        super().__init__(*a)
        self.streams, self.steps = [torch.cuda.Stream(), torch.cuda.Stream()], 0

    def hop(self):
        last, new = self.streams[self.steps % 2], self.streams[(self.steps + 1) % 2]
        new.wait_stream(last)
        self.steps += 1
        return new

    def run(self):
        p = lambda t: t.data_ptr()  # noqa: E731
        at = lambda: self.hop().cuda_stream  # noqa: E731
        ops.rms_norm_fp8_dev(p(self.x), self.m, HIDDEN, p(self.norms[0]), EPS, p(self.q[0]), p(self.s[0]), self.ty, stream=at())
        self.product(0, self.gu, at())
        ops.swiglu_fp8_dev(p(self.gu), self.m, FFN, p(self.q[1]), p(self.s[1]), self.ty, stream=at())
        self.product(1, self.down, at())
        ops.rms_norm_fp8_dev(p(self.down), self.m, HIDDEN, p(self.norms[1]), EPS, p(self.q[2]), p(self.s[2]), self.ty, residual=p(self.x), sum_out=p(self.total), stream=at())
        self.product(2, self.z, at())
        o = self.out
        ops.logprobs_dev(p(self.z), self.m, VOCAB, p(self.ids), p(o[0]), p(o[1]), TOP, p(o[2]), p(o[3]), self.ty, stream=at())


@pytest.mark.parametrize("m", [1, 24, 160, 700])
def test_steps_on_two_streams_by_turns(m):
    """In streams, then in one graph with a second chain beside it: an event keeps a step back as the stream itself does."""
    a, b = Hopping(m, ops.BF16, 1), Hopping(m, ops.BF16, 2)
    here = torch.cuda.current_stream()
    xs = [torch.randn(m, HIDDEN, device="cuda", generator=torch.Generator(device="cuda").manual_seed(i)).to(TYPES[a.ty]) for i in range(10)]
    for x in xs:
        a.x.copy_(x)
        for st in a.streams:
            st.wait_stream(here)
        a.run()
        for st in a.streams:
            here.wait_stream(st)
    a.check()
    b.streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        inside = torch.cuda.current_stream()
        for c in (a, b):
            for st in c.streams:
                st.wait_stream(inside)
        for c in (a, b):
            c.run()
        for c in (a, b):
            for st in c.streams:
                inside.wait_stream(st)
    for t in a.results() + b.results():
        t.zero_()
    for _ in range(5):
        graph.replay()
    torch.cuda.synchronize()
    a.check()
    b.check()

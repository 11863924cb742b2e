"""Products that pass sums of ranges of K, or copies of unaligned rows, through the stream's
workspace: captured, in two graphs of one stream, from several threads, and one token of them
alone. Every case asserts that its product uses the workspace."""
from __future__ import annotations

import threading

import pytest
import torch

from tests import _w8a8 as P
from tests import _w8a8_forms as F

pytestmark = pytest.mark.gpu

# tokens, channels, columns, projections; K cut, rows copied
CASES = [(2304, 256, 11008, 1, True, False), (2360, 416, 555, 1, False, True), (829, 2444, 16565, 1, True, True),
         (2226, 107, 2768, 2, True, False), (700, 1999, 1001, 2, False, True), (907, 2367, 13209, 2, True, True)]


class Product:
    """One product with its weights; x's codes and scales are given."""

    def __init__(self, m, n, k, projections, cut, copied, seed=0):
        f = F.form(m, n, k, projections)
        assert F.workspace(m, n, k, projections) > 0
        assert (f.ranges > 1, f.copies == 1) == (cut, copied)
        self.m, self.k, self.projections = m, k, projections
        self.w = [P.qt(*P.codes(n, k, seed + 10 + p)) for p in range(projections)]
        self.bias = torch.randn(n, generator=torch.Generator().manual_seed(seed)).half().cuda()

    def inputs(self, seed):
        x, s = P.codes(self.m, self.k, seed)
        return x, s * (20 / self.k ** 0.5)

    def __call__(self, x, s):
        from cublade_amd.quantization import gated_w8a8, linear_w8a8
        if self.projections == 1:
            return linear_w8a8(P.qt(x, s), self.w[0], self.bias, out_dtype=torch.float32)
        return gated_w8a8(P.qt(x, s), *self.w, gate_bias=self.bias, out_dtype=torch.float32)


def _warm(stream, *calls):
    with torch.cuda.stream(stream):
        for f in calls:
            f()
    torch.cuda.synchronize()


@pytest.mark.parametrize("case", CASES)
def test_graph(case):
    """Replays with new inputs, eager calls and other work on the stream between them."""
    p = Product(*case)
    x, s = p.inputs(0)
    stream, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    _warm(stream, lambda: p(x, s))
    with torch.cuda.graph(g, stream=stream):
        y = p(x, s)
    other = Product(*CASES[0], seed=3)
    ox = other.inputs(4)
    ow = other(*ox)
    for seed in range(1, 5):
        nx, ns = p.inputs(seed)
        x.copy_(nx)
        s.copy_(ns)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            g.replay()
            o = other(*ox)
            want = p(nx, ns)
        torch.cuda.synchronize()
        assert torch.equal(y, want) and torch.equal(o, ow)
        if case[3] == 1:
            rows = slice(0, 40)
            assert torch.equal(y[rows].cpu(), P.linear(nx[rows], ns[rows], p.w[0].data, p.w[0].scale, p.bias,
                                                       torch.float32))


def test_two_graphs_of_one_stream():
    ps = [Product(*CASES[0], seed=1), Product(*CASES[1], seed=2), Product(*CASES[5], seed=3)]
    ins = [p.inputs(5) for p in ps]
    stream = torch.cuda.Stream()
    _warm(stream, *[lambda p=p, i=i: p(*i) for p, i in zip(ps, ins)])
    graphs, outs = [], []
    for p, i in zip(ps, ins):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(p(*i))
        graphs.append(g)
    for seed in range(6, 9):
        for p, i in zip(ps, ins):
            for old, new in zip(i, p.inputs(seed)):
                old.copy_(new)
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            for k in (0, 1, 2, 0, 2, 1):
                graphs[k].replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(stream):
            want = [p(*i) for p, i in zip(ps, ins)]
        torch.cuda.synchronize()
        assert all(torch.equal(o, w) for o, w in zip(outs, want))


@pytest.mark.parametrize("own_streams", [False, True])
def test_threads(own_streams):
    """Four threads, each with another product or input, on one stream and on their own."""
    ps = [Product(*c, seed=i) for i, c in enumerate((CASES[0], CASES[1], CASES[3], CASES[0]))]
    ins = [p.inputs(20 + i) for i, p in enumerate(ps)]
    want = [p(*i) for p, i in zip(ps, ins)]
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()
    streams = [torch.cuda.Stream() for _ in ps] if own_streams else [shared] * 4
    bad = []

    def work(i):
        with torch.cuda.stream(streams[i]):
            for _ in range(25):
                y = ps[i](*ins[i])
                streams[i].synchronize()
                if not torch.equal(y, want[i]):
                    bad.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


@pytest.mark.parametrize("case", CASES)
def test_a_token_alone(case):
    """A token of a product whose K is cut or whose rows are copied: the bits of a call on it
    alone, or on a few."""
    p = Product(*case)
    x, s = p.inputs(9)
    y = p(x, s)
    for r in (slice(0, 1), slice(100, 117), slice(p.m - 60, p.m)):
        assert F.workspace(r.stop - r.start, y.shape[1], p.k, p.projections) == 0
        assert torch.equal(p(x[r], s[r]), y[r])


def test_layers_with_columns_of_any_number():
    """The layers on such products (their weights are copied in the call)."""
    from cublade_amd.quantization import cuBladeW8A8LinearLayer, linear_w8a8, quantize_tensor
    torch.manual_seed(0)
    lin = torch.nn.Linear(555, 416).half().cuda()
    layer = cuBladeW8A8LinearLayer.from_linear(lin)
    x = torch.randn(2360, 555, device="cuda").half()
    assert F.form(2360, 416, 555, 1).copies
    q, w = quantize_tensor(x, mode="channel"), quantize_tensor(lin.weight.detach(), mode="channel")
    y = layer(x)
    assert torch.equal(y, linear_w8a8(q, w, lin.bias))
    assert torch.equal(y.cpu(), P.linear(q.data, q.scale, w.data, w.scale, lin.bias.detach(), torch.float16))

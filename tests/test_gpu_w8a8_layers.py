"""The W8A8 layers and the block that they, the norms and the cache's neighbours make:
against fp32 without quantisation, against the operators one by one, captured, on other
streams, from several threads, through quantize_model and state dicts.

Bound of a layer's relative error (root mean square over outputs) against fp32: both
operands err by a uniform rounding of half a step of amax / 127. A Gaussian row of n
values has amax of at most c = sqrt(2 ln(2 n)) + 1 standard deviations (6.1 for n = 11008
with a probability beyond 1 - 1e-6), so a value's error is at most c / 127 / sqrt(12) =
1.4% of the standard deviation, root mean square. Two independent operands: sqrt(2) 1.4%
= 2%; an output's rounding to 16 bits adds 0.2% at most: 2.2%.
A gated block: gate and up err by 2.2% each. silu(g) u: |silu'| <= 1.1, so h errs by at
most 2.2% (1.1 rms(g) rms(u) + rms(silu g) rms(u)) against rms(h) = rms(silu g) rms(u);
with g of standard deviation 1, rms(silu g) = 0.56 (E silu^2 = 0.36 by the integral's
numerical value, rounded down): 2.2% (1.1 / 0.56 + 1) = 6.6%. Then h is quantized: its
rows are products of two Gaussians, whose largest of n values lies within ln(n) + 6 = 15.3
of rms(h)'s unit 0.56: 15.3 / 0.56 / 127 / sqrt(12) = 6.2% at most; the down projection's
weights 1.4%. In all sqrt(6.6^2 + 6.2^2 + 1.4^2) = 9.2%."""
from __future__ import annotations

import copy
import threading

import pytest
import torch
import torch.nn as nn

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _linear(n_in, n_out, seed, dtype, bias=True):
    torch.manual_seed(seed)
    m = nn.Linear(n_in, n_out, bias=bias)
    with torch.no_grad():
        m.weight.normal_(0, n_in ** -0.5)
    return m.to(dtype).to(DEV)


def _rel(y, want):
    return float((y.double() - want.double()).norm() / want.double().norm())


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("n_in,n_out", [(1024, 1536), (1000, 333)])
def test_layer_follows_fp32(dtype, n_in, n_out):
    from cublade_amd.quantization import cuBladeW8A8LinearLayer, norm_tensor
    lin = _linear(n_in, n_out, 0, dtype)
    layer = cuBladeW8A8LinearLayer.from_linear(lin)
    for shape in ((n_in,), (1, n_in), (3, 50, n_in), (700, n_in)):
        x = torch.randn(*shape, device=DEV).to(dtype)
        y = layer(x)
        want = x.float() @ lin.weight.float().t() + lin.bias.float()
        assert y.shape == want.shape and y.dtype == dtype
        assert _rel(y, want) <= 0.022
    # a QuantizedTensor is taken as it is
    q = norm_tensor(x)
    assert torch.equal(layer(q), layer(q)) and layer(q).dtype == dtype


def test_layer_is_its_operators():
    from cublade_amd.quantization import cuBladeW8A8LinearLayer, linear_w8a8, quantize_tensor
    lin = _linear(512, 256, 1, torch.bfloat16)
    layer = cuBladeW8A8LinearLayer.from_linear(lin)
    x = torch.randn(40, 512, device=DEV).bfloat16()
    qx, qw = quantize_tensor(x, mode="channel"), quantize_tensor(lin.weight.detach(), mode="channel")
    assert torch.equal(layer.int8_weights, qw.data) and torch.equal(layer.scales, qw.scale)
    assert torch.equal(layer(x), linear_w8a8(qx, qw, lin.bias))
    # a tensor-wide scale
    qs = quantize_tensor(x, mode="tensor")
    assert _rel(linear_w8a8(qs, qw, lin.bias), layer(x)) <= 0.05
    assert not layer(x).requires_grad


class MLP(nn.Module):
    def __init__(self, hidden, inter, dtype, seed=2):
        super().__init__()
        self.gate = _linear(hidden, inter, seed, dtype, bias=False)
        self.up = _linear(hidden, inter, seed + 1, dtype, bias=False)
        self.down = _linear(inter, hidden, seed + 2, dtype, bias=False)

    def forward(self, x):
        return self.down(nn.functional.silu(self.gate(x)) * self.up(x))


def test_quantize_model_and_state_dict():
    from cublade_amd.quantization import cuBladeW8A8LinearLayer, quantize_model
    mlp = MLP(512, 1024, torch.float16)
    x = torch.randn(2, 30, 512, device=DEV).half()
    want = copy.deepcopy(mlp).float()(x.float())
    q = quantize_model(mlp, "w8a8", exclude_modules=["down"], inplace=False)
    assert isinstance(q.gate, cuBladeW8A8LinearLayer) and isinstance(q.down, nn.Linear)
    q = quantize_model(mlp, "w8a8")
    assert all(isinstance(m, cuBladeW8A8LinearLayer) for m in (q.gate, q.up, q.down))
    y = q(x)
    assert _rel(y, want) <= 0.092
    fresh = quantize_model(MLP(512, 1024, torch.float16, seed=9), "w8a8")
    fresh.load_state_dict(q.state_dict())
    assert torch.equal(fresh(x), y)
    half = copy.deepcopy(q).bfloat16()      # the scales stay fp32
    assert half.gate.scales.dtype == torch.float32 and half(x.bfloat16()).dtype == torch.bfloat16
    back = copy.deepcopy(q).cpu().to(DEV)
    assert torch.equal(back(x), y)


@pytest.mark.parametrize("act,fn", [("silu", nn.functional.silu), ("gelu", nn.functional.gelu)])
def test_gated_mlp(act, fn):
    from cublade_amd.quantization import cuBladeW8A8GatedMLP, quantize_tensor
    m = MLP(512, 1376, torch.bfloat16)
    q = cuBladeW8A8GatedMLP(m.gate, m.up, m.down, activation=act)
    for tokens in (1, 40, 300):
        x = torch.randn(tokens, 512, device=DEV).bfloat16()
        xf = x.float()
        h = fn(xf @ m.gate.weight.float().t()) * (xf @ m.up.weight.float().t())
        y = q(x)
        assert y.shape == x.shape and _rel(y, h @ m.down.weight.float().t()) <= 0.092
        assert torch.equal(q(quantize_tensor(x, mode="channel")), y)
    assert set(q.state_dict()) == {f"{n}.{p}" for n in ("gate", "up", "down") for p in ("int8_weights", "scales")}


class Block(nn.Module):
    """norm -> W8A8 gated MLP -> norm after the block, gate, residual -> the next norm."""

    def __init__(self, hidden, inter, dtype):
        from cublade_amd.quantization import cuBladeW8A8GatedMLP
        super().__init__()
        m = MLP(hidden, inter, dtype)
        self.mlp = cuBladeW8A8GatedMLP(m.gate, m.up, m.down)
        g = torch.Generator().manual_seed(5)
        self.w = [(1 + 0.2 * torch.randn(hidden, generator=g)).to(dtype).to(DEV) for _ in range(4)]

    def forward(self, x):
        from cublade_amd.quantization import norm_tensor, residual_norm
        q = norm_tensor(x, self.w[0])
        return residual_norm(self.mlp(q), x, self.w[1], post_norm=True, post_weight=self.w[2],
                             gate=self.w[3], scale=0.5)


def _norm(x, w):
    return x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()


@pytest.mark.parametrize("tokens", [1, 70, 520])
def test_block(tokens):
    from cublade_amd.quantization import dequantize_tensor
    b = Block(512, 1376, torch.bfloat16)
    x = torch.randn(tokens, 512, device=DEV).bfloat16()
    h, q = b(x)
    m = MLP(512, 1376, torch.bfloat16).float()
    want = x.float() + 0.5 * b.w[3].float() * _norm(m(_norm(x.float(), b.w[0])), b.w[2])
    # the MLP's 9.2% (and its norm's, of as much: the mean square errs by no more) of the
    # half that it adds: |w3 norm(.)| / 2 against |x + ...|, both terms of order 1
    assert _rel(h, want) <= 0.092 * 2
    # the last norm is that of h: codes' rounding, 1.4%, and bf16's, 0.4%
    assert _rel(dequantize_tensor(q), _norm(h.float(), b.w[1])) <= 0.02


def _replays(fn, x, inputs, stream):
    with torch.cuda.stream(stream):
        for _ in range(2):
            fn()
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=stream):
        out = fn()
    for new in inputs:
        x.copy_(new)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = fn()
        torch.cuda.synchronize()
        for a, b in zip(out, want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("tokens,hidden,inter", [(1, 512, 1376), (200, 1024, 4096), (700, 1000, 1001), (64, 512, 2064)])
def test_graph(tokens, hidden, inter):
    """Captured with ranges of K (tokens = 200), with copies of unaligned rows (inter =
    1001), and without either; each replay equals the eager call."""
    b = Block(hidden, inter, torch.float16)
    x = torch.randn(tokens, hidden, device=DEV).half()

    def fn():
        h, q = b(x)
        return h, q.data, q.scale

    _replays(fn, x, [torch.randn(tokens, hidden, device=DEV).half() for _ in range(4)], torch.cuda.Stream())


def test_two_captured_graphs_with_eager_work_between():
    """Two graphs of one stream share its workspace: replayed in turn, with eager calls
    of both between them."""
    a, b = Block(1024, 4096, torch.bfloat16), Block(512, 11008, torch.bfloat16)
    xa, xb = (torch.randn(200, n, device=DEV).bfloat16() for n in (1024, 512))
    s = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(s):
        for _ in range(2):
            a(xa), b(xb)
    torch.cuda.synchronize()
    for m, x in ((a, xa), (b, xb)):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            outs.append(m(x)[0])
        graphs.append(g)
    for i in range(3):
        xa.normal_()
        xb.normal_()
        with torch.cuda.stream(s):
            s.wait_stream(torch.cuda.default_stream())
            graphs[0].replay()
            graphs[1].replay()
            graphs[0].replay()
            want = a(xa)[0], b(xb)[0]
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1])


def test_streams_and_threads():
    """Calls of several threads on one stream and on their own, all with workspaces."""
    b = Block(1024, 4096, torch.bfloat16)
    xs = [torch.randn(200, 1024, device=DEV).bfloat16() for _ in range(4)]
    want = [b(x) for x in xs]
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()
    bad = []

    def work(i, stream):
        with torch.cuda.stream(stream):
            for _ in range(25):
                h, q = b(xs[i])
                stream.synchronize()
                if not (torch.equal(h, want[i][0]) and torch.equal(q.data, want[i][1].data)):
                    bad.append(i)

    for streams in ([shared] * 4, [torch.cuda.Stream() for _ in xs]):
        threads = [threading.Thread(target=work, args=(i, s)) for i, s in enumerate(streams)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert not bad


def test_refusals_with_gpu_tensors():
    from cublade_amd.quantization import (QuantizedTensor, cuBladeW8A8LinearLayer, gated_w8a8, linear_w8a8,
                                          quantize_tensor)
    x, w = (quantize_tensor(torch.randn(n, 64, device=DEV).half(), mode="channel") for n in (5, 8))
    other = quantize_tensor(torch.randn(8, 48, device=DEV).half(), mode="channel")
    zero = torch.zeros((), device=DEV)

    def q(**kw):
        f = dict(data=w.data, scale=w.scale, zero_point=zero, mode="channel", axis=0, group_size=32,
                 dtype=torch.int8, original_dtype=torch.float16)
        return QuantizedTensor(**{**f, **kw})

    b = torch.zeros(8, device=DEV)
    for args, kw, needle in (
            ((x, other), {}, r"\[rows, 64\]"), ((x, w, b[:7]), {}, "bias"), ((x, w, b.double()), {}, "bias"),
            ((x, w, b.cpu()), {}, "bias"), ((x, w), dict(out_dtype=torch.float64), "out_dtype"),
            ((x, q(scale=w.scale[:7])), {}, "one scale for each"), ((x, q(scale=w.scale.half())), {}, "float32"),
            ((x, q(data=w.data.cpu())), {}, "must be on"), ((x, q(scale=w.scale.cpu())), {}, "must be on")):
        with pytest.raises(RuntimeError, match=needle):
            linear_w8a8(*args, **kw)
    for kw, needle in ((dict(activation="tanh"), "activation"), (dict(gate_bias=b, up_bias=b.half()), "one dtype"),
                       (dict(up=quantize_tensor(torch.randn(9, 64, device=DEV).half(), mode="channel")), "equally")):
        with pytest.raises(RuntimeError, match=needle):
            gated_w8a8(x, w, kw.pop("up", w), **kw)
    long = torch.zeros(1, 131072, dtype=torch.int8, device=DEV)
    with pytest.raises(RuntimeError, match="131071"):
        linear_w8a8(q(data=long, scale=zero, mode="tensor"), q(data=long, scale=zero, mode="tensor"))
    with pytest.raises(ValueError, match="features"):
        cuBladeW8A8LinearLayer(32, 8).to(DEV)(x)

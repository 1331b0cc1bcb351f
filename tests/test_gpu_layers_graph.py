"""The operators around a linear layer only enqueue kernels, so a HIP graph captures them: every replay, on inputs of its own
and with eager work between replays, gives what eager calls give; and the native calls give the bits of the general way."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from operators_util import randn

pytestmark = pytest.mark.gpu


class Step:
    """Every operator on tensors of its own, at sizes on either side of the kernels' choices."""

    def __init__(self, dtype, m, n, k):
        gen = torch.Generator().manual_seed(m + n + k)
        to = lambda *shape: randn(gen, *shape).to(dtype).to(dev())  # noqa: E731
        self.x, self.g, self.r = to(m, n), to(m, n), to(m, k)
        self.w, self.b, self.weight = to(n), to(n), to(k, n)
        self.bias = to(k)
        self.y, self.gx, self.gw, self.gb = (torch.empty_like(t) for t in (self.x, self.x, self.w, self.b))
        self.mean, self.rstd = (torch.empty(m, device=dev()) for _ in range(2))
        self.o, self.back, self.out = torch.empty_like(self.weight), torch.empty_like(self.weight), torch.empty_like(self.r)
        blocks = -(-n // 32)
        self.codes, self.scales = (torch.empty((k, c * blocks), dtype=torch.uint8, device=dev()) for c in (16, 1))
        space = lambda size: torch.empty(size, dtype=torch.uint8, device=dev())  # noqa: E731
        self.ns = [space(F.layer_norm_workspace(p, m, n)) for p in (0, 1)]
        self.os, self.ls = space(F.orthogonalize_workspace(1, k, n)), space(F.linear_mx4_workspace(m, n, k))

    def inputs(self):
        return [self.x, self.g, self.r, self.weight]

    def results(self):
        return [self.y, self.gx, self.gw, self.gb, self.mean, self.rstd, self.o, self.back, self.out, self.codes, self.scales]

    def run(self, stream=None):
        s = stream
        codes = [
            F.layer_norm_fprop(self.x, self.w, self.b, self.y, self.ns[0], 1e-5, self.mean, self.rstd, stream=s),
            F.layer_norm_bprop(self.x, self.w, self.mean, self.rstd, self.g, self.gx, self.gw, self.gb, self.ns[1], stream=s),
            F.orthogonalize(self.weight, self.o, self.os, scale=0.5, stream=s),
            F.mx4_quantize(self.weight, self.codes, self.scales, stream=s),
            F.mx4_dequantize(self.codes, self.scales, self.back, stream=s),
            F.linear_mx4_fprop(self.y, self.codes, self.scales, self.bias, self.out, self.ls, "gelu", self.r, stream=s)]
        assert codes == [F.Success] * 6


def captured(step):
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step.run()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step.run()
    torch.cuda.synchronize()
    return graph


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 70, 40), (50, 300, 64), (300, 2100, 600)])
def test_replays_are_eager_calls(dtype, m, n, k):
    step = Step(dtype, m, n, k)
    step.run()
    torch.cuda.synchronize()
    graph = captured(step)
    gen = torch.Generator().manual_seed(7)
    for _ in range(3):
        for t in step.inputs():
            t.copy_(randn(gen, *t.shape).to(dev()))
        for t in step.results():
            t.fill_(77)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in step.results()]
        for t in step.results():
            t.fill_(99)
        step.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step.results()))


def test_two_graphs_in_turn():
    """Two captured calls with workspaces of their own, one replayed after the other without waiting."""
    steps = [Step(torch.bfloat16, 40, 200, 64), Step(torch.bfloat16, 7, 96, 130)]
    want = []
    for s in steps:
        s.run()
        torch.cuda.synchronize()
        want.append([t.clone() for t in s.results()])
    graphs = [captured(s) for s in steps]
    for s in steps:
        for t in s.results():
            t.fill_(77)
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for s, w in zip(steps, want):
        assert all(torch.equal(a, b) for a, b in zip(s.results(), w))


def test_native_calls_are_the_general_way():
    step = Step(torch.float16, 20, 330, 33)
    kept = []
    for stream in (None, torch.cuda.current_stream()):
        for t in step.results():
            t.fill_(3)
        step.run(stream)
        torch.cuda.synchronize()
        kept.append([t.clone() for t in step.results()])
    assert all(torch.equal(a, b) for a, b in zip(*kept))
    native = F._load_native()
    x = step.x
    assert native.layer_norm_fprop(x, None, None, step.y, None, None, 1e-5, step.ns[0]) == F.Success
    for args in [(x.cpu(), None, None, step.y, None, None, 1e-5, None), (x.double(), None, None, step.y, None, None, 1e-5, None),
                 (x, None, None, step.y, None, None, 1, None), (x, None, None, step.y)]:
        assert native.layer_norm_fprop(*args) is NotImplemented
    for args in [(x, step.o, [1.0] * 15, 1e-7, 1.0, None), (x, step.o, (1.0, 2.0), 1e-7, 1.0, None),
                 (x, step.o, (1, 2, 3), 1e-7, 1.0, None), (x, step.o, (1.0,) * 99, 1e-7, 1.0, None)]:
        assert native.orthogonalize(*args) is NotImplemented
    for args in [(x, step.codes, step.scales[:1]), (x, step.codes.to(torch.int8), step.scales), (x, step.codes.t(), step.scales.t()),
                 (x, step.codes.cpu(), step.scales)]:
        assert native.mx4_quantize(*args) is NotImplemented
    with pytest.raises(ValueError):
        F.mx4_quantize(step.weight, step.codes, step.scales[:1])
    with pytest.raises(TypeError):
        F.mx4_quantize(step.weight, step.codes.to(torch.int8), step.scales)
    with pytest.raises(ValueError):
        F.mx4_dequantize(step.codes, step.scales.t(), step.back)
    torch.cuda.synchronize()


def test_refused_calls_leave_results_alone():
    step = Step(torch.float32, 50, 300, 64)
    for t in step.results():
        t.fill_(5)
    n = F.UnsupportedDimension
    assert F.layer_norm_fprop(step.x, step.w[:7], step.b, step.y, None) == n
    assert F.layer_norm_fprop(step.x, step.w, step.b, step.y, None, eps=-1.0) == F.UnsupportedSize
    assert F.layer_norm_bprop(step.x, step.w, step.mean, step.rstd, step.g, step.gx, step.gw, step.gb, step.ns[1][:256]) == n
    assert F.orthogonalize(step.weight, step.o, step.os[:512]) == n
    assert F.orthogonalize(step.weight, step.o, step.os, steps=0) == F.UnsupportedSize
    assert F.orthogonalize(step.weight, step.o, step.os, coefficients=(40.0, 0.0, 0.0)) == F.UnsupportedSize
    assert F.orthogonalize(step.weight, step.o.t(), step.os) == n
    assert F.mx4_quantize(step.weight[:, :200], step.codes, step.scales) == n
    assert F.mx4_dequantize(step.codes, step.scales, step.back[:9]) == n
    assert F.linear_mx4_fprop(step.x, step.codes, step.scales, step.bias[:5], step.out, step.ls) == n
    assert F.linear_mx4_fprop(step.x.half(), step.codes, step.scales, step.bias, step.out, step.ls) == n
    assert F.linear_mx4_fprop(step.x[:, :200], step.codes, step.scales, step.bias, step.out, step.ls) == n
    torch.cuda.synchronize()
    assert all(bool((t == 5).all()) for t in step.results())

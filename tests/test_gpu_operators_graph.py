"""The operators around a convolution layer only enqueue kernels, so a HIP graph captures them: every replay, on inputs
of its own and with eager work between replays, gives what eager calls give; and the native calls give the bits of the
general way."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from operators_util import randn

pytestmark = pytest.mark.gpu


class Step:
    """Forward and backward of each operator on tensors of its own.  Sizes on either side of the kernels' choices: groups in
    registers or in two launches, few rows, ranges of k, whole tiles."""

    def __init__(self, dtype, side, m):
        gen = torch.Generator().manual_seed(side + m)
        to = lambda *shape: randn(gen, *shape).to(dtype).to(dev())  # noqa: E731
        self.x, self.g = (to(2, side, side, 24).permute(0, 3, 1, 2) for _ in range(2))
        self.w, self.b = to(24), to(24)
        self.rows, self.weight, self.up = to(m, 264), to(136, 264), to(m, 136)
        self.bias = to(136)
        like = lambda t, **kw: torch.empty_like(t, **kw)  # noqa: E731
        self.y, self.gx, self.gw, self.gb = like(self.x), like(self.x), like(self.w), like(self.b)
        self.mean, self.rstd = (torch.empty((2, 4), device=dev()) for _ in range(2))
        self.o, self.z = like(self.up), like(self.up)
        self.grow, self.gweight, self.gbias = like(self.rows), like(self.weight), like(self.bias)
        self.d = like(self.up)
        space = lambda n: torch.empty(n, dtype=torch.uint8, device=dev())  # noqa: E731
        self.ns = [space(F.group_norm_workspace(p, self.x, 4)) for p in (0, 1)]
        self.ls = [space(F.linear_workspace(p, m, 264, 136, dtype)) for p in (0, 1)]

    def inputs(self):
        return [self.x, self.g, self.rows, self.weight, self.up]

    def results(self):
        return [self.y, self.gx, self.gw, self.gb, self.mean, self.rstd, self.o, self.z, self.grow, self.gweight, self.gbias,
                self.d]

    def run(self, stream=None):
        s = stream
        codes = [
            F.group_norm_fprop(self.x, self.w, self.b, self.y, 4, self.ns[0], "silu", 1e-5, self.mean, self.rstd, stream=s),
            F.group_norm_bprop(self.x, self.w, self.b, self.mean, self.rstd, self.g, self.gx, self.gw, self.gb, 4, self.ns[1],
                               "silu", stream=s),
            F.linear_fprop(self.rows, self.weight, self.bias, self.o, self.ls[0], "gelu", self.up, self.z, stream=s),
            F.linear_bprop(self.rows, self.weight, self.up, self.z, self.grow, self.gweight, self.gbias, self.ls[1], "gelu",
                           stream=s),
            F.dropout_fprop(self.o, self.d, 0.2, 3, 4, residual=self.up, stream=s)]
        assert codes == [F.Success] * 5


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("side,m", [(9, 1), (9, 70), (200, 700)])
def test_replays_are_eager_calls(dtype, side, m):
    step = Step(dtype, side, m)
    step.run()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        step.run()
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step.run()
    torch.cuda.synchronize()
    gen = torch.Generator().manual_seed(7)
    for _ in range(3):
        for t in step.inputs():
            t.copy_(randn(gen, *t.shape).to(dev()))
        for t in step.results():
            t.fill_(float("nan"))
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in step.results()]
        step.run()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, step.results()))


def test_native_calls_are_the_general_way():
    step = Step(torch.float16, 20, 33)
    kept = []
    for stream in (None, torch.cuda.current_stream()):
        for t in step.results():
            t.fill_(-3.0)
        step.run(stream)
        torch.cuda.synchronize()
        kept.append([t.clone() for t in step.results()])
    assert all(torch.equal(a, b) for a, b in zip(*kept))
    native = F._load_native()
    x = step.x
    assert native.group_norm_fprop(x, None, None, step.y, None, None, 4, 1e-5, 0, step.ns[0]) == F.Success
    for args in [(x.cpu(), None, None, step.y, None, None, 4, 1e-5, 0, None), (x.double(), None, None, step.y, None, None, 4, 1e-5, 0, None),
                 (x, None, None, step.y, None, None, 4.0, 1e-5, 0, None), (x, None, None, step.y)]:
        assert native.group_norm_fprop(*args) is NotImplemented
    with pytest.raises(TypeError):
        F.dropout_fprop(x, step.y, 0.1, 1, 2, step=torch.zeros(1, device=dev()))
    with pytest.raises(ValueError):
        F.dropout_fprop(x, step.y, 0.1, -1, 2)
    torch.cuda.synchronize()


def test_refused_calls_leave_results_alone():
    step = Step(torch.float32, 9, 70)
    step.y.fill_(5.0)
    step.o.fill_(5.0)
    assert F.group_norm_fprop(step.x, step.w, step.b, step.y, 5, step.ns[0]) == F.UnsupportedSize
    assert F.group_norm_fprop(step.x, step.w[:7], step.b, step.y, 4, step.ns[0]) == F.UnsupportedDimension
    assert F.linear_fprop(step.rows, step.weight[:, 1:], step.bias, step.o, step.ls[0]) == F.UnsupportedDimension
    assert F.linear_fprop(step.rows.half(), step.weight, step.bias, step.o, step.ls[0]) == F.UnsupportedDimension
    assert F.linear_bprop(step.rows, step.weight, step.up, step.z, step.grow, step.gweight, step.gbias, step.ls[1][:256],
                          "gelu") == F.UnsupportedDimension
    assert F.dropout_fprop(step.up, step.o[:3], 0.5, 1, 2) == F.UnsupportedDimension
    torch.cuda.synchronize()
    assert bool((step.y == 5.0).all()) and bool((step.o == 5.0).all())

"""The operators as examples/served_layer.py runs them together: the gradients and the update of a step are those of the same
block in 64 bits with torch's own differentiation, and rows served in 4 bits those of the quantised formula."""
import importlib.util
import math
import os

import pytest
import torch

from layers_util import QUINTIC, orthogonal, orthogonal_bound, quantized, values_of

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("served_layer", os.path.join(ROOT, "examples", "served_layer.py"))
E = importlib.util.module_from_spec(spec)
spec.loader.exec_module(E)


def norm(x, gamma, beta):
    mean = x.mean(-1, keepdim=True)
    return (x - mean) / (x.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt() * gamma + beta


def test_it_trains_and_serves_and_is_reproducible():
    losses = []
    for _ in range(2):
        block = E.Block(rows=100, width=40, hidden=72)
        losses.append(E.train(block, *E.data(block), 6))
    assert all(math.isfinite(v) for v in losses[0]) and losses[0] == losses[1]
    x, _ = E.data(block)
    served = E.Served(block, rows=3)
    assert bool(torch.isfinite(served(x[:3])).all())


@pytest.mark.parametrize("rows,width,hidden", [(3, 20, 33), (130, 96, 320)])
def test_gradients_and_update_of_a_step(rows, width, hidden):
    block = E.Block(rows, width, hidden, seed=4)
    x, target = E.data(block)
    off = block.forward(x) - target
    dx = block.backward(x, off * (2 / off.numel()))
    p = {k: v.cpu().double().requires_grad_() for k, v in block.params.items()}
    x64 = x.cpu().double().requires_grad_()
    h = torch.nn.functional.gelu(norm(x64, p["gamma"], p["beta"]) @ p["w1"].t() + p["b1"])
    loss = (h @ p["w2"].t() + p["b2"] + x64 - target.cpu().double()).square().mean()
    loss.backward()
    assert abs(float(off.square().mean()) - loss.item()) < 1e-5 * loss.item()
    for k, got, want in [("x", dx, x64.grad)] + [(k, block.grads[k], v.grad) for k, v in p.items()]:
        # fp32 through five operators
        far = float((got.cpu().double() - want).norm() / want.norm())
        assert far < 1e-5, "%s: %.2e" % (k, far)
    before = {k: block.params[k].clone() for k in block.update}
    block.step(rate=0.5)
    for k, w in before.items():
        scale = max(1.0, w.shape[0] / w.shape[1]) ** 0.5
        want, bound, _ = orthogonal_bound(block.grads[k][None], [QUINTIC] * 5, 1e-7, scale)
        moved = (w - block.params[k]).cpu().double() / 0.5
        # (and the roundings of w and of its difference)
        assert float((moved - want[0]).norm()) < float(bound) + 2 * 2.0 ** -24 / 0.5 * float(w.norm()) + 2.0 ** -23 * float(want.norm())


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 5, 70])
def test_served_rows(rows, dtype):
    block = E.Block(100, 64, 200, seed=5, dtype=dtype)
    x, _ = E.data(block)
    served = E.Served(block, rows)
    y = served(x[:rows])
    v = lambda t: values_of(*quantized(t.cpu()), t.shape[1])  # noqa: E731
    p = block.params
    # from what each operator was given: a rounding may move a value into the next code
    n = norm(x[:rows].cpu().double(), p["gamma"].cpu().double(), p["beta"].cpu().double())
    u = {torch.float32: 2.0 ** -20, torch.bfloat16: 2.0 ** -8}[dtype]
    assert bool(((served.n.cpu().double() - n).abs() <= u * (1 + n.abs())).all())
    h = torch.nn.functional.gelu(v(served.n) @ v(p["w1"]).t() + p["b1"].cpu().double())
    assert bool(((served.h.cpu().double() - h).abs() <= u * (1 + h.abs())).all())
    want = v(served.h) @ v(p["w2"]).t() + p["b2"].cpu().double() + x[:rows].cpu().double()
    assert bool(((y.cpu().double() - want).abs() <= u * (1 + want.abs())).all())


def test_a_served_row_in_a_graph():
    block = E.Block(16, 64, 200, seed=6, dtype=torch.bfloat16)
    x, _ = E.data(block)
    served, row = E.Served(block), x[:1].clone()
    served(row)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        with torch.cuda.graph(graph, stream=stream):
            served(row)
    torch.cuda.synchronize()
    for i in range(5):
        row.copy_(x[i:i + 1])
        graph.replay()
        torch.cuda.synchronize()
        got = served.y.clone()
        assert torch.equal(served(row), got)
        torch.cuda.synchronize()

"""The operators around a linear layer at their largest sizes, with operands of unlike types, and large ones in graphs."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import quantized, values_of
from operators_util import NAMES, TYPES, linear, randn, rounded, within
from test_gpu_mx4 import matrix, packed, quantize
from test_gpu_orthogonalize import check as updates

pytestmark = pytest.mark.gpu


def whole(gen, *shape):
    """Whole numbers that 4 bits hold under the scale 1: blocks whose largest magnitude is 4.  Their products' sums are exact."""
    v = torch.randint(-3, 4, shape, generator=gen, device=dev())
    v[:, ::32] = 4
    return v.to(torch.bfloat16)


def space(m, k, n):
    return torch.empty(F.linear_mx4_workspace(m, k, n), dtype=torch.uint8, device=dev())


@pytest.mark.parametrize("m,n", [((1 << 23) - 1, 3), (3, (1 << 23) - 1), ((1 << 23) - 1, 130)])
def test_as_many_rows_and_outputs_as_there_may_be(m, n):
    gen = torch.Generator(device=dev()).manual_seed(1)
    x, w = whole(gen, m, 40), whole(gen, n, 40)
    y = torch.full((m, n), 7.0, dtype=torch.float16, device=dev())
    weight = quantize(w)
    for rows in (None, quantize(x)):
        if rows is None:
            assert F.linear_mx4_fprop(x.half(), *weight, None, y, space(m, 40, n)) == F.Success
        else:
            assert F.linear_mx4_fprop(rows[0], *weight, None, y, space(m, 40, n), inputScales=rows[1]) == F.Success
        torch.cuda.synchronize()
        assert torch.equal(y, (x.float() @ w.float().t()).half())
        y.fill_(7.0)


def test_rows_as_long_as_they_may_be():
    gen = torch.Generator(device=dev()).manual_seed(2)
    for m, k, n in ((2, 1 << 22, 5), (20, (1 << 22) - 5, 17), (140, (1 << 21) + 3, 130)):
        x, w = whole(gen, m, k), whole(gen, n, k)
        y = torch.full((m, n), 7.0, device=dev())
        assert F.linear_mx4_fprop(x.float(), *quantize(w), None, y, space(m, k, n)) == F.Success
        torch.cuda.synchronize()
        # (whole numbers around k / 2, as their partial sums are: exact below 2^24)
        want = x.double() @ w.double().t()
        assert float(want.abs().max()) < 1 << 23 and torch.equal(y.double(), want)
        del x, w


def test_more_values_than_a_launch_has_lanes_for():
    """2^18 times 2^15 values and more, all rows the same one."""
    gen = torch.Generator().manual_seed(3)
    m, k = (1 << 18) + 3, 1 << 15
    row = matrix(randn(gen, 1, k), torch.float16)
    codes, scales = packed(m, k)
    assert F.mx4_quantize(row.expand(m, k), codes, scales) == F.Success
    torch.cuda.synchronize()
    want = quantized(row)
    assert torch.equal(codes[-1:].cpu(), want[0]) and torch.equal(scales[-1:].cpu(), want[1])
    assert bool((codes == codes[-1:]).all()) and bool((scales == scales[-1:]).all())
    y = torch.full((m, k), 7.0, dtype=torch.bfloat16, device=dev())
    assert F.mx4_dequantize(codes, scales, y) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y[-1:].cpu(), values_of(*want, k).to(torch.bfloat16)) and bool((y == y[-1:]).all())


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("kind", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(1, 96, 70), (40, 500, 135), (1111, 1151, 1009), (1031, 333, 7183), (264, 4352, 1304)], ids=str)
def test_biases_of_every_type_and_stride(shape, kind, dtype):
    m, k, n = shape
    gen = torch.Generator().manual_seed(4)
    x, w = matrix(randn(gen, m, k), dtype), quantize(matrix(randn(gen, n, k) * k ** -0.5, dtype))
    bias = matrix(randn(gen, n, 1), kind, "apart")[:, 0]
    assert bias.stride(0) > 1 or n == 1
    y = torch.full((m, n), 7.0, dtype=dtype, device=dev())
    assert F.linear_mx4_fprop(x, *w, bias, y, space(m, k, n), activation="relu") == F.Success
    torch.cuda.synchronize()
    want, bound, _, _ = linear(values_of(*quantize(x), k), values_of(*w, k), bias, None, "relu")
    within(y, want, rounded(want, dtype) + bound)
    again = torch.full_like(y, 7.0)
    assert F.linear_mx4_fprop(x, *w, bias.contiguous(), again, space(m, k, n), activation="relu") == F.Success
    torch.cuda.synchronize()
    assert torch.equal(again, y)


@pytest.mark.parametrize("shape", [(1111, 1151, 1009), (1031, 333, 7183), (264, 4352, 1304)], ids=str)
def test_tiles_in_a_graph(shape):
    m, k, n = shape
    gen = torch.Generator().manual_seed(5)
    x, w = matrix(randn(gen, m, k), torch.bfloat16), quantize(matrix(randn(gen, n, k), torch.bfloat16))
    replays_are_eager(x, torch.empty((m, n), dtype=torch.bfloat16, device=dev()), lambda y, ws: F.linear_mx4_fprop(x, *w, None, y, ws, "gelu"),
                      F.linear_mx4_workspace(m, k, n))


@pytest.mark.parametrize("shape", [(3, 97, 2164), (31, 3203, 206), (8, 1412, 1469), (1, 2047, 4000)], ids=str)
def test_large_matrices_in_a_graph(shape):
    gen = torch.Generator().manual_seed(6)
    x = randn(gen, *shape).to(torch.bfloat16).to(dev())
    replays_are_eager(x, torch.empty_like(x), lambda y, ws: F.orthogonalize(x, y, ws), F.orthogonalize_workspace(*shape))


def replays_are_eager(x, y, call, size):
    spaces = [torch.empty(size, dtype=torch.uint8, device=dev()) for _ in range(2)]
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        assert call(y, spaces[0]) == F.Success
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            assert call(y, spaces[0]) == F.Success
    torch.cuda.synchronize()
    for i in range(3):
        x.mul_(-1.5)
        spaces[0].fill_(255)
        y.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        want = torch.full_like(y, 9.0)
        assert call(want, spaces[1]) == F.Success
        torch.cuda.synchronize()
        assert torch.equal(y, want)


def test_workspaces_that_are_no_memory_of_the_gpu_are_refused():
    g = torch.ones((300, 300), device=dev())
    y = torch.full_like(g, 7.0)
    small, host = torch.empty(256, dtype=torch.uint8, device=dev())[:1].expand(1 << 30), torch.empty(1 << 24, dtype=torch.uint8)
    for stream in (None, torch.cuda.current_stream()):  # (the native call, and the general way)
        assert F.orthogonalize(g, y, small, stream=stream) == F.UnsupportedDimension
        with pytest.raises(ValueError):
            F.orthogonalize(g, y, host, stream=stream)
        with pytest.raises(ValueError):
            F.layer_norm_bprop(g, None, g[0], g[0], g, y, y[0], y[0], host, stream=stream)
    torch.cuda.synchronize()
    assert bool((y == 7).all())


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(20, 40), (130, 150), (300, 1200)], ids=str)
def test_matrices_far_smaller_than_eps(shape, dtype):
    """X is then small in front of every step, and the least step of what is held between products, 2^-35, counts."""
    gen = torch.Generator().manual_seed(7)
    g = randn(gen, *shape).to(dtype).to(dev())
    for eps in (1e1, 1e4, 1e6, 1e9):
        updates(g, eps=eps * float(g.norm()))

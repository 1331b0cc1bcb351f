"""Products with bias, activation and residual in their epilogue, and their gradients, against their plain form in 64
bits."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from operators_util import ACTS, NAMES, R, TYPES, linear, linear_grads, randn, rounded, within

pytestmark = pytest.mark.gpu


def matrix(values, dtype, form="rows"):
    r, c = values.shape
    v = values.to(dtype).to(dev())
    if form == "rows":
        return v
    if form == "cols":  # the first index is contiguous
        return v.t().contiguous().t()
    if form == "pitch":  # rows apart, off any 16-byte boundary
        t = torch.zeros((r, c + 7), dtype=dtype, device=dev())[:, 3:3 + c]
    else:  # every second element of every third row
        t = torch.zeros((3 * r, 2 * c), dtype=dtype, device=dev())[::3, ::2]
    return t.copy_(v)


def space(pass_, m, k, n, dtype):
    return torch.empty(F.linear_workspace(pass_, m, k, n, dtype), dtype=torch.uint8, device=dev())


def make(m, k, n, dtype, seed, form="rows", wform="rows"):
    gen = torch.Generator().manual_seed(seed)
    x, w = randn(gen, m, k), randn(gen, n, k, std=max(1, k) ** -0.5)
    bias, r, gy = randn(gen, n, std=0.3), randn(gen, m, n), randn(gen, m, n, std=0.1)
    return (matrix(x, dtype, form), matrix(w, dtype, wform), bias.float().to(dev()), matrix(r, dtype, form),
            matrix(gy, dtype, form))


def check_forward(x, w, bias, r, name, save=True, form="rows"):
    m, k = x.shape
    n = w.shape[0]
    fill = torch.full((m, n), 7.0, dtype=torch.float64)
    y, z = matrix(fill, x.dtype, form), matrix(fill, x.dtype, form) if save else None
    assert F.linear_fprop(x, w, bias, y, space(0, m, k, n, x.dtype), activation=name, residual=r,
                          preactivation=z) == F.Success
    torch.cuda.synchronize()
    wy, by, wz, bz = linear(x, w, bias, r, name)
    within(y, wy, rounded(wy, x.dtype) + by)
    if save:
        within(z, wz, rounded(wz, x.dtype) + bz)
    return y, z


def check_backward(x, w, gy, z, name, form="rows"):
    m, k = x.shape
    n = w.shape[0]
    fill = lambda a, b: matrix(torch.full((a, b), 7.0, dtype=torch.float64), x.dtype, form)  # noqa: E731
    gx, gw, gb = fill(m, k), fill(n, k), torch.full((n,), 7.0, device=dev())
    z = None if name == "none" else z
    assert F.linear_bprop(x, w, gy, z, gx, gw, gb, space(1, m, k, n, x.dtype), activation=name) == F.Success
    torch.cuda.synchronize()
    (wx, bx), (ww, bw), (wb, bb) = linear_grads(x, w, gy, z, name, x.dtype)
    within(gx, wx, rounded(wx, x.dtype) + bx)
    within(gw, ww, rounded(ww, x.dtype) + bw)
    within(gb, wb, rounded(wb, torch.float32) + bb)
    return gx, gw, gb


# (M, K, N): single rows, columns and products; the sides of tiles and steps and one beyond; ragged ones; long sums
SHAPES = [(1, 1, 1), (1, 2048, 33), (1, 96, 1000), (2, 64, 64), (5, 333, 70), (16, 128, 48), (17, 40, 200), (33, 31, 1),
          (64, 64, 64), (65, 72, 130), (128, 32, 128), (129, 33, 127), (200, 264, 256), (300, 1151, 100), (257, 96, 520),
          (4, 4104, 16), (40, 16, 3000), (3000, 24, 40)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, dtype):
    m, k, n = shape
    name = ACTS[(m + k + n) % 4]
    x, w, bias, r, gy = make(m, k, n, dtype, 1)
    _, z = check_forward(x, w, bias, r, name)
    check_backward(x, w, gy, z, name)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("form,wform", [("cols", "rows"), ("rows", "cols"), ("cols", "cols"), ("pitch", "pitch"),
                                        ("apart", "rows"), ("rows", "apart"), ("apart", "apart")])
@pytest.mark.parametrize("shape", [(1, 72, 40), (3, 50, 67), (130, 72, 136), (70, 45, 33), (520, 256, 264)], ids=str)
def test_strides(shape, form, wform, dtype):
    m, k, n = shape
    x, w, bias, r, gy = make(m, k, n, dtype, 2, form, wform)
    _, z = check_forward(x, w, bias, r, "silu", form=form)
    check_backward(x, w, gy, z, "silu", form=form)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("m", [1, 12, 150, 1100])
def test_activations_and_what_may_be_left_out(m, dtype, name):
    k, n = 128, 264
    x, w, bias, r, gy = make(m, k, n, dtype, 3)
    _, z = check_forward(x, w, bias, r, name)
    check_forward(x, w, None, None, name, save=False)
    grads = check_backward(x, w, gy, z, name)
    z = None if name == "none" else z
    only = [torch.full_like(g, 7.0) for g in grads]
    ws = space(1, m, k, n, dtype)
    assert F.linear_bprop(None, w, gy, z, only[0], None, None, ws, activation=name) == F.Success
    assert F.linear_bprop(x, None, gy, z, None, only[1], None, ws, activation=name) == F.Success
    assert F.linear_bprop(None, None, gy, z, None, None, only[2], ws, activation=name) == F.Success
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(only, grads))  # and reproducible


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_large(dtype):
    """Whole tiles of every size, long reductions, many tiles."""
    x, w, bias, r, gy = make(1536, 1024, 1280, dtype, 4)
    _, z = check_forward(x, w, bias, r, "gelu")
    check_backward(x, w, gy, z, "gelu")


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("m", [1, 40, 600])
def test_broadcast_operands_and_residual_in_place(m, dtype):
    x, w, bias, r, _ = make(m, 64, 96, dtype, 5)
    check_forward(x[:1].expand(m, 64), w, bias, r[:1].expand(m, 96), "silu")
    wy, by, _, _ = linear(x, w, bias, r, "relu")
    assert F.linear_fprop(x, w, bias.to(dtype), r, space(0, m, 64, 96, dtype), activation="relu", residual=r) == F.Success
    if dtype == torch.float32:
        within(r, wy, rounded(wy, dtype) + by)
    else:
        wy, by, _, _ = linear(x, w, bias.to(dtype), make(m, 64, 96, dtype, 5)[3], "relu")
        within(r, wy, rounded(wy, dtype) + by)


def test_nothing_to_sum():
    d = dev()
    bias, r = torch.randn(8, device=d), torch.randn(3, 8, device=d)
    y = torch.full((3, 8), 7.0, device=d)
    assert F.linear_fprop(torch.empty((3, 0), device=d), torch.empty((8, 0), device=d), bias, y, None, residual=r) == F.Success
    assert torch.equal(y, bias + r)
    assert F.linear_fprop(torch.empty((0, 5), device=d), torch.empty((8, 5), device=d), bias,
                          torch.empty((0, 8), device=d), None) == F.Success
    # no rows: the gradients of the weights are sums of nothing
    gw, gb = torch.full((8, 5), 7.0, device=d), torch.full((8,), 7.0, device=d)
    assert F.linear_bprop(torch.empty((0, 5), device=d), torch.empty((8, 5), device=d), torch.empty((0, 8), device=d), None,
                          torch.empty((0, 5), device=d), gw, gb, None) == F.Success
    assert not bool(gw.any()) and not bool(gb.any())
    # no outputs: the input's gradient is one
    gx = torch.full((3, 5), 7.0, device=d)
    assert F.linear_bprop(torch.empty((3, 5), device=d), torch.empty((0, 5), device=d), torch.empty((3, 0), device=d), None,
                          gx, torch.empty((0, 5), device=d), torch.empty((0,), device=d), None) == F.Success
    assert not bool(gx.any())


@pytest.mark.parametrize("m", [2, 100, 700])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_values_that_are_not_finite_stay_in_their_rows(m, dtype):
    x, w, bias, _, _ = make(m, 96, 136, dtype, 6)
    x[1, 5] = float("nan")
    y, _ = torch.empty((m, 136), dtype=dtype, device=dev()), None
    assert F.linear_fprop(x, w, bias, y, space(0, m, 96, 136, dtype)) == F.Success
    assert bool(torch.isnan(y[1]).all())
    assert bool(torch.isfinite(y[torch.arange(m, device=dev()) != 1]).all())
    x[1, 5] = float("inf")
    assert F.linear_fprop(x, w, bias, y, space(0, m, 96, 136, dtype)) == F.Success
    assert not bool(torch.isfinite(y[1]).any())
    assert bool(torch.isfinite(y[torch.arange(m, device=dev()) != 1]).all())


def test_float32_keeps_its_range():
    """Pieces of large and small numbers: nothing overflows in the cut, and small ones keep their bits."""
    gen = torch.Generator().manual_seed(7)
    for scale, other in ((3e38, 1e-3), (1e-30, 1.0), (1e30, 1e-25)):
        x, w = randn(gen, 70, 40).clamp(-1, 1) * scale, randn(gen, 50, 40).clamp(-1, 1) * other
        x, w = x.float().to(dev()), w.float().to(dev())
        y = torch.empty((70, 50), device=dev())
        assert F.linear_fprop(x, w, None, y, space(0, 70, 40, 50, torch.float32)) == F.Success
        want = x.cpu().double() @ w.cpu().double().t()
        size = x.cpu().double().abs() @ w.cpu().double().abs().t()
        within(y, want, R * (8 + 2 * 40 ** 0.5) * size)


@pytest.mark.parametrize("m", [3, 200])
def test_gradients_are_differences(m):
    gen = torch.Generator().manual_seed(8)
    k, n, h = 48, 80, 1e-2
    v, d, r = randn(gen, m, k), randn(gen, m, k), randn(gen, m, n)
    weight, dw, bias, db = randn(gen, n, k) * k ** -0.5, randn(gen, n, k) * k ** -0.5, randn(gen, n), randn(gen, n)
    to = lambda t: t.float().to(dev())  # noqa: E731

    def loss(s):
        x, w, b = to(v + s * d), to(weight + s * dw), to(bias + s * db)
        y, z = torch.empty((m, n), device=dev()), torch.empty((m, n), device=dev())
        assert F.linear_fprop(x, w, b, y, space(0, m, k, n, torch.float32), activation="gelu", preactivation=z) == F.Success
        return float((y.double().cpu() * r).sum()), (x, w, b, z)

    _, (x, w, b, z) = loss(0.0)
    gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    assert F.linear_bprop(x, w, to(r), z, gx, gw, gb, space(1, m, k, n, torch.float32), activation="gelu") == F.Success
    slope = sum(float((g.double().cpu() * e).sum()) for g, e in ((gx, d), (gw, dw), (gb, db)))
    # h^2 / 6 times a third derivative: z moves by about 2 a unit of h and twice its square, so about 40 a term
    allowed = (h * h / 6 * 40 * 4 + 16 * R / h) * (m * n) ** 0.5
    assert abs((loss(h)[0] - loss(-h)[0]) / (2 * h) - slope) <= allowed


def test_other_streams_and_the_general_way():
    x, w, bias, r, gy = make(90, 64, 72, torch.bfloat16, 9)
    y, z = torch.empty((90, 72), dtype=torch.bfloat16, device=dev()), torch.empty((90, 72), dtype=torch.bfloat16, device=dev())
    ws = space(0, 90, 64, 72, torch.bfloat16)
    assert F.linear_fprop(x, w, bias, y, ws, activation="silu", residual=r) == F.Success
    torch.cuda.synchronize()
    assert F.linear_fprop(x, w, bias, z, ws, activation="silu", residual=r, stream=torch.cuda.Stream()) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_offsets_past_32_bits():
    far = (1 << 32) + 8
    store = torch.zeros(2 * far + 512, dtype=torch.bfloat16, device=dev())
    x = store.as_strided((3, 64), (far, 1))
    gen = torch.Generator().manual_seed(10)
    x.copy_(randn(gen, 3, 64).to(dev()))
    w = randn(gen, 40, 64).to(torch.bfloat16).to(dev())
    check_forward(x, w, None, None, "none")
    # 40 rows: a tile, not the way of a few rows
    x = store.as_strided((40, 64), ((1 << 26) * 3 + 8, 1))
    x.copy_(randn(gen, 40, 64).to(dev()))
    check_forward(x, w, None, None, "none")
    del store


def test_rows_of_64_images_of_256_by_256():
    m, k, n = 1 << 22, 16, 16
    x, w, bias, r, gy = make(m, k, n, torch.bfloat16, 12)
    check_forward(x, w, bias, None, "relu")
    check_backward(x, w, gy, r, "relu")


@pytest.mark.parametrize("name", ["none", "silu"])
@pytest.mark.parametrize("m", [65535 * 32, 65535 * 32 + 1])
def test_backward_of_many_rows(m, name):
    """Parts of 32 rows, as many as 16 bits count and one more: the pixels of 32 images of 256 x 256 are that many rows."""
    x, w, bias, r, gy = make(m, 8, 16, torch.bfloat16, 11)
    check_backward(x, w, gy, r, name)

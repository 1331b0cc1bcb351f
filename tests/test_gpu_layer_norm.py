"""Layer norm of rows and its gradients against their plain form in 64 bits."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import layer_norm, layer_norm_grads
from operators_util import NAMES, R, TYPES, randn, rounded, within

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


def space(pass_, m, n):
    return torch.empty(F.layer_norm_workspace(pass_, m, n), dtype=torch.uint8, device=dev())


def make(m, n, dtype, seed, form="rows"):
    gen = torch.Generator().manual_seed(seed)
    x = randn(gen, m, n) * (0.5 + randn(gen, m, 1).abs()) + randn(gen, m, 1, std=0.5)
    w, b = randn(gen, n, std=0.3, mean=1.0), randn(gen, n, std=0.3)
    return matrix(x, dtype, form), w.float().to(dev()), b.float().to(dev()), matrix(randn(gen, m, n), dtype, form)


def check_forward(x, w, b, eps=1e-5, form="rows", save=True):
    m, n = x.shape
    y = matrix(torch.full((m, n), 7.0, dtype=torch.float64), x.dtype, form)
    mean, rstd = (torch.full((m,), 7.0, device=dev()) for _ in range(2)) if save else (None, None)
    assert F.layer_norm_fprop(x, w, b, y, space(0, m, n), eps=eps, mean=mean, rstd=rstd) == F.Success
    torch.cuda.synchronize()
    (wy, by), (wm, bm), (wr, br) = layer_norm(x, w, b, eps)
    within(y, wy, rounded(wy, x.dtype) + by)
    if save:
        within(mean, wm, bm + R * wm.abs())
        within(rstd, wr, br)
    return y, mean, rstd


def check_backward(x, w, mean, rstd, g, form="rows", kind=torch.float32):
    m, n = x.shape
    gx = matrix(torch.full((m, n), 7.0, dtype=torch.float64), x.dtype, form)
    gw, gb = (torch.full((n,), 7.0, dtype=kind, device=dev()) for _ in range(2))
    assert F.layer_norm_bprop(x, w, mean, rstd, g, gx, gw, gb, space(1, m, n)) == F.Success
    torch.cuda.synchronize()
    (wx, bx), (ww, bw), (wb, bb) = layer_norm_grads(x, w, mean, rstd, g)
    within(gx, wx, rounded(wx, x.dtype) + bx)
    within(gw, ww, rounded(ww, kind) + bw)
    within(gb, wb, rounded(wb, kind) + bb)
    return gx, gw, gb


# single rows and values; the sides of words, waves and workgroups and one beyond; rows that no registers hold
SHAPES = [(1, 1), (3, 1), (5, 2), (4, 7), (2, 8), (7, 9), (9, 31), (130, 32), (33, 63), (17, 64), (70, 65), (6, 127), (257, 128),
          (300, 192), (5, 255), (64, 256), (3, 511), (1, 512), (19, 513), (40, 1000), (2, 1024), (35, 1025), (1, 2048), (600, 2048),
          (3, 2049), (5, 4096), (2, 4100), (9, 8191), (1, 8192), (2, 8200), (3, 16384), (2, 16390), (1, 32768), (2, 40001),
          (1, 70000), (5000, 24), (2100, 129)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, dtype):
    x, w, b, g = make(*shape, dtype, 1)
    _, mean, rstd = check_forward(x, w, b)
    check_backward(x, w, mean, rstd, g)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("form", ["cols", "pitch", "apart"])
@pytest.mark.parametrize("shape", [(1, 40), (37, 72), (70, 133), (9, 520), (12, 2048), (5, 4103), (2, 20000)], ids=str)
def test_strides(shape, form, dtype):
    x, w, b, g = make(*shape, dtype, 2, form)
    _, mean, rstd = check_forward(x, w, b, form=form)
    check_backward(x, w, mean, rstd, g, form=form)
    # operands of unlike layouts
    y = torch.empty(shape, dtype=dtype, device=dev())
    assert F.layer_norm_fprop(x, w, b, y, space(0, *shape)) == F.Success
    (wy, by), _, _ = layer_norm(x, w, b, 1e-5)
    within(y, wy, rounded(wy, dtype) + by)
    check_backward(x, w, mean, rstd, g.contiguous(), form=form)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(3, 30), (200, 96), (50, 1000), (11, 5000), (2, 33000)], ids=str)
def test_what_may_be_left_out(shape, dtype):
    m, n = shape
    x, w, b, g = make(m, n, dtype, 3)
    check_forward(x, None, None)
    check_forward(x, w, None, save=False)
    check_forward(x, None, b, eps=0.0)
    _, mean, rstd = check_forward(x, w.to(dtype), b.to(dtype))
    check_backward(x, None, mean, rstd, g)
    grads = check_backward(x, w.to(dtype), mean, rstd, g, kind=dtype)
    only = [torch.full_like(t, 7.0) for t in grads]
    ws, p = space(1, m, n), w.to(dtype)
    assert F.layer_norm_bprop(x, p, mean, rstd, g, only[0], None, None, ws) == F.Success
    assert F.layer_norm_bprop(x, p, mean, rstd, g, None, only[1], None, ws) == F.Success
    assert F.layer_norm_bprop(x, p, mean, rstd, g, None, None, only[2], ws) == F.Success
    torch.cuda.synchronize()
    assert all(torch.equal(a, c) for a, c in zip(only, grads))  # and reproducible
    # parameters and statistics that are not dense
    far = torch.zeros((n, 3), device=dev())
    far[:, 1] = w
    stats = torch.zeros((m, 2), device=dev())
    y, z = torch.empty_like(x), torch.empty_like(x)
    assert F.layer_norm_fprop(x, far[:, 1], b, y, space(0, m, n), mean=stats[:, 0], rstd=stats[:, 1]) == F.Success
    assert F.layer_norm_fprop(x, w, b, z, space(0, m, n)) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, z) and torch.equal(stats[:, 0], mean) and torch.equal(stats[:, 1], rstd)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("form", ["rows", "pitch", "cols"])
@pytest.mark.parametrize("shape", [(40, 64), (7, 1500), (3, 9000), (2, 36000)], ids=str)
def test_in_place(shape, form, dtype):
    x, w, b, g = make(*shape, dtype, 4, form)
    want, mean, rstd = check_forward(x, w, b, form=form)
    gx, gw, gb = check_backward(x, w, mean, rstd, g, form=form)
    for target in (g, x):
        operand = {"x": x, "g": g}
        again = matrix(target.clone(), dtype, form)
        operand["g" if target is g else "x"] = again
        aw, ab = torch.empty_like(gw), torch.empty_like(gb)
        assert F.layer_norm_bprop(operand["x"], w, mean, rstd, operand["g"], again, aw, ab, space(1, *shape)) == F.Success
        torch.cuda.synchronize()
        assert torch.equal(again, gx) and torch.equal(aw, gw) and torch.equal(ab, gb)
    assert F.layer_norm_fprop(x, w, b, x, space(0, *shape)) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(x, want)


@pytest.mark.parametrize("n", [5, 64, 1000, 4096, 9001, 40000])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_rows_of_one_value_and_far_from_zero(n, dtype):
    """Rows without variance, and rows whose deviation is small beside their mean."""
    gen = torch.Generator().manual_seed(5)
    x = torch.full((6, n), 3.0, dtype=torch.float64)
    x[1] = 0
    x[2] = -700.0
    x[3] = 1000 + randn(gen, n)
    x[4] = -5 + 0.01 * randn(gen, n)
    x[5] = 30000 + 16 * randn(gen, n)
    x = matrix(x, dtype)
    w, b = randn(gen, n).float().to(dev()), randn(gen, n).float().to(dev())
    _, mean, rstd = check_forward(x, w, b)
    check_backward(x, w, mean, rstd, matrix(randn(gen, 6, n), dtype))


@pytest.mark.parametrize("n", [40, 600, 5000, 35000])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_values_that_are_not_finite_stay_in_their_rows(n, dtype):
    x, w, b, g = make(9, n, dtype, 6)
    clean = torch.ones(9, dtype=torch.bool, device=dev())
    x[2, 3], x[5, n - 1] = float("nan"), float("inf")
    clean[2] = clean[5] = False
    y, mean, rstd = torch.empty_like(x), torch.empty(9, device=dev()), torch.empty(9, device=dev())
    assert F.layer_norm_fprop(x, w, b, y, space(0, 9, n), mean=mean, rstd=rstd) == F.Success
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[5]).all())
    assert bool(torch.isfinite(y[clean]).all())
    gx, gw, gb = torch.empty_like(x), torch.empty(n, device=dev()), torch.empty(n, device=dev())
    assert F.layer_norm_bprop(x, w, mean, rstd, g, gx, gw, gb, space(1, 9, n)) == F.Success
    assert bool(torch.isnan(gx[2]).all()) and bool(torch.isfinite(gx[clean]).all())
    assert bool(torch.isnan(gw).all()) and bool(torch.isfinite(gb).all())


def test_nothing_to_norm():
    d = dev()
    empty = torch.empty((0, 12), device=d)
    stats = torch.empty((0,), device=d)
    assert F.layer_norm_fprop(empty, None, None, empty, None, mean=stats, rstd=stats) == F.Success
    gw, gb = torch.full((12,), 7.0, device=d), torch.full((12,), 7.0, device=d)
    assert F.layer_norm_bprop(empty, None, stats, stats, empty, empty, gw, gb, None) == F.Success
    assert not bool(gw.any()) and not bool(gb.any())
    none = torch.empty((3, 0), device=d)
    assert F.layer_norm_fprop(none, None, None, none, None) == F.Success
    s = torch.zeros(3, device=d)
    assert F.layer_norm_bprop(none, None, s, s, none, none, none[0], none[0], None) == F.Success


@pytest.mark.parametrize("n", [48, 3000, 33000])
def test_gradients_are_differences(n):
    gen = torch.Generator().manual_seed(8)
    m, h = 6, 1e-2
    v, d, r = randn(gen, m, n), randn(gen, m, n), randn(gen, m, n)
    weight, dw, bias, db = randn(gen, n, mean=1.0), randn(gen, n), randn(gen, n), randn(gen, n)
    to = lambda t: t.float().to(dev())  # noqa: E731

    def loss(s):
        x, w, b = to(v + s * d), to(weight + s * dw), to(bias + s * db)
        y, mean, rstd = torch.empty_like(x), torch.empty(m, device=dev()), torch.empty(m, device=dev())
        assert F.layer_norm_fprop(x, w, b, y, space(0, m, n), mean=mean, rstd=rstd) == F.Success
        return float((y.double().cpu() * r).sum()), (x, w, mean, rstd)

    _, (x, w, mean, rstd) = loss(0.0)
    gx, gw, gb = torch.empty_like(x), torch.empty(n, device=dev()), torch.empty(n, device=dev())
    assert F.layer_norm_bprop(x, w, mean, rstd, to(r), gx, gw, gb, space(1, m, n)) == F.Success
    slope = sum(float((g.double().cpu() * e).sum()) for g, e in ((gx, d), (gw, dw), (gb, db)))
    # h^2 / 6 times a third derivative: xh and its derivatives are about 1 to 6 a term, times weights of about 2
    allowed = (h * h / 6 * 60 + 32 * R / h) * (m * n) ** 0.5
    assert abs((loss(h)[0] - loss(-h)[0]) / (2 * h) - slope) <= allowed


def test_broadcast_rows():
    x, w, b, g = make(1, 300, torch.bfloat16, 9)
    rows = x.expand(50, 300)
    _, mean, rstd = check_forward(rows, w, b)
    check_backward(rows, w, mean, rstd, g.expand(50, 300))


def test_other_streams():
    x, w, b, g = make(90, 520, torch.float16, 10)
    y, z = torch.empty_like(x), torch.empty_like(x)
    assert F.layer_norm_fprop(x, w, b, y, space(0, 90, 520)) == F.Success
    torch.cuda.synchronize()
    assert F.layer_norm_fprop(x, w, b, z, space(0, 90, 520), stream=torch.cuda.Stream()) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_offsets_past_32_bits():
    far = (1 << 32) + 8
    store = torch.zeros(3 * far, dtype=torch.bfloat16, device=dev())
    x, w, b, g = make(3, 520, torch.bfloat16, 11)
    for wide in (x, g):
        apart = store.as_strided((3, 520), (far, 1))
        apart.copy_(wide)
        _, mean, rstd = check_forward(apart, w, b)
        check_backward(apart, w, mean, rstd, g)
        y = torch.empty_like(x)
        assert F.layer_norm_fprop(apart, w, b, y, space(0, 3, 520)) == F.Success
        assert F.layer_norm_fprop(apart, w, b, apart, space(0, 3, 520)) == F.Success
        torch.cuda.synchronize()
        assert torch.equal(apart, y)
    del store


@pytest.mark.parametrize("m,n", [((1 << 21) + 5, 16), (3, (1 << 22) + 3)])
def test_many(m, n):
    x, w, b, g = make(m, n, torch.bfloat16, 12)
    _, mean, rstd = check_forward(x, w, b)
    check_backward(x, w, mean, rstd, g)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(64, 12801), (120, 8192), (33, 24000), (250, 4100), (260, 4100), (500, 3300), (520, 3300), (96, 16384)],
                         ids=str)
@pytest.mark.parametrize("form", ["rows", "pitch"])
def test_few_long_rows(shape, form, dtype):  # (whose columns are summed by themselves, or not quite)
    m, n = shape
    x, w, b, g = make(m, n, dtype, 8, form)
    _, mean, rstd = check_forward(x, w, b, form=form)
    gx, gw, gb = check_backward(x, w, mean, rstd, g, form=form)
    ws = space(1, m, n)
    w2, b2 = torch.full_like(gw, 7.0), torch.full_like(gb, 7.0)
    assert F.layer_norm_bprop(x, w, mean, rstd, g, None, w2, None, ws) == F.Success
    assert F.layer_norm_bprop(x, w, mean, rstd, g, None, None, b2, ws) == F.Success
    into = g.clone() if form == "rows" else g
    assert F.layer_norm_bprop(x, w, mean, rstd, into, into, gw.zero_(), gb.zero_(), ws) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(into, gx) and torch.equal(w2, gw) and torch.equal(b2, gb)

"""Group norm with an activation, forward and backward, against its plain form in 64 bits."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from operators_util import ACTS, NAMES, R, TYPES, act, norm, norm_grads, randn, rounded, within

pytestmark = pytest.mark.gpu

LAYOUTS = ["last", "planes", "crop", "slice", "turned"]


def images(values, dtype, layout):
    """values [B][C][H][W] on the GPU with the strides that `layout` names."""
    b, c, h, w = values.shape
    v = values.to(dtype).to(dev())
    if layout == "last":
        return v.permute(0, 2, 3, 1).contiguous().permute(0, 3, 1, 2)
    if layout == "planes":
        return v.contiguous()
    if layout == "crop":  # a window of larger planes: rows apart
        t = torch.zeros((b, c, h + 2, w + 3), dtype=dtype, device=dev())[:, :, 1:1 + h, 2:2 + w]
    elif layout == "slice":  # some channels of more, channels last, off any 16-byte boundary
        t = torch.zeros((b, h, w, c + 5), dtype=dtype, device=dev())[..., 3:3 + c].permute(0, 3, 1, 2)
    else:  # images innermost
        t = torch.zeros((c, w, h, b), dtype=dtype, device=dev()).permute(3, 0, 2, 1)
    return t.copy_(v)


def space(pass_, x, groups):
    return torch.empty(F.group_norm_workspace(pass_, x, groups), dtype=torch.uint8, device=dev())


def make(shape, groups, dtype, layout, seed, params=torch.float32):
    gen = torch.Generator().manual_seed(seed)
    b, c, h, w = shape
    x = randn(gen, b, c, h, w) * (0.5 + randn(gen, 1, c, 1, 1).abs()) + randn(gen, 1, c, 1, 1, std=0.7)
    weight, bias = randn(gen, c, std=0.3, mean=1.0), randn(gen, c, std=0.3)
    gy = randn(gen, b, c, h, w, std=0.1)
    return (images(x, dtype, layout), weight.to(params).to(dev()), bias.to(params).to(dev()), images(gy, dtype, layout))


def check_forward(x, weight, bias, groups, name, layout, eps=1e-5, out=None):
    y = out if out is not None else images(torch.full(x.shape, 7.0, dtype=torch.float64), x.dtype, layout)
    mean, rstd = (torch.full((x.shape[0], groups), 7.0, device=dev()) for _ in range(2))
    want, wm, wr, bound = norm(x, weight, bias, groups, eps, name)
    assert F.group_norm_fprop(x, weight, bias, y, groups, space(0, x, groups), activation=name, eps=eps, mean=mean,
                              rstd=rstd) == F.Success
    torch.cuda.synchronize()
    within(y, want, rounded(want, x.dtype) + bound)
    within(mean, wm, 4 * R * wm.abs() + 1e-12)
    within(rstd, wr, 8 * R * wr)
    return mean, rstd


def check_backward(x, weight, bias, gy, mean, rstd, groups, name, layout, params=torch.float32):
    gx = images(torch.full(x.shape, 7.0, dtype=torch.float64), x.dtype, layout)
    c = x.shape[1]
    gw, gb = (torch.full((c,), 7.0, dtype=params, device=dev()) for _ in range(2))
    (wx, bx), (ww, bw), (wb, bb) = norm_grads(x, weight, bias, mean, rstd, gy, groups, name)
    assert F.group_norm_bprop(x, weight, bias, mean, rstd, gy, gx, gw, gb, groups, space(1, x, groups),
                              activation=name) == F.Success
    torch.cuda.synchronize()
    within(gx, wx, rounded(wx, x.dtype) + bx)
    within(gw, ww, rounded(ww, params) + bw)
    within(gb, wb, rounded(wb, params) + bb)
    return gx, gw, gb


# (B, C, H, W, groups): one value a group, one pixel, odd planes, groups of six channels in words of eight and four, one
# group of all, every channel its own, groups wider than a workgroup, images larger than one
SHAPES = [(1, 1, 1, 1, 1), (2, 8, 1, 1, 2), (3, 12, 1, 7, 3), (2, 64, 27, 27, 8), (4, 192, 23, 23, 32), (2, 48, 9, 11, 8),
          (1, 32, 64, 64, 1), (2, 30, 5, 5, 30), (1, 4100, 3, 2, 1), (2, 40, 33, 31, 4), (1, 16, 150, 131, 2),
          (70, 24, 4, 4, 4)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", LAYOUTS)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_forward_and_backward(shape, layout, dtype):
    groups = shape[4]
    name = ACTS[(shape[1] + LAYOUTS.index(layout)) % 4]
    x, weight, bias, gy = make(shape[:4], groups, dtype, layout, 1)
    mean, rstd = check_forward(x, weight, bias, groups, name, layout)
    check_backward(x, weight, bias, gy, mean, rstd, groups, name, layout)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", ["last", "planes"])
@pytest.mark.parametrize("shape", [(2, 32, 12, 13, 4), (2, 32, 140, 140, 4)], ids=str)
def test_activations(shape, layout, dtype, name):
    x, weight, bias, gy = make(shape[:4], shape[4], dtype, layout, 2, params=dtype)
    mean, rstd = check_forward(x, weight, bias, shape[4], name, layout)
    check_backward(x, weight, bias, gy, mean, rstd, shape[4], name, layout, params=dtype)


@pytest.mark.parametrize("shape", [(2, 24, 10, 10, 4), (2, 24, 200, 190, 4)], ids=str)
@pytest.mark.parametrize("layout", ["last", "planes"])
def test_without_parameters_and_in_place(layout, shape):
    x, _, _, gy = make(shape[:4], shape[4], torch.float32, layout, 3)
    mean, rstd = check_forward(x.clone(memory_format=torch.preserve_format), None, None, shape[4], "silu", layout)
    check_backward(x, None, None, gy, mean, rstd, shape[4], "silu", layout)
    want, _, _, bound = norm(x, None, None, shape[4], 1e-5, "gelu")
    assert F.group_norm_fprop(x, None, None, x, shape[4], space(0, x, shape[4]), activation="gelu") == F.Success
    within(x, want, rounded(want, x.dtype) + bound)
    # gradInput in the place of gradOutput, without the parameters' gradients
    (wx, bx), _, _ = norm_grads(x, None, None, mean, rstd, gy, shape[4], "silu")
    assert F.group_norm_bprop(x, None, None, mean, rstd, gy, gy, None, None, shape[4], space(1, x, shape[4]),
                              activation="silu") == F.Success
    within(gy, wx, rounded(wx, x.dtype) + bx)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(3, 2602, 3, 5, 2), (2, 96, 70, 71, 48), (3, 130, 80, 33, 130), (1, 512, 40, 40, 64)], ids=str)
@pytest.mark.parametrize("layout", ["last", "slice"])
def test_many_channels_and_many_groups(layout, shape, dtype):
    """Groups wider than a row of lanes, several of them and images; and bands of 2, 1 and 8 channels to a group."""
    x, weight, bias, gy = make(shape[:4], shape[4], dtype, layout, 9)
    mean, rstd = check_forward(x, weight, bias, shape[4], "silu", layout)
    check_backward(x, weight, bias, gy, mean, rstd, shape[4], "silu", layout)


@pytest.mark.parametrize("layout", ["last", "planes"])
@pytest.mark.parametrize("side", [16, 160])
def test_variance_far_below_the_squared_mean(layout, side):
    """Means of 1000 deviations: a difference of fp32 sums would leave nothing of the variance.  And a corner far
    from everything else."""
    gen = torch.Generator().manual_seed(4)
    v = randn(gen, 2, 16, side, side, std=0.01, mean=10.0)
    v[1, :, 0, 0] = 0.0
    x = images(v, torch.float32, layout)
    check_forward(x, None, None, 4, "none", layout)


@pytest.mark.parametrize("layout", ["last", "planes"])
@pytest.mark.parametrize("side", [4, 180])
def test_constant_groups_and_values_that_are_not_finite(layout, side):
    gen = torch.Generator().manual_seed(5)
    v = randn(gen, 4, 16, side, side)
    v[0] = 3.0                       # no variance: the bias's activation
    v[1, 3, 0, 0] = float("nan")     # reaches its own group of its own image
    v[2, 9, -1, -1] = float("inf")
    x = images(v, torch.float32, layout)
    bias = torch.randn(16, generator=gen).to(dev())
    y = torch.empty_like(x)
    assert F.group_norm_fprop(x, None, bias, y, 4, space(0, x, 4), activation="silu") == F.Success
    want, _, _, bound = norm(x, None, bias, 4, 1e-5, "silu")
    got = y.cpu().double()
    within(got[0], want[0], rounded(want[0], x.dtype) + bound[0])
    within(got[3], want[3], rounded(want[3], x.dtype) + bound[3])
    for image, group in ((1, 0), (2, 2)):
        for g in range(4):
            part = slice(4 * g, 4 * g + 4)
            if g == group:
                assert bool(torch.isnan(got[image, part]).all())
            else:
                within(got[image, part], want[image, part], rounded(want[image, part], x.dtype) + bound[image, part])


@pytest.mark.parametrize("layout", ["last", "planes"])
@pytest.mark.parametrize("side", [6, 170])
def test_gradients_are_differences(layout, side):
    """The sum of r * output, at x + h d and x - h d."""
    gen = torch.Generator().manual_seed(6)
    shape, groups, h = (2, 12, side, side), 3, 1e-2
    v, d, r = (randn(gen, *shape) for _ in range(3))
    weight, bias = randn(gen, 12, mean=1.0), randn(gen, 12)
    dw, db = randn(gen, 12), randn(gen, 12)
    to = lambda t: images(t, torch.float32, layout) if t.dim() == 4 else t.float().to(dev())  # noqa: E731

    def loss(s):
        x, w, b = to(v + s * d), to(weight + s * dw), to(bias + s * db)
        y, mean, rstd = torch.empty_like(x), *(torch.empty((2, groups), device=dev()) for _ in range(2))
        assert F.group_norm_fprop(x, w, b, y, groups, space(0, x, groups), activation="silu", mean=mean,
                                  rstd=rstd) == F.Success
        return float((y.double().cpu() * r).sum()), (x, w, b, mean, rstd)

    _, (x, w, b, mean, rstd) = loss(0.0)
    gx, gw, gb = torch.empty_like(x), torch.empty_like(w), torch.empty_like(b)
    assert F.group_norm_bprop(x, w, b, mean, rstd, to(r), gx, gw, gb, groups, space(1, x, groups),
                              activation="silu") == F.Success
    slope = sum(float((g.double().cpu() * e).sum()) for g, e in ((gx, d), (gw, dw), (gb, db)))
    # what the difference leaves out is h^2 / 6 times a third derivative, of the sum's size sqrt(n) times about 10
    # in products of normal numbers; fp32 results add 2^-24 sqrt(n) / h
    n = v.numel()
    allowed = (h * h / 6 * 40 + 8 * R / h) * n ** 0.5
    assert abs((loss(h)[0] - loss(-h)[0]) / (2 * h) - slope) <= allowed


@pytest.mark.parametrize("layout", ["last", "planes"])
def test_empty_and_partial_calls(layout):
    x = torch.empty((0, 8, 4, 4), device=dev())
    stats = torch.empty((0, 2), device=dev())
    gw, gb = torch.full((8,), 7.0, device=dev()), torch.full((8,), 7.0, device=dev())
    assert F.group_norm_fprop(x, None, None, x, 2, None) == F.Success
    assert F.group_norm_bprop(x, None, None, stats, stats, x, x, gw, gb, 2, None) == F.Success
    assert not bool(gw.any()) and not bool(gb.any())  # sums over no images
    x, weight, bias, gy = make((2, 8, 30, 30), 2, torch.float32, layout, 7)
    mean, rstd = check_forward(x, weight, bias, 2, "silu", layout)
    gx, gw, gb = check_backward(x, weight, bias, gy, mean, rstd, 2, "silu", layout)
    only = [torch.full_like(t, 7.0) for t in (gx, gw, gb)]
    for i in range(3):
        args = [t if i == k else None for k, t in enumerate(only)]
        assert F.group_norm_bprop(x, weight, bias, mean, rstd, gy, *args, 2, space(1, x, 2), activation="silu") == F.Success
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(only, (gx, gw, gb)))  # and reproducible


def test_other_streams_and_the_general_way():
    x, weight, bias, gy = make((3, 32, 40, 40), 4, torch.bfloat16, "last", 8)
    y, z = torch.empty_like(x), torch.empty_like(x)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    assert F.group_norm_fprop(x, weight, bias, y, 4, space(0, x, 4), activation="silu") == F.Success
    ws = space(0, x, 4)
    torch.cuda.synchronize()
    assert F.group_norm_fprop(x, weight, bias, z, 4, ws, activation="silu", stream=stream) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_offsets_past_32_bits():
    """Two images and the pixels of an image more than 2^32 elements apart."""
    far = (1 << 32) + 24
    store = torch.zeros(2 * far + 4096, dtype=torch.bfloat16, device=dev())
    x = store.as_strided((2, 8, 1, 2), (64, 1, 8, far))
    gen = torch.Generator().manual_seed(9)
    v = randn(gen, 2, 8, 1, 2)
    x.copy_(v.to(dev()))
    check_forward(x, None, None, 2, "silu", "planes")
    del store


def test_forward_of_more_lanes_than_a_launch_holds():
    """2^24 images whose channels a workgroup takes, and 2^26 groups of a wave each: both pass 2^32 lanes, and go in several
    launches.  Images do not depend on each other: they have the bits that they have in smaller batches."""
    for shape, groups, layout in (((1 << 24, 8, 1, 2), 1, "last"), ((1 << 26, 2, 1, 1), 1, "planes")):
        n = shape[0]
        gen = torch.Generator(device=dev()).manual_seed(12)
        dense = torch.randn(n, 1, 2, 8, generator=gen, device=dev(), dtype=torch.float16) if layout == "last" else None
        x = dense.permute(0, 3, 1, 2) if layout == "last" else torch.randn(shape, generator=gen, device=dev(), dtype=torch.float16)
        assert x.shape == shape
        w, b = torch.randn(shape[1], generator=gen, device=dev()), torch.randn(shape[1], generator=gen, device=dev())
        y, part = torch.full_like(x, 7.0), torch.empty_like(x[:n // 16])
        stats = [torch.full((n, groups), 7.0, device=dev()) for _ in range(2)]
        assert F.group_norm_fprop(x, w, b, y, groups, space(0, x, groups), activation="silu", mean=stats[0],
                                  rstd=stats[1]) == F.Success
        for k in range(16):
            inside = slice(k * (n // 16), (k + 1) * (n // 16))
            few = [torch.empty((n // 16, groups), device=dev()) for _ in range(2)]
            assert F.group_norm_fprop(x[inside], w, b, part, groups, space(0, part, groups), activation="silu", mean=few[0],
                                      rstd=few[1]) == F.Success
            assert torch.equal(y[inside], part)
            assert torch.equal(stats[0][inside], few[0]) and torch.equal(stats[1][inside], few[1])
        want, _, _, bound = norm(x[-3:], w, b, groups, 1e-5, "silu")
        within(y[-3:], want, rounded(want, x.dtype) + bound)


@pytest.mark.parametrize("layout", ["planes", "last"])
def test_backward_of_more_lanes_than_a_launch_holds(layout):
    """[65536][1024][1][1], a wave to each of 2^26 planes, and 2^24 images of two pixels, channels last: gradInput as in
    smaller batches, the parameters' gradients from 64-bit sums."""
    b, c, h, w, groups = (65536, 1024, 1, 1, 8) if layout == "planes" else (1 << 24, 4, 1, 2, 1)
    gen = torch.Generator(device=dev()).manual_seed(13)
    x, gy = (torch.randn(b, h, w, c, generator=gen, device=dev(), dtype=torch.float16).permute(0, 3, 1, 2) for _ in range(2))
    weight, bias = torch.randn(c, generator=gen, device=dev()), torch.randn(c, generator=gen, device=dev())
    mean, rstd = torch.randn(b, groups, generator=gen, device=dev()), torch.rand(b, groups, generator=gen, device=dev()) + 0.5
    gx, gw, gb = torch.full_like(x, 7.0), torch.full_like(weight, 7.0), torch.full_like(weight, 7.0)
    args = (weight, bias, mean, rstd)
    assert F.group_norm_bprop(x, *args, gy, gx, gw, gb, groups, space(1, x, groups)) == F.Success
    want, n = torch.zeros(4, c, dtype=torch.float64), b // 16
    for k in range(16):
        inside = slice(k * n, (k + 1) * n)
        part = torch.empty_like(x[inside])
        assert F.group_norm_bprop(x[inside], weight, bias, mean[inside], rstd[inside], gy[inside], part, None, None, groups,
                                  space(1, part, groups)) == F.Success
        assert torch.equal(gx[inside], part)
        each = lambda v: v[inside].repeat_interleave(c // groups, 1)[:, :, None, None].double()  # noqa: E731
        dz, xh = gy[inside].double(), (x[inside].double() - each(mean)) * each(rstd)
        size = gy[inside].double().abs() * (1 + (x[inside].double().abs() + each(mean).abs()) * each(rstd))
        for i, v in enumerate((dz, dz * xh, dz.abs(), size)):
            want[i] += v.sum((0, 2, 3)).cpu()
    # roundings of the terms, and of sums over b h w values in 32 bits: a random walk's share of their number
    chain = R * (16 + 2 * (b * h * w) ** 0.5)
    within(gb, want[0], rounded(want[0], torch.float32) + chain * want[2])
    within(gw, want[1], rounded(want[1], torch.float32) + chain * want[3])
    one = slice(b - 2, b)
    (wx, bx), _, _ = norm_grads(x[one], weight, bias, mean[one], rstd[one], gy[one], groups, "none")
    within(gx[one], wx, rounded(wx, x.dtype) + bx)


def test_the_largest_group():
    """2^31 - 2^16 values, one plane: places that run past its end stay 31-bit numbers.  The sums of its parts in 64 bits."""
    n, piece = (1 << 31) - (1 << 16), 1 << 26
    gen = torch.Generator(device=dev()).manual_seed(14)
    x, gy = (torch.randn(1, 1, 1, n, generator=gen, device=dev(), dtype=torch.float16) for _ in range(2))
    w, b = torch.tensor([1.25], device=dev()), torch.tensor([0.5], device=dev())
    y, mean, rstd = torch.full_like(x, 7.0), torch.empty((1, 1), device=dev()), torch.empty((1, 1), device=dev())
    assert F.group_norm_fprop(x, w, b, y, 1, space(0, x, 1), mean=mean, rstd=rstd) == F.Success
    pieces = [slice(k, min(k + piece, n)) for k in range(0, n, piece)]
    s1 = sum(x[0, 0, 0, p].double().sum() for p in pieces)
    s2 = sum(x[0, 0, 0, p].double().square().sum() for p in pieces)
    centre = s1 / n
    scale = 1 / torch.sqrt(s2 / n - centre ** 2 + 1e-5)
    within(mean, centre.view(1, 1).cpu(), 4 * R * centre.abs().cpu() + 1e-12)
    within(rstd, scale.view(1, 1).cpu(), 8 * R * scale.cpu())
    gx, gw, gb = gy.clone(), torch.empty_like(w), torch.empty_like(b)
    assert F.group_norm_bprop(x, w, b, mean, rstd, gx, gx, gw, gb, 1, space(1, x, 1)) == F.Success
    m, r = mean.double().item(), rstd.double().item()
    of = lambda p: (gy[0, 0, 0, p].double(), (x[0, 0, 0, p].double() - m) * r)  # noqa: E731
    total = [sum(float(v.sum()) for v in parts) for parts in zip(*((g, g * xh, g.abs(), (g * xh).abs()) for g, xh in map(of, pieces)))]
    chain = R * (16 + 2 * n ** 0.5)
    within(gb, torch.tensor([total[0]]), torch.tensor([chain * total[2]]))
    within(gw, torch.tensor([total[1]]), torch.tensor([chain * total[3]]))
    for p in (slice(0, 1 << 16), slice(n // 2, n // 2 + (1 << 16)), slice(n - (1 << 16), n)):
        g, xh = of(p)
        want = (x[0, 0, 0, p].double() - centre) * scale * 1.25 + 0.5
        within(y[0, 0, 0, p], want.cpu(), (rounded(want, x.dtype) + 16 * R * (want.abs() + 1)).cpu())
        want = r * 1.25 * (g - total[0] / n - xh * total[1] / n)
        within(gx[0, 0, 0, p], want.cpu(), (rounded(want, x.dtype) + 32 * R * (g.abs() + xh.abs() + 1)).cpu())


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", ["last", "planes", "slice"])
@pytest.mark.parametrize("side", [4, 180])
def test_constant_groups_are_the_biases_activation(layout, side, dtype):
    """x - mean is 0 whatever the values' size and the deviation's (1 / sqrt(eps) = 316 stands for it): nothing of the mean is
    left, in any type, on the path in registers and in two launches.  And both passes agree on what a ReLU lets through."""
    gen = torch.Generator().manual_seed(15)
    v = torch.empty(4, 16, side, side, dtype=torch.float64)
    for image, values in enumerate([(3.0, -7.0), (100.0, 0.25), (1000.0, 1008.0), (30000.0, -512.0)]):
        v[image, :8], v[image, 8:] = values
    x = images(v, dtype, layout)
    assert torch.equal(x.cpu().double(), v.to(dtype).double())
    weight, bias = randn(gen, 16, std=0.3, mean=1.0), randn(gen, 16, std=0.3)
    bias[::3] = 0.0
    weight, bias = weight.float().to(dev()), bias.float().to(dev())
    ones = images(torch.ones_like(v), dtype, layout)
    for name in ACTS:
        y, mean, rstd = torch.full_like(x, 7.0), torch.empty((4, 2), device=dev()), torch.empty((4, 2), device=dev())
        assert F.group_norm_fprop(x, weight, bias, y, 2, space(0, x, 2), activation=name, mean=mean, rstd=rstd) == F.Success
        z = bias.cpu().double()[None, :, None, None].expand_as(v)
        want = act(z, name)
        within(y, want, rounded(want, dtype) + 8 * R * (1 + z.abs()) * (name != "none"))
        if name == "relu":
            gx, gw, gb = torch.empty_like(x), torch.empty_like(weight), torch.empty_like(bias)
            assert F.group_norm_bprop(x, weight, bias, mean, rstd, ones, gx, gw, gb, 2, space(1, x, 2),
                                      activation=name) == F.Success
            assert torch.equal(gb.cpu(), (y > 0).sum((0, 2, 3)).float().cpu())


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("layout", ["last", "planes"])
@pytest.mark.parametrize("side", [12, 160])
def test_means_far_above_the_deviation(layout, side, dtype):
    """Values of a few neighbouring numbers of their type around 1000 and -30000: what the mean's own rounding costs, and no
    more than that, is allowed."""
    gen = torch.Generator().manual_seed(16)
    step = 1000 * torch.finfo(dtype).eps
    v = randn(gen, 2, 16, side, side, std=2 * step, mean=1000.0)
    v[1] = v[1] * -30
    x = images(v, dtype, layout)
    weight, bias = randn(gen, 16, std=0.3, mean=1.0).float().to(dev()), randn(gen, 16, std=0.3).float().to(dev())
    y = torch.full_like(x, 7.0)
    assert F.group_norm_fprop(x, weight, bias, y, 4, space(0, x, 4)) == F.Success
    want, mean, rstd, _ = norm(x, weight, bias, 4, 1e-5, "none")
    each = lambda t: t.repeat_interleave(4, 1)[:, :, None, None]  # noqa: E731
    w = weight.cpu().double()[None, :, None, None].abs()
    # half a unit of the mean, and three roundings of products and sums
    bound = R * each(mean.abs() * rstd) * w + 4 * R * ((want - bias.cpu().double()[None, :, None, None]).abs() + want.abs())
    within(y, want, rounded(want, dtype) + bound + 16 * R * want.abs())


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(2, 64, 27, 27, 8), (4, 192, 23, 23, 32), (3, 30, 5, 7, 5), (1, 16, 90, 91, 2), (2, 600, 6, 5, 2)],
                         ids=str)
@pytest.mark.parametrize("inner,outer", [("planes", "last"), ("last", "planes"), ("planes", "crop"), ("slice", "planes")])
def test_layouts_that_differ(inner, outer, shape, dtype):
    """What a convolution leaves as planes and a linear layer takes as rows of channels, and other pairs: the output and its
    gradient in one layout, the input and its gradient in another; then each gradient in the other's."""
    groups = shape[4]
    x, weight, bias, gy = make(shape[:4], groups, dtype, inner, 17)
    gy = images(gy.cpu().double(), dtype, outer)
    y = images(torch.full(x.shape, 7.0, dtype=torch.float64), dtype, outer)
    mean, rstd = check_forward(x, weight, bias, groups, "silu", outer, out=y)
    check_backward(x, weight, bias, gy, mean, rstd, groups, "silu", inner)
    check_backward(x, weight, bias, images(gy.cpu().double(), dtype, inner), mean, rstd, groups, "silu", outer)

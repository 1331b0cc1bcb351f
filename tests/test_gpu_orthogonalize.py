"""Newton-Schulz products against the formula in 64 bits."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import QUINTIC, TINY, U, orthogonal, orthogonal_bound
from operators_util import NAMES, TYPES, randn

pytestmark = pytest.mark.gpu


def stored(values, dtype, form="rows"):
    b, r, c = values.shape
    v = values.to(dtype).to(dev())
    if form == "rows":
        return v
    if form == "cols":  # rows contiguous
        return v.transpose(1, 2).contiguous().transpose(1, 2)
    if form == "pitch":
        t = torch.zeros((b, r + 2, c + 7), dtype=dtype, device=dev())[:, 1:1 + r, 3:3 + c]
    else:  # the batch innermost
        t = torch.zeros((r, c, b), dtype=dtype, device=dev()).permute(2, 0, 1)
    return t.copy_(v)


def gradient(gen, b, r, c):
    k = max(1, min(r, c) // 8)
    return (randn(gen, b, r, k) @ randn(gen, b, k, c) * (0.3 / k ** 0.5) + randn(gen, b, r, c, std=0.1)) * 1e-2


def space(b, r, c):
    return torch.empty(F.orthogonalize_workspace(b, r, c), dtype=torch.uint8, device=dev())


def check(g, steps=5, coefficients=QUINTIC, eps=1e-7, scale=1.0, form="rows"):
    flat = g.dim() == 2
    b, r, c = (1, *g.shape) if flat else g.shape
    y = stored(torch.full((b, r, c), 7.0, dtype=torch.float64), g.dtype, form)
    y = y[0] if flat else y
    assert F.orthogonalize(g, y, space(b, r, c), steps=steps, coefficients=coefficients, eps=eps, scale=scale) == F.Success
    torch.cuda.synchronize()
    triples = [coefficients] * steps if not hasattr(coefficients[0], "__len__") else coefficients
    want, norms, most = orthogonal_bound(g[None] if flat else g, triples, eps, scale)
    off = (y[None] if flat else y).cpu().double() - want
    assert bool(torch.isfinite(off).all())
    half = U[g.dtype] * want.abs() + TINY[g.dtype]
    far = off.square().sum((1, 2)).sqrt()
    allowed = norms + half.square().sum((1, 2)).sqrt()
    assert bool((far <= allowed).all()), "off by %.2e of %.2e allowed" % (float((far / allowed).max()), 1.0)
    assert bool((off.abs() <= half + 2 * most[:, None, None]).all())
    return y


SHAPES = [(1, 1), (1, 7), (7, 1), (2, 2), (3, 50), (31, 31), (32, 32), (33, 32), (32, 33), (40, 200), (64, 64), (65, 64), (63, 129),
          (128, 128), (129, 130), (100, 1000), (1000, 100), (192, 1600), (257, 256), (300, 517), (640, 512), (17, 4100)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matrices(shape, dtype):
    gen = torch.Generator().manual_seed(1)
    check(gradient(gen, 1, *shape)[0].to(dtype).to(dev()))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("form", ["rows", "cols", "pitch", "inner"])
@pytest.mark.parametrize("shape", [(3, 20, 37), (5, 81, 40), (2, 130, 131), (40, 9, 9), (3, 200, 70)], ids=str)
def test_batches_and_strides(shape, form, dtype):
    gen = torch.Generator().manual_seed(2)
    g = gradient(gen, *shape) * torch.exp(randn(gen, shape[0], 1, 1))  # every matrix of its own size
    check(stored(g, dtype, form), form=form)


@pytest.mark.parametrize("shape", [(1280, 2100), (500, 2100), (2100, 700)], ids=str)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=NAMES.get)
def test_large(shape, dtype):
    gen = torch.Generator().manual_seed(3)
    check(gradient(gen, 1, *shape)[0].to(dtype).to(dev()))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("noise", [1e-1, 1e-2, 1e-4])
@pytest.mark.parametrize("shape", [(90, 100), (100, 700), (640, 96)], ids=str)
def test_few_strong_directions(shape, noise, dtype):
    """One direction over noise: small singular values that the first steps multiply by 3.4 each, and what rounding put beside
    them.  The result stays within a rounding of bfloat16 (2.3e-3 of its norm on average) of the formula."""
    gen = torch.Generator().manual_seed(11)
    g = (randn(gen, shape[0], 1) @ randn(gen, 1, shape[1]) + noise * randn(gen, *shape)).to(dtype).to(dev())
    y = check(g).cpu().double()
    want = orthogonal(g[None], [QUINTIC] * 5, 1e-7, 1.0)[0]
    assert float((y - want).norm() / want.norm()) < {torch.float32: 2e-4, torch.float16: 5e-4, torch.bfloat16: 2.3e-3}[dtype]


@pytest.mark.parametrize("batch", [1, 3])
@pytest.mark.parametrize("steps", [1, 2, 3, 7])
def test_steps_of_long_matrices(steps, batch):
    gen = torch.Generator().manual_seed(12)
    g = gradient(gen, batch, 64, 1000).to(torch.bfloat16).to(dev())
    check(g, steps=steps)
    check(g.transpose(1, 2).contiguous(), steps=steps, scale=0.5)
    check(g, steps=steps, coefficients=(1.5, -0.5, 0.0))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [(48, 60), (150, 140)], ids=str)
def test_steps_coefficients_and_scale(shape, dtype):
    gen = torch.Generator().manual_seed(4)
    g = gradient(gen, 1, *shape)[0].to(dtype).to(dev())
    check(g, steps=1)
    check(g, steps=2, coefficients=(1.5, -0.5, 0.0))
    check(g, steps=10, coefficients=(1.5, -0.5, 0.0), scale=-0.25)
    check(g, steps=3, coefficients=[(2.0, -1.5, 0.5), (1.875, -1.25, 0.375), (3.0, -3.0, 1.0)], scale=3.0)
    check(g, steps=1, coefficients=(0.0, 0.0, 1.0))
    check(g, steps=6, eps=0.0)
    check(g, eps=0.1)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_sizes_of_values(dtype):
    """The norm is taken out whatever it is: squares of float32 values pass its range, or vanish in it."""
    gen = torch.Generator().manual_seed(5)
    g = gradient(gen, 1, 50, 70)[0]
    g = g / g.abs().max()
    for scale in {torch.float32: (1e38, 1e-30, 1e-40), torch.float16: (6e4, 1e-4), torch.bfloat16: (1e38, 1e-30)}[dtype]:
        check((g * scale).to(dtype).to(dev()), eps=0.0)


@pytest.mark.parametrize("shape", [(20, 40), (200, 130), (300, 700)], ids=str)
def test_nothing_and_what_is_not_finite(shape):
    b = 4
    gen = torch.Generator().manual_seed(6)
    g = gradient(gen, b, *shape)
    g[1] = 0
    g[2, 3, 7] = float("nan")
    g[3, shape[0] - 1, 0] = float("inf")
    g = g.float().to(dev())
    y = torch.full_like(g, 7.0)
    assert F.orthogonalize(g, y, space(b, *shape)) == F.Success
    torch.cuda.synchronize()
    assert bool(torch.isfinite(y[0]).all()) and not bool(y[1].any())
    assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(y[3]).all())
    check(g[0])


def test_one_singular_value():
    """A matrix of rank one keeps its direction: the polynomials of 1 after each other."""
    gen = torch.Generator().manual_seed(7)
    u, v = randn(gen, 90, 1), randn(gen, 1, 150)
    g = (u @ v).float().to(dev())
    check(g)
    s = 1.0
    for _ in range(5):
        s = QUINTIC[0] * s + QUINTIC[1] * s ** 3 + QUINTIC[2] * s ** 5
    want = orthogonal(g[None], [QUINTIC] * 5, 1e-7, 1.0)[0]
    assert abs(float(torch.linalg.matrix_norm(want, 2)) - s) < 1e-3  # (the polynomial's own slope at 1 is 0.7 to 3 a step)


@pytest.mark.parametrize("shape", [(96, 160), (160, 96)], ids=str)
def test_singular_values_come_near_one(shape):
    gen = torch.Generator().manual_seed(8)
    q, _ = torch.linalg.qr(randn(gen, 160, 96))
    r, _ = torch.linalg.qr(randn(gen, 96, 96))
    s = torch.logspace(0, -1.5, 96, dtype=torch.float64)
    g = q @ torch.diag(s) @ r
    g = (g if shape[0] == 160 else g.t()).float().to(dev())
    y = check(g)
    found = torch.linalg.svdvals(y.cpu().double())
    # (|g| is 2.8 times its largest, so they start from 0.0113 to 0.36: inside what five steps bring to 0.68 ... 1.21)
    assert 0.67 < float(found.min()) and float(found.max()) < 1.22


def test_reproducible_and_other_streams():
    gen = torch.Generator().manual_seed(9)
    g = gradient(gen, 2, 200, 333).to(torch.bfloat16).to(dev())
    y, z, ws = torch.empty_like(g), torch.empty_like(g), space(2, 200, 333)
    assert F.orthogonalize(g, y, ws) == F.Success
    torch.cuda.synchronize()
    ws.fill_(255)
    torch.cuda.synchronize()
    assert F.orthogonalize(g, z, ws, stream=torch.cuda.Stream()) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_offsets_past_32_bits():
    gen = torch.Generator().manual_seed(10)
    far = (1 << 32) + 8
    store = torch.zeros(3 * far, dtype=torch.bfloat16, device=dev())
    g = gradient(gen, 3, 40, 50).to(torch.bfloat16).to(dev())
    apart = store.as_strided((3, 40, 50), (far, 50, 1))
    apart.copy_(g)
    want = check(apart)
    assert F.orthogonalize(g, apart, space(3, 40, 50)) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(apart, want)
    apart = store.as_strided((3, 50), (far, 1))
    apart.copy_(g[0, :3])
    check(apart)
    del store


def test_nothing():
    d = dev()
    for shape in ((0, 5), (5, 0), (0, 3, 4), (2, 0, 4)):
        t = torch.empty(shape, device=d)
        assert F.orthogonalize(t, t, None) == F.Success

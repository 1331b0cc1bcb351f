"""Newton-Schulz products in every kernel that a plan may choose, on sizes that end inside tiles and words: against the formula in
64 bits, computed on the GPU."""
import math

import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import QUINTIC
from operators_util import NAMES, TINY, TYPES, U
from plan_cases import PAIRS

pytestmark = pytest.mark.gpu


def formula(g, steps, moved=lambda v, k: v):
    x = g.double()
    turn = x.shape[1] > x.shape[2]
    x = (x.transpose(1, 2) if turn else x).contiguous()
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + 1e-7)
    p, q = x.shape[1:]
    a, b, c = QUINTIC
    for i in range(steps):
        x = moved(x, 1 if i == 0 else p)
        gram = moved(x @ x.transpose(1, 2).contiguous(), q)
        poly = moved(b * gram + c * (gram @ gram), p)
        x = a * x + poly @ x
    x = moved(x, p)
    return x.transpose(1, 2) if turn else x


def bound(g, steps):
    """The formula, and how far 22 bits of every value between the products and 32-bit sums of them may leave a result off, as a norm
    and at one place: every such value moved by a random part of its rounding, four times, three times the largest (of the many
    results of these sizes; layers_util.orthogonal_bound has the terms)."""
    gen = torch.Generator(device=dev()).manual_seed(1)

    def moved(v, k):
        part = lambda: torch.rand(v.shape, generator=gen, dtype=torch.float64, device=v.device) * 2 - 1  # noqa: E731
        size = v.square().mean((1, 2), keepdim=True).sqrt()
        return v + part() * (2.0 ** -22 * v.abs() + 2.0 ** -35) + part() * 2.0 ** -24 * math.sqrt(k) * size

    want = formula(g, steps)
    offs = [formula(g, steps, moved) - want for _ in range(4)]
    norms = torch.stack([o.square().sum((1, 2)).sqrt() for o in offs]).amax(0)
    return want, 3 * norms, 3 * torch.stack([o.abs().amax((1, 2)) for o in offs]).amax(0)


def check(g, y, steps=5):
    b, r, c = g.shape
    ws = torch.empty(F.orthogonalize_workspace(b, r, c), dtype=torch.uint8, device=dev())
    assert F.orthogonalize(g, y, ws, steps=steps) == F.Success
    torch.cuda.synchronize()
    want, norms, most = bound(g, steps)
    off = y.double() - want
    assert bool(torch.isfinite(off).all())
    half = U[g.dtype] * want.abs() + TINY[g.dtype]
    far, allowed = off.square().sum((1, 2)).sqrt(), norms + half.square().sum((1, 2)).sqrt()
    assert bool((far <= allowed).all()), "off by %.2e of what is allowed" % float((far / allowed).max())
    assert bool((off.abs() <= half + 2 * most[:, None, None]).all())


def gradient(b, r, c, dtype):
    gen = torch.Generator(device=dev()).manual_seed(2)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev())  # noqa: E731
    k = max(1, min(r, c) // 8)
    return ((randn(b, r, k) @ randn(b, k, c) * (0.3 / k ** 0.5) + 0.1 * randn(b, r, c)) * 1e-2).to(dtype)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("shape", [s for s, _ in PAIRS], ids=str)
def test_matrices(shape, dtype):
    b, r, c = shape
    g = gradient(b, r, c, dtype)
    check(g, torch.full_like(g, 7.0))
    # one step, of single pieces where values have 16 bits, straight to the result; and the other way round, into rows with gaps
    y = torch.full((b, c, r + 5), 7.0, dtype=dtype, device=dev())
    check(g.transpose(1, 2), y[:, :, 2:r + 2], steps=1)
    assert bool((y[:, :, :2] == 7).all()) and bool((y[:, :, r + 2:] == 7).all())
    # rows as columns, and every second element
    check(g, torch.full((b, c, r), 7.0, dtype=dtype, device=dev()).transpose(1, 2), steps=2)
    check(g, torch.full((b, r, 2 * c), 7.0, dtype=dtype, device=dev())[:, :, ::2], steps=2)

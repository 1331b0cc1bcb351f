"""Newton-Schulz products of long bfloat16 matrices: as near to the formula as those of every other shape, and no coefficients
that the entry point takes leave the range of what is held between products."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import QUINTIC, U, orthogonal_bound
from operators_util import randn

pytestmark = pytest.mark.gpu


def result(g, **more):
    y = torch.empty_like(g)
    ws = torch.empty(F.orthogonalize_workspace(1, *g.shape), dtype=torch.uint8, device=dev())
    assert F.orthogonalize(g, y, ws, **more) == F.Success
    torch.cuda.synchronize()
    return y.cpu()


def check(g, triples):
    """Results are the formula's, rounded, but where an error e before the rounding moves one past the middle between two
    neighbours `step` apart: a share |e| / step of places, each `step` off.  So the squares of what differs from the rounded
    formula add up to the sum of |e| step, at most the norms of e and of the steps multiplied.  e: what 22 bits of the values
    between the products and 32-bit sums of them leave, whatever the matrix's shape (that of a float32 matrix)."""
    y = result(g, steps=len(triples), coefficients=triples).double()
    want, norms, _ = orthogonal_bound(g.float()[None], triples, 1e-7, 1.0)
    want, near = want[0], want[0].to(torch.bfloat16).double()
    step = 2.0 ** (torch.frexp(want)[1].double() - 8)  # eight bits of a number in [0.5, 1) times 2^e
    off = float((y - near).square().sum())
    allowed = float(norms) * float(step.norm())
    assert off <= allowed, "%.2e of the norm beside the rounded formula, %.2e allowed" % tuple(
        v ** 0.5 / float(want.norm()) for v in (off, allowed))


@pytest.mark.parametrize("shape", [(64, 1000), (100, 700), (1000, 100), (260, 1100), (2100, 700)], ids=str)
@pytest.mark.parametrize("noise", [None, 1e-1, 1e-2, 1e-3])
def test_long_matrices(shape, noise):
    gen = torch.Generator().manual_seed(1)
    r, c = shape
    if noise is None:  # many strong directions
        k = min(r, c) // 8
        g = randn(gen, r, k) @ randn(gen, k, c) * (0.3 / k ** 0.5) + randn(gen, r, c, std=0.1)
    else:
        g = randn(gen, r, 1) @ randn(gen, 1, c) + noise * randn(gen, r, c)
    g = g.to(torch.bfloat16).to(dev())
    check(g, [QUINTIC] * 5)
    check(g, [(1.5, -0.5, 0.0)] * 4)
    check(g, [(2.0, -1.5, 0.5), QUINTIC, (1.875, -1.25, 0.375)])


@pytest.mark.parametrize("shape", [(100, 1000), (1000, 100), (64, 1000)], ids=str)
@pytest.mark.parametrize("rank", [None, 1, 20])
def test_a_step_that_shrinks_after_steps_that_grew(shape, rank):
    """The six first steps multiply a small singular value by 1670, the last one by 0.2; rows that fill a matrix up, and
    matrices without full rank, have singular values of 0."""
    gen = torch.Generator().manual_seed(2)
    r, c = shape
    g = randn(gen, r, c) if rank is None else randn(gen, r, rank) @ randn(gen, rank, c)
    g = g.to(torch.bfloat16).to(dev())
    triples = [QUINTIC] * 6 + [(0.2, 0.0, 0.0)]
    y = result(g, steps=7, coefficients=triples).double()
    assert bool(torch.isfinite(y).all())
    want, norms, _ = orthogonal_bound(g.float()[None], triples, 1e-7, 1.0)
    assert float((y - want[0]).norm()) <= float(norms) + U[torch.bfloat16] * float(want.norm())


def test_more_small_matrices_than_a_launch_holds():
    gen = torch.Generator().manual_seed(3)
    few, many = 1031, (1 << 22) + 77
    base = randn(gen, few, 2, 3).float().to(dev())
    want = torch.empty_like(base)
    assert F.orthogonalize(base, want, torch.empty(F.orthogonalize_workspace(few, 2, 3), dtype=torch.uint8, device=dev())) == F.Success
    g = base[torch.arange(many, device=dev()) % few]
    y = torch.full_like(g, 7.0)
    assert F.orthogonalize(g, y, torch.empty(F.orthogonalize_workspace(many, 2, 3), dtype=torch.uint8, device=dev())) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, want[torch.arange(many, device=dev()) % few])

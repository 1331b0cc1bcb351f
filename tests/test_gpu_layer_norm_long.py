"""The parameters' gradients of layer norm over rows as long as they may be: more columns, and columns times rows, than a launch
holds lanes for.  All rows are the same one in memory, under statistics of their own."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import chain
from operators_util import R

pytestmark = pytest.mark.gpu


def check(m, n, step, want_bias=True):
    gen = torch.Generator(device=dev()).manual_seed(1)
    row = lambda: torch.randn(n * step, generator=gen, device=dev()).to(torch.bfloat16)  # noqa: E731
    x, g = (row().as_strided((m, n), (0, step)) for _ in range(2))
    mean, rstd = torch.randn(m, generator=gen, device=dev()), torch.rand(m, generator=gen, device=dev()) + 0.5
    gw = torch.full((n,), 7.0, device=dev())
    gb = torch.full((n,), 7.0, device=dev()) if want_bias else None
    ws = torch.empty(F.layer_norm_workspace(1, m, n), dtype=torch.uint8, device=dev())
    assert F.layer_norm_bprop(x, None, mean, rstd, g, None, gw, gb, ws) == F.Success
    torch.cuda.synchronize()
    x, g, mean, rstd = x[0].double(), g[0].double(), mean.double(), rstd.double()
    want = g * (x * rstd.sum() - (mean * rstd).sum())
    # each term's three roundings, of numbers up to (|x| + |mean|) rstd, and their sum's
    sizes = g.abs() * (x.abs() * rstd.sum() + (mean.abs() * rstd).sum())
    assert bool(((gw - want).abs() <= (chain(m) + 4 * R) * sizes).all())
    if want_bias:
        assert bool(((gb - m * g).abs() <= (chain(m) + R) * m * g.abs()).all())


@pytest.mark.parametrize("step", [1, 2], ids=["rows", "apart"])
def test_columns_times_rows_past_a_launch(step):
    check(256, (1 << 24) + 5, step)


@pytest.mark.parametrize("m", [7, 40])
def test_columns_past_a_launch_of_their_join(m):
    check(m, (1 << 25) + 9 if m > 32 else (1 << 28) + 9, 2, want_bias=m > 32)

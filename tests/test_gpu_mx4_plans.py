"""Products with 4-bit rows in every kernel that a plan may choose, on sizes that end inside tiles, steps and words: against the
definition in 64 bits."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from operators_util import ACTS, NAMES, TYPES, linear, randn, rounded, within
from layers_util import values_of
from plan_cases import MX4
from test_gpu_mx4 import check, matrix, quantize

pytestmark = pytest.mark.gpu

TILES = [c for c in MX4 if c[2].startswith("tiles")]
SOME = [c for c in TILES if c[0] in ((978, 417, 849), (1111, 1151, 1009), (1031, 333, 7183), (260, 4352, 1300), (264, 4352, 1304),
                                     (2156, 15582, 142))]


def name(c):
    return c[2].replace(" ", "-") + "-%d-%d-%d" % c[0]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("case", MX4, ids=name)
def test_products(case, dtype):
    shape, codes, _ = case
    check(*shape, dtype, ACTS[sum(shape) % 4], 3, codes)


@pytest.mark.parametrize("form", ["cols", "pitch", "apart"])
@pytest.mark.parametrize("case", SOME, ids=name)
def test_strides(case, form):
    shape, codes, _ = case
    check(*shape, torch.bfloat16 if form == "cols" else torch.float32, "silu", 4, codes, form=form, apart=3)


@pytest.mark.parametrize("case", SOME, ids=name)
def test_what_may_be_left_out(case):
    shape, codes, _ = case
    for i, (bias, residual) in enumerate(((False, False), (True, False), (False, True))):
        check(*shape, TYPES[i], ACTS[i + 1], 5, codes, bias=bias, residual=residual)


@pytest.mark.parametrize("case", SOME, ids=name)
def test_values_that_are_not_finite_stay_in_their_rows_and_columns(case):
    (m, k, n), codes, _ = case
    gen = torch.Generator().manual_seed(6)
    x, weight = randn(gen, m, k), randn(gen, n, k)
    x[m - 2, k - 1], x[130, 5] = float("nan"), float("inf")
    weight[n - 3, 0], weight[64, k - 1] = float("nan"), float("-inf")
    x, weight = matrix(x, torch.bfloat16), quantize(matrix(weight, torch.bfloat16))
    rows = quantize(x)
    ws = torch.empty(F.linear_mx4_workspace(m, k, n), dtype=torch.uint8, device=dev())
    y = torch.empty((m, n), device=dev(), dtype=torch.bfloat16)
    assert F.linear_mx4_fprop(rows[0] if codes else x, *weight, None, y, ws, inputScales=rows[1] if codes else None) == F.Success
    bad = torch.zeros((m, n), dtype=torch.bool, device=dev())
    bad[[m - 2, 130]] = True
    bad[:, [n - 3, 64]] = True
    assert torch.equal(torch.isnan(y), bad) and bool(torch.isfinite(y[~bad]).all())


@pytest.mark.parametrize("case", SOME, ids=name)
def test_residual_in_place_and_nothing_beside_the_results(case):
    (m, k, n), codes, _ = case
    gen = torch.Generator().manual_seed(7)
    x, weight = matrix(randn(gen, m, k), torch.bfloat16), quantize(matrix(randn(gen, n, k) * k ** -0.5, torch.bfloat16))
    rows = quantize(x)
    ws = torch.empty(F.linear_mx4_workspace(m, k, n), dtype=torch.uint8, device=dev())
    around = matrix(randn(gen, m + 2, n + 9), torch.bfloat16)
    kept, y = around.clone(), around[1:m + 1, 4:n + 4]
    assert F.linear_mx4_fprop(rows[0] if codes else x, *weight, None, y, ws, residual=y, inputScales=rows[1] if codes else None) == F.Success
    torch.cuda.synchronize()
    want, bound, _, _ = linear(values_of(*rows, k), values_of(*weight, k), None, kept[1:m + 1, 4:n + 4], "none")
    within(y, want, rounded(want, torch.bfloat16) + bound)
    y.copy_(kept[1:m + 1, 4:n + 4])
    assert torch.equal(around, kept)

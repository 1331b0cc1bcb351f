"""Rows in microscaled 4-bit floating point, and products with them, against the definitions in 64 bits."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import quantized, values_of
from operators_util import ACTS, NAMES, TYPES, linear, randn, rounded, within

pytestmark = pytest.mark.gpu


def matrix(values, dtype, form="rows"):
    r, c = values.shape
    v = values.to(dtype).to(dev())
    if form == "rows":
        return v
    if form == "cols":
        return v.t().contiguous().t()
    if form == "pitch":
        t = torch.zeros((r, c + 7), dtype=dtype, device=dev())[:, 3:3 + c]
    else:
        t = torch.zeros((3 * r, 2 * c), dtype=dtype, device=dev())[::3, ::2]
    return t.copy_(v)


def packed(rows, cols, apart=0):
    """Buffers full of something; apart: bytes between rows of scales, and sixteen times that between those of codes."""
    blocks = -(-cols // 32)
    return (torch.full((rows, 16 * (blocks + apart)), 0xA5, dtype=torch.uint8, device=dev())[:, :16 * blocks],
            torch.full((rows, blocks + apart), 0xA5, dtype=torch.uint8, device=dev())[:, :blocks])


def quantize(x, apart=0):
    codes, scales = packed(*x.shape, apart)
    assert F.mx4_quantize(x, codes, scales) == F.Success
    return codes, scales


def spread(gen, rows, cols):
    return randn(gen, rows, cols) * torch.exp(randn(gen, 1, cols))


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("form", ["rows", "cols", "pitch", "apart"])
@pytest.mark.parametrize("shape", [(1, 1), (1, 31), (3, 32), (2, 33), (70, 40), (9, 64), (130, 100), (5, 1151), (64, 256), (2, 8200)],
                         ids=str)
def test_quantize_and_read_back(shape, form, dtype):
    gen = torch.Generator().manual_seed(1)
    x = matrix(spread(gen, *shape), dtype, form)
    apart = 0 if form == "rows" else 3
    codes, scales = quantize(x, apart)
    torch.cuda.synchronize()
    want, wants = quantized(x)
    assert torch.equal(scales.cpu(), wants) and torch.equal(codes.cpu(), want)
    for kind in TYPES:
        y = matrix(torch.full(shape, 7.0, dtype=torch.float64), kind, form)
        assert F.mx4_dequantize(codes, scales, y) == F.Success
        torch.cuda.synchronize()
        assert torch.equal(y.cpu(), values_of(codes, scales, shape[1]).to(kind))


def test_every_code_scale_and_tie():
    """All sixteen values under every scale that reads back; values at, beside and between the places where codes change,
    with the largest of a block anywhere from 4 to just below 8 times its scale."""
    codes = torch.arange(256, dtype=torch.uint8).repeat(16, 1)  # rows of 16 blocks
    scales = torch.arange(256, dtype=torch.uint8).view(16, 16)
    y = torch.empty((16, 512), device=dev())
    assert F.mx4_dequantize(codes.to(dev()), scales.to(dev()), y) == F.Success
    want = values_of(codes, scales, 512)
    fine = torch.isfinite(want.float())
    assert torch.equal(y.cpu()[fine], want.float()[fine])
    assert torch.equal(torch.isnan(y.cpu()), torch.isnan(want))
    gen = torch.Generator().manual_seed(2)
    edges = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64)
    a = torch.cat([edges, edges * (1 + 2.0 ** -23), edges * (1 - 2.0 ** -23)])  # 24 of a block
    for exponent in (-140, -130, -127, -126, -125, -124, -60, -1, 0, 1, 60, 124, 125):
        most = 4 + 4 * torch.rand(40, 1, generator=gen, dtype=torch.float64)
        rest = randn(gen, 40, 7) * 0.5
        x = torch.cat([a.expand(40, 24), most, rest], 1) * 2.0 ** exponent
        sign = 1 - 2 * (torch.rand(40, 32, generator=gen) < 0.5).double()
        x = (x * sign).float()
        got = [t.cpu() for t in quantize(x.to(dev()))]
        want = quantized(x)
        assert torch.equal(got[1], want[1]) and torch.equal(got[0], want[0])


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_blocks_of_nothing_and_of_what_is_not_finite(dtype):
    x = torch.zeros((7, 96), dtype=torch.float64)
    x[1] = -0.0
    x[2, 40], x[3, 95], x[4, 0] = float("nan"), float("inf"), float("-inf")
    x[2:5] += 1.0
    tiny = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}[dtype]
    x[5, ::3] = tiny
    x[6, ::2] = -3 * tiny
    x = matrix(x, dtype)
    got, want = [t.cpu() for t in quantize(x)], quantized(x)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    y = torch.empty((7, 96), device=dev())
    assert F.mx4_dequantize(got[0].to(dev()), got[1].to(dev()), y) == F.Success
    bad = torch.isnan(y).view(7, 3, 32)
    assert bool((bad.all(-1) == bad.any(-1)).all())
    assert bad.any(-1).cpu().nonzero().tolist() == [[2, 1], [3, 2], [4, 0]]


def check(m, k, n, dtype, name, seed, ready=False, form="rows", bias=True, residual=True, apart=0):
    gen = torch.Generator().manual_seed(seed)
    x = matrix(spread(gen, m, k), dtype, "rows" if ready else form)
    wq = quantize(matrix(randn(gen, n, k) * k ** -0.5, dtype), apart)
    xq = quantize(x, apart)
    b = randn(gen, n, std=0.3).float().to(dev()) if bias else None
    r = matrix(randn(gen, m, n), dtype, form) if residual else None
    y = matrix(torch.full((m, n), 7.0, dtype=torch.float64), dtype, form)
    ws = torch.empty(F.linear_mx4_workspace(m, k, n), dtype=torch.uint8, device=dev())
    assert F.linear_mx4_fprop(xq[0] if ready else x, *wq, b, y, ws, activation=name, residual=r,
                              inputScales=xq[1] if ready else None) == F.Success
    torch.cuda.synchronize()
    want, bound, _, _ = linear(values_of(*xq, k), values_of(*wq, k), b, r, name)
    within(y, want, rounded(want, dtype) + bound)
    return y


# (M, K, N): single rows, columns and blocks; the sides of tiles and steps and one beyond; ragged ones; long sums
SHAPES = [(1, 1, 1), (1, 2048, 33), (1, 96, 1000), (2, 32, 64), (5, 333, 70), (16, 128, 48), (17, 40, 200), (33, 31, 1), (64, 64, 64),
          (65, 72, 130), (128, 256, 128), (129, 257, 127), (200, 520, 256), (300, 1151, 100), (257, 96, 520), (4, 4104, 16),
          (40, 16, 3000), (3000, 24, 40), (31, 9000, 65), (48, 511, 129), (100, 1151, 1000)]


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("ready", [False, True], ids=["values", "codes"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_products(shape, ready, dtype):
    check(*shape, dtype, ACTS[sum(shape) % 4], 3, ready)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("form", ["cols", "pitch", "apart"])
@pytest.mark.parametrize("shape", [(1, 72, 40), (3, 50, 67), (130, 300, 136), (70, 45, 33), (40, 700, 264)], ids=str)
def test_strides(shape, form, dtype):
    check(*shape, dtype, "silu", 4, form=form, apart=3)
    check(*shape, dtype, "silu", 4, form=form, apart=2, ready=True)


@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("m", [1, 12, 150, 1100])
def test_activations_and_what_may_be_left_out(m, name):
    for bias, residual in ((False, False), (True, False), (False, True)):
        check(m, 160, 264, torch.bfloat16, name, 5, bias=bias, residual=residual)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_large(dtype):
    """Whole tiles, long reductions, many tiles."""
    check(1536, 4096, 1280, dtype, "gelu", 6)


@pytest.mark.parametrize("m", [1, 16, 60, 600])
def test_residual_in_place_and_broadcast(m):
    gen = torch.Generator().manual_seed(7)
    x, r = matrix(randn(gen, m, 64), torch.bfloat16), matrix(randn(gen, m, 96), torch.bfloat16)
    w = quantize(matrix(randn(gen, 96, 64), torch.bfloat16))
    ws = torch.empty(F.linear_mx4_workspace(m, 64, 96), dtype=torch.uint8, device=dev())
    y = torch.empty_like(r)
    assert F.linear_mx4_fprop(x, *w, None, y, ws, residual=r) == F.Success
    assert F.linear_mx4_fprop(x, *w, None, r, ws, residual=r) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(r, y)
    row = x[:1].expand(m, 64)
    assert F.linear_mx4_fprop(row, *w, None, y, ws, residual=r[:1].expand(m, 96)) == F.Success
    want, bound, _, _ = linear(values_of(*quantize(row.contiguous()), 64), values_of(*w, 64), None, r[:1].expand(m, 96), "none")
    within(y, want, rounded(want, torch.bfloat16) + bound)


@pytest.mark.parametrize("m", [2, 40, 100, 700])
def test_values_that_are_not_finite_stay_in_their_rows(m):
    gen = torch.Generator().manual_seed(8)
    x = matrix(randn(gen, m, 300), torch.bfloat16)
    weight = matrix(randn(gen, 136, 300), torch.bfloat16)
    ws = torch.empty(F.linear_mx4_workspace(m, 300, 136), dtype=torch.uint8, device=dev())
    y = torch.empty((m, 136), dtype=torch.bfloat16, device=dev())
    others = torch.arange(m, device=dev()) != 1
    for at, value in ((5, "nan"), (299, "inf"), (31, "-inf")):
        bad = x.clone()
        bad[1, at] = float(value)
        assert F.linear_mx4_fprop(bad, *quantize(weight), None, y, ws) == F.Success
        assert bool(torch.isnan(y[1]).all()) and bool(torch.isfinite(y[others]).all())
    weight[7, 290] = float("nan")
    assert F.linear_mx4_fprop(x, *quantize(weight), None, y, ws) == F.Success
    columns = torch.arange(136, device=dev()) != 7
    assert bool(torch.isnan(y[:, 7]).all()) and bool(torch.isfinite(y[:, columns]).all())


def test_nothing_to_sum():
    d = dev()
    bias, r = torch.randn(8, device=d), torch.randn(3, 8, device=d)
    y = torch.full((3, 8), 7.0, device=d)
    empty = lambda rows: (torch.empty((rows, 0), dtype=torch.uint8, device=d),) * 2  # noqa: E731
    assert F.linear_mx4_fprop(torch.empty((3, 0), device=d), *empty(8), bias, y, None, residual=r) == F.Success
    assert torch.equal(y, bias + r)
    w = quantize(torch.randn(8, 40, device=d))
    assert F.linear_mx4_fprop(torch.empty((0, 40), device=d), *w, bias, torch.empty((0, 8), device=d), None) == F.Success
    assert F.mx4_quantize(torch.empty((0, 40), device=d), *packed(0, 40)) == F.Success
    assert F.mx4_quantize(torch.empty((4, 0), device=d), *empty(4)) == F.Success


def test_tails_and_gaps_stay_as_they_are():
    gen = torch.Generator().manual_seed(9)
    codes = torch.full((6, 16 * 5), 0x5A, dtype=torch.uint8, device=dev())
    scales = torch.full((6, 7), 0x5A, dtype=torch.uint8, device=dev())
    x = matrix(randn(gen, 5, 100), torch.float32)
    assert F.mx4_quantize(x, codes[:5, :64], scales[:5, :4]) == F.Success
    torch.cuda.synchronize()
    assert bool((codes[5] == 0x5A).all()) and bool((codes[:, 64:] == 0x5A).all())
    assert bool((scales[5] == 0x5A).all()) and bool((scales[:, 4:] == 0x5A).all())
    assert not bool(codes[:5, 50:64].any())  # 100 values end inside the last block
    y = torch.full((6, 103), 7.0, device=dev())
    assert F.mx4_dequantize(codes[:5, :64], scales[:5, :4], y[:5, :100]) == F.Success
    torch.cuda.synchronize()
    assert bool((y[5] == 7).all()) and bool((y[:, 100:] == 7).all())


def test_other_streams():
    gen = torch.Generator().manual_seed(10)
    x = matrix(randn(gen, 90, 640), torch.bfloat16)
    w = quantize(matrix(randn(gen, 72, 640), torch.bfloat16))
    ws = torch.empty(F.linear_mx4_workspace(90, 640, 72), dtype=torch.uint8, device=dev())
    y, z = (torch.empty((90, 72), dtype=torch.bfloat16, device=dev()) for _ in range(2))
    assert F.linear_mx4_fprop(x, *w, None, y, ws) == F.Success
    torch.cuda.synchronize()
    assert F.linear_mx4_fprop(x, *w, None, z, ws, stream=torch.cuda.Stream()) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_offsets_past_32_bits():
    gen = torch.Generator().manual_seed(11)
    far = 1 << 22  # bytes between rows; 1100 of them are over 2^32
    store = torch.zeros(1100 * far, dtype=torch.uint8, device=dev())
    values = randn(gen, 1100, 64).to(torch.bfloat16)
    x = store.view(torch.bfloat16).as_strided((1100, 64), (far // 2, 1))
    x.copy_(values.to(dev()))
    codes, scales = store.as_strided((1100, 32), (far, 1), 256), store.as_strided((1100, 2), (far, 1), 512)
    assert F.mx4_quantize(x, codes, scales) == F.Success
    torch.cuda.synchronize()
    want = quantized(values)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])
    y = store.view(torch.bfloat16).as_strided((1100, 64), (far // 2, 1), 512)
    assert F.mx4_dequantize(codes, scales, y) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y.cpu().double(), values_of(*want, 64))
    # as rows, and as the weight
    other = quantize(matrix(randn(gen, 40, 64), torch.bfloat16))
    ws = torch.empty(F.linear_mx4_workspace(1100, 64, 1100), dtype=torch.uint8, device=dev())
    for rows, weight in (((codes, scales), other), (other, (codes, scales))):
        out = torch.empty((rows[0].shape[0], weight[0].shape[0]), device=dev())
        assert F.linear_mx4_fprop(rows[0], *weight, None, out, ws, inputScales=rows[1]) == F.Success
        want, bound, _, _ = linear(values_of(*rows, 64), values_of(*weight, 64), None, None, "none")
        within(out, want, rounded(want, torch.float32) + bound)
    del store


def test_many_rows():
    gen = torch.Generator().manual_seed(12)
    check((1 << 21) + 3, 16, 16, torch.bfloat16, "relu", 12)
    x = matrix(randn(gen, (1 << 22) + 5, 20), torch.bfloat16)
    codes, scales = quantize(x)
    want = quantized(x)
    assert torch.equal(codes.cpu(), want[0]) and torch.equal(scales.cpu(), want[1])

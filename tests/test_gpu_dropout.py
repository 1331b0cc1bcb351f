"""Dropout of a counter-based generator against its plain form: the generator's published outputs, the same mask for
every layout and type, and the values."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from operators_util import NAMES, TYPES, dropout, halves, randn, rounded, within

pytestmark = pytest.mark.gpu


def check(x, residual, p, seed, offset, y):
    want, bound = dropout(x, residual, p, seed, offset)
    assert F.dropout_fprop(x, y, p, seed, offset, residual=residual) == F.Success
    torch.cuda.synchronize()
    within(y, want, rounded(torch.nan_to_num(want, posinf=0.0, neginf=0.0, nan=0.0), x.dtype) + bound)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("n", [1, 7, 8, 9, 2000, 2047, 2048, 2049, 70001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 1.0])
def test_lengths(n, p, dtype):
    gen = torch.Generator().manual_seed(n)
    x, r = (randn(gen, n).to(dtype).to(dev()) for _ in range(2))
    check(x, r, p, 0x1234567890ABCDEF, 77, torch.full_like(x, 7.0))
    check(x, None, p, 2 ** 64 - 1, 2 ** 64 - 1, torch.full_like(x, 7.0))
    g = torch.full_like(x, 7.0)
    assert F.dropout_bprop(x, g, p, 0x1234567890ABCDEF, 77) == F.Success
    check(x, None, p, 0x1234567890ABCDEF, 77, y := torch.empty_like(x))
    assert torch.equal(g, y)


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_the_mask_follows_the_logical_place_whatever_the_strides(dtype):
    gen = torch.Generator().manual_seed(1)
    v = randn(gen, 3, 5, 7, 2, 11).to(dtype).to(dev())
    base = torch.empty_like(v)
    check(v, None, 0.4, 5, 6, base)
    forms = [v.permute(4, 2, 0, 1, 3).contiguous().permute(2, 3, 1, 4, 0),
             torch.zeros((3, 5, 7, 2, 14), dtype=dtype, device=dev())[..., 1:12].copy_(v),
             torch.zeros((6, 5, 7, 2, 11), dtype=dtype, device=dev())[::2].copy_(v)]
    for x in forms:
        for y in (torch.empty_like(v), torch.empty_strided(x.shape, x.stride(), dtype=dtype, device=dev())):
            assert F.dropout_fprop(x, y, 0.4, 5, 6) == F.Success
            assert torch.equal(y, base)
            assert F.dropout_fprop(x, y, 0.4, 5, 6, residual=forms[1]) == F.Success
            check(v, v, 0.4, 5, 6, both := torch.empty_like(v))
            assert torch.equal(y, both)
    # one row for all: a residual and an input of stride 0
    row = v[:1, :1, :1, :1].expand_as(v)
    check(row, row, 0.4, 5, 6, torch.empty_like(v))


@pytest.mark.parametrize("rows,cols,pitch", [(1, 1, 1), (3, 5, 5), (9, 16, 24), (70, 33, 38), (64, 256, 261), (5, 4096, 4104)])
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_rows_apart(rows, cols, pitch, dtype):
    gen = torch.Generator().manual_seed(2)
    x, r = (randn(gen, rows, pitch).to(dtype).to(dev())[:, :cols] for _ in range(2))
    y = torch.full((rows, pitch), 7.0, dtype=dtype, device=dev())
    check(x, r, 0.25, 3, 4, y[:, :cols])
    assert bool((y[:, cols:] == 7.0).all())


@pytest.mark.parametrize("shape", [(301, 2, 3), (7, 5, 3, 2), (11, 9, 13), (2, 3, 1, 5, 7), (5, 1, 1, 17)], ids=str)
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_gaps_after_every_dimension(shape, dtype):
    """A thread's eight elements cross the ends of rows, planes and images, each followed by a gap of its own."""
    gen = torch.Generator().manual_seed(7)
    wide = [n + d for d, n in enumerate(shape)]
    inner = tuple(slice(0, n) for n in shape)
    x, r = (randn(gen, *wide).to(dtype).to(dev())[inner] for _ in range(2))
    y = torch.full(wide, 7.0, dtype=dtype, device=dev())
    check(x, r, 0.25, 3, 4, y[inner])
    assert int((y == 7.0).sum()) >= y.numel() - x.numel()
    check(x, r.permute(*reversed(range(r.dim()))).contiguous().permute(*reversed(range(r.dim()))), 0.25, 3, 4, y[inner])


def test_published_numbers():
    """Philox4x32-10's known answer for a counter and key of zeros, 6627e8d5 e169c58d bc57ac4c 9b00dbd8: element j is
    kept for a threshold of its own number and dropped for one more."""
    want = [0xE8D5, 0x6627, 0xC58D, 0xE169, 0xAC4C, 0xBC57, 0xDBD8, 0x9B00]
    assert halves(8, 0, 0).tolist() == want
    x = torch.ones(8, device=dev())
    y = torch.empty_like(x)
    for j, u in enumerate(want):
        assert F.dropout_fprop(x, y, u / 65536, 0, 0) == F.Success
        assert float(y[j]) > 0
        assert F.dropout_fprop(x, y, (u + 1) / 65536, 0, 0) == F.Success
        assert float(y[j]) == 0


def test_share_and_mean():
    n, p = 1 << 22, 0.3
    x = torch.ones(n, device=dev())
    y = torch.empty_like(x)
    assert F.dropout_fprop(x, y, p, 11, 12) == F.Success
    kept = float((y > 0).double().mean())
    sigma = (p * (1 - p) / n) ** 0.5
    assert abs(kept - (1 - p)) < 6 * sigma + 2.0 ** -17
    assert abs(float(y.double().mean()) - 1) < 6 * sigma / (1 - p)
    assert F.dropout_fprop(x, z := torch.empty_like(x), p, 11, 13) == F.Success
    both = float(((y > 0) & (z > 0)).double().mean())  # another offset: another mask, independent of the first
    assert abs(both - (1 - p) ** 2) < 6 * ((1 - p) ** 2 * (1 - (1 - p) ** 2) / n) ** 0.5 + 2.0 ** -16


@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
def test_dropped_values_are_zero_whatever_they_hold_and_in_place(dtype):
    x = torch.full((4096,), float("inf"), dtype=dtype, device=dev())
    x[::3] = float("nan")
    check(x, None, 0.5, 8, 9, torch.empty_like(x))
    keep = (halves(4096, 8, 9) >= 32768).to(dev())
    y = torch.empty_like(x)
    assert F.dropout_fprop(x, y, 0.5, 8, 9) == F.Success
    assert not bool(y[~keep].any())
    gen = torch.Generator().manual_seed(3)
    v, r = (randn(gen, 5000).to(dtype).to(dev()) for _ in range(2))
    check(v, r, 0.5, 8, 9, want := torch.empty_like(v))
    a, b = v.clone(), r.clone()
    assert F.dropout_fprop(a, a, 0.5, 8, 9, residual=r) == F.Success
    assert F.dropout_fprop(v, b, 0.5, 8, 9, residual=b) == F.Success
    assert torch.equal(a, want) and torch.equal(b, want)


def test_step_in_a_captured_graph():
    """Every replay adds to the step and draws the mask that an eager call with that offset draws."""
    gen = torch.Generator().manual_seed(4)
    x = randn(gen, 10000).float().to(dev())
    y, step = torch.empty_like(x), torch.zeros(1, dtype=torch.int64, device=dev())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(stream):
        assert F.dropout_fprop(x, y, 0.3, 21, 5, step=step) == F.Success
        stream.synchronize()
        with torch.cuda.graph(graph, stream=stream):
            step.add_(1)
            assert F.dropout_fprop(x, y, 0.3, 21, 5, step=step) == F.Success
    torch.cuda.synchronize()
    for replay in range(1, 4):
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        want = torch.empty_like(x)
        assert F.dropout_fprop(x, want, 0.3, 21, 5 + replay) == F.Success
        assert torch.equal(y, want)
        assert F.dropout_bprop(x, want, 0.3, 21, 5, step=step) == F.Success  # the backward pass of the same step
        assert torch.equal(y, want)


def test_empty_and_other_streams():
    e = torch.empty((3, 0, 2), device=dev())
    assert F.dropout_fprop(e, e, 0.5, 1, 2) == F.Success
    x = torch.randn(3000, device=dev())
    y, z = torch.empty_like(x), torch.empty_like(x)
    assert F.dropout_fprop(x, y, 0.5, 1, 2) == F.Success
    torch.cuda.synchronize()
    assert F.dropout_fprop(x, z, 0.5, 1, 2, stream=torch.cuda.Stream()) == F.Success
    torch.cuda.synchronize()
    assert torch.equal(y, z)


def test_offsets_past_32_bits():
    far = (1 << 32) + 8
    store = torch.zeros(2 * far + 64, dtype=torch.bfloat16, device=dev())
    x = store.as_strided((3, 40), (far, 1))
    gen = torch.Generator().manual_seed(5)
    x.copy_(randn(gen, 3, 40).to(dev()))
    check(x, x, 0.5, 6, 7, torch.empty((3, 40), dtype=torch.bfloat16, device=dev()))
    # more elements than 32 bits count: the last ones, from the generator's counter above 2^29
    n = (1 << 32) + 1000
    flat = store[:n]
    flat.fill_(1.0)
    assert F.dropout_fprop(flat, flat, 0.5, 6, 7) == F.Success
    assert float(flat[:1000].float().sum()) > 0
    tail = flat[-1000:].cpu()
    import numpy as np
    from operators_util import halves_at
    keep = torch.from_numpy(halves_at(np.arange(n - 1000, n), 6, 7) >= 32768)
    assert torch.equal(tail > 0, keep)
    del store, flat

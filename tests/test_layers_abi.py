"""CPU-only checks of the operators around a linear layer: what the C entry points refuse before anything is enqueued, and the
Python wrappers' errors.  Addresses here are made up: nothing follows them."""
import ctypes

import pytest
import torch

import fbcuda_amd as F
from test_operators_abi import BF16, BIG, F16, F32, WS, arr


def norm(x=arr(4, 6), w=None, b=None, y=arr(4, 6), mean=None, rstd=None, eps=1e-5, ws=WS, size=BIG):
    return F.lib().fbfft_layer_norm_fprop(x, w, b, y, mean, rstd, eps, ws, size, None)


def norm_back(x=arr(4, 6), w=None, mean=arr(4), rstd=arr(4), g=arr(4, 6), gx=arr(4, 6), gw=None, gb=None, ws=WS, size=BIG):
    return F.lib().fbfft_layer_norm_bprop(x, w, mean, rstd, g, gx, gw, gb, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), 2), (dict(y=None), 2), (dict(x=arr(24)), 2), (dict(x=arr(2, 2, 6)), 2), (dict(y=arr(4, 7)), 2),
    (dict(y=arr(4, 6, kind=F16)), 2), (dict(x=arr(4, 6, kind=3)), 2), (dict(x=arr(4, 6, data=None)), 2),
    (dict(x=arr(4, 6, data=(1 << 16) + 2)), 2), (dict(x=arr(-4, 6)), 2), (dict(w=arr(5)), 2), (dict(b=arr(6, 1)), 2),
    (dict(w=arr(6, data=None)), 2), (dict(mean=arr(6)), 2), (dict(rstd=arr(4, kind=F16)), 2), (dict(rstd=arr(4, data=None)), 2),
    (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(eps=float("inf")), 1),
    (dict(x=arr(1 << 31, 2, kind=F16), y=arr(1 << 31, 2, kind=F16)), 1),
    (dict(x=arr(2, 1 << 31, kind=F16), y=arr(2, 1 << 31, kind=F16)), 1), (dict(x=arr(1 << 30, 1 << 30)), 2)])
def test_layer_norm_forward_refuses(change, code):
    assert norm(**change) == code


@pytest.mark.parametrize("change,code", [
    (dict(x=None), 2), (dict(g=None), 2), (dict(mean=None), 2), (dict(rstd=None), 2), (dict(g=arr(4, 5)), 2),
    (dict(gx=arr(4, 6, kind=BF16)), 2), (dict(gw=arr(4)), 2), (dict(gb=arr(6, kind=5)), 2), (dict(mean=arr(6)), 2),
    (dict(rstd=arr(4, kind=BF16)), 2), (dict(w=arr(4)), 2), (dict(ws=None, gw=arr(6)), 2), (dict(size=8, gw=arr(6)), 2),
    (dict(ws=ctypes.c_void_p((1 << 20) + 16), gb=arr(6)), 2)])
def test_layer_norm_backward_refuses(change, code):
    assert norm_back(**change) == code


def test_layer_norm_of_nothing():
    none = arr(0, 6, data=None)
    assert norm(x=none, y=none, ws=None, size=0) == 0
    assert norm(x=arr(4, 0), y=arr(4, 0), ws=None, size=0) == 0
    assert norm_back(gx=None) == 0  # no gradient is wanted


QUINTIC = (3.4445, -4.7750, 2.0315)


def orth(x=arr(4, 6), y=arr(4, 6), coefficients=QUINTIC * 5, steps=5, eps=1e-7, scale=1.0, ws=WS, size=BIG):
    c = None if coefficients is None else (ctypes.c_float * len(coefficients))(*coefficients)
    return F.lib().fbfft_orthogonalize(x, y, c, steps, eps, scale, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), 2), (dict(y=None), 2), (dict(x=arr(24), y=arr(24)), 2), (dict(x=arr(1, 1, 4, 6), y=arr(1, 1, 4, 6)), 2),
    (dict(y=arr(6, 4)), 2), (dict(y=arr(1, 4, 6)), 2), (dict(y=arr(4, 6, kind=BF16)), 2), (dict(x=arr(4, 6, kind=4)), 2),
    (dict(x=arr(4, 6, data=None)), 2), (dict(coefficients=None), 2), (dict(ws=None), 2), (dict(size=64), 2),
    (dict(ws=ctypes.c_void_p((1 << 20) + 64)), 2), (dict(steps=0), 1), (dict(steps=33, coefficients=QUINTIC * 33), 1),
    (dict(steps=-1), 1), (dict(eps=-1e-9), 1), (dict(eps=float("nan")), 1), (dict(eps=float("inf")), 1),
    (dict(scale=float("inf")), 1), (dict(scale=float("nan")), 1),
    (dict(x=arr(65537, 2), y=arr(65537, 2)), 1), (dict(x=arr(2, 65537), y=arr(2, 65537)), 1)])
def test_orthogonalize_refuses(change, code):
    assert orth(**change) == code


@pytest.mark.parametrize("coefficients", [
    (float("nan"), 0.0, 0.0), (1.0, float("inf"), 0.0), (33.0, 0.0, 0.0), (0.0, 33.0, 0.0), (0.0, 0.0, -33.0),
    (3.0,) + (0.0,) * 2 + (12.0, 0.0, 0.0), (4.0, 3.0, 3.0) * 4, (6.0, 0.0, 0.0, 1.0, 0.0, 0.0), (0.0, 130.0, -130.0)])
def test_orthogonalize_refuses_coefficients_that_pass_what_pieces_hold(coefficients):
    assert orth(coefficients=coefficients, steps=len(coefficients) // 3) == 1


def test_orthogonalize_of_nothing():
    for size in ((0, 6), (4, 0), (0, 4, 6), (3, 0, 6)):
        none = arr(*size, data=None)
        assert orth(x=none, y=none, ws=None, size=0) == 0


def packed(rows, blocks, codes=1 << 16, scales=(1 << 16) + 1, stride=None, scale_stride=None):
    return F.Mx4(codes, scales, rows, blocks, 16 * blocks if stride is None else stride, blocks if scale_stride is None else scale_stride)


BAD = [(None, 2), (packed(3, 2), 2), (packed(4, 1), 2), (packed(4, 2, codes=None), 2), (packed(4, 2, scales=None), 2),
       (packed(4, 2, codes=(1 << 16) + 8), 2), (packed(4, 2, stride=40), 2), (packed(4, 2, stride=16), 2),
       (packed(4, 2, stride=-32), 2), (packed(4, 2, scale_stride=1), 2), (packed(-4, 2), 2), (packed(4, -2), 2),
       (packed(4, 2, stride=(1 << 22) + 16), 1), (packed(4, 2, scale_stride=(1 << 22) + 1), 1)]


@pytest.mark.parametrize("q,code", BAD)
def test_mx4_refuses(q, code):
    assert F.lib().fbfft_mx4_quantize(arr(4, 40), q, None) == code
    assert F.lib().fbfft_mx4_dequantize(q, arr(4, 40), None) == code


def test_mx4_refuses_arrays():
    for x in (None, arr(4), arr(1, 4, 40), arr(4, 40, kind=7), arr(4, 40, data=None), arr(4, 65)):
        assert F.lib().fbfft_mx4_quantize(x, packed(4, 2), None) == 2
        assert F.lib().fbfft_mx4_dequantize(packed(4, 2), x, None) == 2
    wide = (1 << 22) + 1
    assert F.lib().fbfft_mx4_quantize(arr(1, wide), packed(1, (1 << 17) + 1), None) == 1
    assert F.lib().fbfft_mx4_quantize(arr(1 << 31, 1), packed(1 << 31, 1), None) == 1
    assert F.lib().fbfft_mx4_dequantize(packed(1 << 31, 1), arr(1 << 31, 1), None) == 1


def test_mx4_of_nothing():
    none = F.Mx4(None, None, 0, 2, 0, 0)
    assert F.lib().fbfft_mx4_quantize(arr(0, 40, data=None), none, None) == 0
    assert F.lib().fbfft_mx4_dequantize(F.Mx4(None, None, 4, 0, 0, 0), arr(4, 0, data=None), None) == 0


def linear(x=arr(4, 40), q=None, w=packed(5, 2), bias=None, r=None, y=arr(4, 5), act=0, ws=WS, size=BIG):
    return F.lib().fbfft_linear_mx4_fprop(x, q, w, bias, r, y, act, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), 2), (dict(q=packed(4, 2)), 2), (dict(w=None), 2), (dict(y=None), 2), (dict(x=arr(4, 32)), 2), (dict(x=arr(4, 65)), 2),
    (dict(x=arr(5, 40)), 2), (dict(x=arr(4, 40, kind=F16)), 2), (dict(x=arr(4, 40, data=None)), 2), (dict(w=packed(6, 2)), 2),
    (dict(w=packed(5, 2, stride=24)), 2), (dict(y=arr(4, 6)), 2), (dict(y=arr(20)), 2), (dict(bias=arr(4)), 2), (dict(r=arr(5, 4)), 2),
    (dict(r=arr(4, 5, kind=BF16)), 2), (dict(act=4), 2), (dict(act=-1), 2), (dict(x=None, q=packed(3, 2)), 2),
    (dict(x=None, q=packed(4, 3)), 2), (dict(x=None, q=packed(4, 2, codes=(1 << 16) + 4)), 2), (dict(w=packed(5, 2, stride=1 << 23)), 1),
    (dict(x=None, q=packed(4, 2, scale_stride=1 << 23)), 1), (dict(x=arr(1 << 23, 40), y=arr(1 << 23, 5)), 1),
    (dict(w=packed(1 << 23, 2), y=arr(4, 1 << 23)), 1)])
def test_linear_mx4_refuses(change, code):
    assert linear(**change) == code


def test_linear_mx4_refuses_workspaces():
    x, y, w = arr(600, 4096), arr(600, 512), packed(512, 128)
    assert F.lib().fbfft_linear_mx4_workspace(600, 4096, 512) > 0
    assert linear(x=x, y=y, w=w, ws=None) == 2
    assert linear(x=x, y=y, w=w, size=256) == 2
    assert linear(x=x, y=y, w=w, ws=ctypes.c_void_p((1 << 20) + 128)) == 2


def test_linear_mx4_refuses_what_no_launch_holds():
    """2^32 lanes and more, known before anything is enqueued (without a GPU, a launch is another error)."""
    n = (1 << 23) - 1
    for kind in (F32, F16, BF16):
        assert linear(x=arr(n, 1, kind=kind), w=packed(1 << 16, 1), y=arr(n, 1 << 16, kind=kind), size=1 << 50) == 1
        assert linear(x=arr(n, 0, kind=kind), w=packed(1 << 17, 0), y=arr(n, 1 << 17, kind=kind), size=1 << 50) == 1


def test_linear_mx4_of_nothing():
    assert linear(x=arr(0, 40), y=arr(0, 5), ws=None, size=0) == 0
    assert linear(w=packed(0, 2), y=arr(4, 0), ws=None, size=0) == 0


def test_workspace_sizes():
    L = F.lib()
    for bad in [(2, 4, 4), (-1, 4, 4), (0, 0, 4), (1, 4, 0), (1, 1 << 31, 4), (1, 4, 1 << 31), (1, 1 << 30, 1 << 30)]:
        assert L.fbfft_layer_norm_workspace(*bad) == 0
    assert L.fbfft_layer_norm_workspace(1, 4, 4) > 0
    for bad in [(0, 4, 4), (-1, 4, 4), (1, 0, 4), (1, 4, -4), (1, 65537, 4), (1, 4, 65537), (1 << 40, 4, 4)]:
        assert L.fbfft_orthogonalize_workspace(*bad) == 0
    assert L.fbfft_orthogonalize_workspace(2, 4, 4) > 0
    for bad in [(0, 4, 4), (4, -1, 4), (4, 4, 0), (1 << 23, 4, 4), (4, 4, 1 << 23), (4, (1 << 22) + 1, 4)]:
        assert L.fbfft_linear_mx4_workspace(*bad) == 0


def test_python_wrappers_refuse():
    x, q, s = torch.zeros((4, 64)), torch.zeros((4, 32), dtype=torch.uint8), torch.zeros((4, 2), dtype=torch.uint8)
    with pytest.raises(ValueError):
        F.layer_norm_fprop(x, None, None, x, None)  # not on the GPU
    with pytest.raises(ValueError):
        F.layer_norm_bprop(x, None, x[:, 0], x[:, 0], x, x, None, None, None)
    with pytest.raises(ValueError):
        F.orthogonalize(x, x, None)
    for coefficients in ((1.0, 2.0), [(1.0, 2.0, 3.0)] * 4, [(1.0, 2.0)] * 5):
        with pytest.raises(ValueError):
            F.orthogonalize(x, x, None, coefficients=coefficients)
    with pytest.raises(ValueError):
        F.mx4_quantize(x, q, s)
    with pytest.raises(ValueError):
        F.mx4_dequantize(q, s, x)
    with pytest.raises(ValueError):
        F.linear_mx4_fprop(x, q, s, None, x, None)
    with pytest.raises(ValueError):
        F.linear_mx4_fprop(x, q, s, None, x, None, activation="tanh")
    with pytest.raises(TypeError):
        F.packed_rows(x, s)
    with pytest.raises(TypeError):
        F.packed_rows(q, None)
    for codes, scales in ((q[:3], s), (q[:, :31], s), (q.t(), s.t()), (torch.zeros((4, 64), dtype=torch.uint8)[:, ::2], s), (q[0], s[0])):
        with pytest.raises(ValueError):
            F.packed_rows(codes, scales)
    assert F.packed_rows(None, None) is None
    assert ctypes.sizeof(F.Mx4) == 48


def test_words_that_products_read_lie_in_their_operands():
    """tests/cpp/steps_check.cpp: every word that products of pairs and of 4-bit rows move straight to LDS, over ragged rows and
    k and ranges of k."""
    import os
    import subprocess
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
    subprocess.check_call(["make", "-C", at, "-B", "steps_check"], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    out = subprocess.run([os.path.join(at, "steps_check")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout

"""CPU-only checks of the operators around a convolution layer: the struct's layout, what the C entry points refuse
before anything is enqueued, and the Python wrappers' errors.  Addresses here are made up: nothing follows them."""
import ctypes

import pytest
import torch

import fbcuda_amd as F

F32, F16, BF16 = range(3)
WS = ctypes.c_void_p(1 << 20)  # 256-byte aligned
BIG = 1 << 40


def arr(*size, kind=F32, stride=None, data=1 << 16):
    a = F.Array()
    a.data, a.dim, a.type = data, len(size), kind
    step = 1
    for i in range(min(len(size), F.MAX_DIM) - 1, -1, -1):
        a.size[i], a.stride[i] = size[i], step
        step *= max(1, size[i])
    if stride:
        a.stride[:len(stride)] = stride
    return a


def test_array_layout():
    # pointer, 5 strides, 5 sizes, rank, type
    assert (F.Array.data.offset, F.Array.stride.offset, F.Array.size.offset) == (0, 8, 48)
    assert (F.Array.dim.offset, F.Array.type.offset, ctypes.sizeof(F.Array)) == (88, 92, 96)
    t = torch.zeros((3, 4, 5), dtype=torch.bfloat16).permute(2, 0, 1)
    a = F.array(t)
    assert (a.dim, a.type, a.data) == (3, BF16, t.data_ptr())
    assert list(a.size)[:3] == [5, 3, 4] and list(a.stride)[:3] == [1, 20, 5]
    assert F.array(None) is None


def norm(input=arr(2, 8, 3, 3), weight=None, bias=None, output=arr(2, 8, 3, 3), mean=None, rstd=None, groups=2, eps=1e-5,
         act=0, ws=WS, size=BIG):
    return F.lib().fbfft_group_norm_fprop(input, weight, bias, output, mean, rstd, groups, eps, act, ws, size, None)


def norm_back(input=arr(2, 8, 3, 3), weight=None, bias=None, mean=arr(2, 2), rstd=arr(2, 2), g=arr(2, 8, 3, 3),
              gi=arr(2, 8, 3, 3), gw=None, gb=None, groups=2, act=0, ws=WS, size=BIG):
    return F.lib().fbfft_group_norm_bprop(input, weight, bias, mean, rstd, g, gi, gw, gb, groups, act, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(input=None), 2), (dict(output=None), 2), (dict(input=arr(2, 8, 9)), 2), (dict(output=arr(2, 8, 3, 4)), 2),
    (dict(output=arr(2, 8, 3, 3, kind=F16)), 2), (dict(input=arr(2, 8, 3, 3, kind=3)), 2),
    (dict(input=arr(2, 8, 3, 3, kind=-1)), 2), (dict(input=arr(2, 8, 3, 3, data=None)), 2),
    (dict(input=arr(2, 8, 3, 3, data=(1 << 16) + 2)), 2), (dict(input=arr(2, -8, 3, 3)), 2),
    (dict(groups=0), 1), (dict(groups=3), 1), (dict(groups=-2), 1), (dict(groups=16), 1),
    (dict(weight=arr(7)), 2), (dict(bias=arr(8, 1)), 2), (dict(weight=arr(8, data=None)), 2),
    (dict(mean=arr(2, 3)), 2), (dict(rstd=arr(2, 2, kind=F16)), 2), (dict(rstd=arr(2, 2, data=None)), 2),
    (dict(act=4), 2), (dict(act=-1), 2), (dict(eps=-1.0), 1), (dict(eps=float("nan")), 1), (dict(eps=float("inf")), 1),
    (dict(input=arr(1 << 20, 1 << 12, 1, 1), output=arr(1 << 20, 1 << 12, 1, 1)), 1),
    (dict(input=arr(1, 2, 1 << 16, 1 << 16), output=arr(1, 2, 1 << 16, 1 << 16)), 1),
    (dict(input=arr(1 << 30, 8, 1 << 30, 1 << 30)), 2)])
def test_group_norm_forward_refuses(change, code):
    assert norm(**change) == code


@pytest.mark.parametrize("change,code", [
    (dict(input=None), 2), (dict(g=None), 2), (dict(mean=None), 2), (dict(rstd=None), 2), (dict(g=arr(2, 8, 3, 2)), 2),
    (dict(gi=arr(2, 8, 3, 3, kind=BF16)), 2), (dict(gw=arr(9)), 2), (dict(gb=arr(8, kind=5)), 2), (dict(mean=arr(2, 8)), 2),
    (dict(rstd=arr(2, 2, kind=BF16)), 2), (dict(groups=5), 1), (dict(act=9), 2), (dict(ws=None), 2), (dict(size=8), 2),
    (dict(ws=ctypes.c_void_p((1 << 20) + 16)), 2), (dict(weight=arr(2)), 2)])
def test_group_norm_backward_refuses(change, code):
    assert norm_back(**change) == code


def test_group_norm_refuses_what_no_launch_holds():
    """One image of 2^32 lanes and more, known before anything is enqueued (without a GPU, a launch is another error)."""
    c, most = 1 << 28, 1 << 50
    x = arr(1, c, 1, 1, kind=F16)
    assert norm(input=x, output=x, groups=c, size=most) == 1
    stats = arr(1, c // 2)
    assert norm_back(input=x, g=x, gi=x, mean=stats, rstd=stats, groups=c // 2, size=most) == 1


@pytest.mark.parametrize("size", [(1, 1, 1, 0x7fff0001), (1, 1, 1, 0x7ffff000), (1, 3, 1, 0x7ffffff // 3 * 16)])
def test_group_norm_refuses_groups_whose_ends_31_bits_do_not_pass(size):
    """A lane steps past the end of its group by up to 14336 values and more before it compares: of a group of 2^31 - 4096
    its 32-bit place would come out negative, in front of the group."""
    x, most = arr(*size, kind=F16), 1 << 50
    assert norm(input=x, output=x, groups=1, size=most) == 1
    assert norm_back(input=x, g=x, gi=x, mean=arr(1, 1), rstd=arr(1, 1), groups=1, size=most) == 1


def test_group_norm_of_nothing():
    assert norm(input=arr(0, 8, 3, 3, data=None), output=arr(0, 8, 3, 3, data=None), ws=None, size=0) == 0
    assert norm(input=arr(2, 8, 0, 3), output=arr(2, 8, 0, 3), ws=None, size=0) == 0
    assert norm_back(gi=None) == 0  # no gradient is wanted


def linear(x=arr(4, 6), w=arr(5, 6), bias=None, r=None, y=arr(4, 5), z=None, act=0, ws=WS, size=BIG):
    return F.lib().fbfft_linear_fprop(x, w, bias, r, y, z, act, ws, size, None)


def linear_back(x=arr(4, 6), w=arr(5, 6), g=arr(4, 5), z=None, gx=arr(4, 6), gw=arr(5, 6), gb=arr(5), act=0, ws=WS, size=BIG):
    return F.lib().fbfft_linear_bprop(x, w, g, z, gx, gw, gb, act, ws, size, None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), 2), (dict(w=None), 2), (dict(y=None), 2), (dict(x=arr(4, 7)), 2), (dict(w=arr(5, 6, kind=F16)), 2),
    (dict(y=arr(5, 4)), 2), (dict(y=arr(4, 5, kind=BF16)), 2), (dict(x=arr(1, 4, 6)), 2), (dict(bias=arr(4)), 2),
    (dict(r=arr(4, 6)), 2), (dict(r=arr(4, 5, kind=F16)), 2), (dict(z=arr(5, 5)), 2), (dict(act=7), 2),
    (dict(x=arr(4, 6, data=None)), 2), (dict(w=arr(5, 6, data=(1 << 16) + 1)), 2),
    (dict(x=arr(1 << 23, 6), y=arr(1 << 23, 5)), 1), (dict(w=arr(1 << 23, 6), y=arr(4, 1 << 23)), 1)])
def test_linear_forward_refuses(change, code):
    assert linear(**change) == code


@pytest.mark.parametrize("change,code", [
    (dict(g=None), 2), (dict(x=None), 2), (dict(w=None), 2), (dict(act=1), 2), (dict(act=2, z=arr(4, 6)), 2),
    (dict(act=4, z=arr(4, 5)), 2), (dict(gx=arr(4, 5)), 2), (dict(gw=arr(6, 5)), 2), (dict(gb=arr(6)), 2), (dict(ws=None), 2),
    (dict(size=16), 2), (dict(ws=ctypes.c_void_p((1 << 20) + 128)), 2), (dict(g=arr(4, 5, kind=F16)), 2),
    (dict(w=arr(5)), 2), (dict(x=arr(5, 6)), 2)])
def test_linear_backward_refuses(change, code):
    assert linear_back(**change) == code


@pytest.mark.parametrize("change", [
    dict(x=None, w=arr(1, 4000000), g=arr(4000000, 1), gx=None, gw=None, gb=arr(1)),
    dict(x=arr(100, 4000000), w=None, g=arr(100, 400000), gx=None, gw=None, gb=arr(400000))])
def test_linear_backward_refuses_products_that_no_workspace_is_made_for(change):
    """gradBias alone: M K or N K, of an operand that is not given, above 2^40.  The workspace's size is 0 there, and a call
    without one would take address 0 for it."""
    assert linear_back(ws=None, size=0, **change) == 1


@pytest.mark.parametrize("kind", [F32, F16, BF16])
def test_linear_refuses_what_no_launch_holds(kind):
    """2^32 lanes and more, known before anything is enqueued (without a GPU, a launch is another error)."""
    n, most = 1 << 20, 1 << 50  # bytes of a workspace
    a = lambda *size: arr(*size, kind=kind)  # noqa: E731
    assert linear(x=a(n, 0), w=a(n, 0), y=a(n, n), size=most) == 1  # results that are the bias's activation
    assert linear(x=a(n, 1), w=a(n, 1), y=a(n, n), size=most) == 1
    assert linear(x=a(1 << 19, 4), w=a(n, 4), y=arr(1 << 19, n, kind=kind, stride=(1, 1 << 19)), size=most) == 1
    assert linear_back(x=None, w=None, g=a(n, n), gx=None, gw=None, gb=arr(n), size=most) == 1
    assert linear_back(x=None, w=a(1, n), g=a(n, 1), gx=a(n, n), gw=None, gb=None, size=most) == 1
    assert linear_back(x=a(1, n), w=None, g=a(1, n), gx=None, gw=a(n, n), gb=None, size=most) == 1


def test_linear_of_nothing():
    assert linear(x=arr(0, 6), y=arr(0, 5), ws=None, size=0) == 0
    assert linear(w=arr(0, 6), y=arr(4, 0), ws=None, size=0) == 0


def drop(x=arr(10), r=None, y=arr(10), p=0.5, step=None):
    return F.lib().fbfft_dropout_fprop(x, r, y, p, 1, 2, step, None)


@pytest.mark.parametrize("change,code", [
    (dict(x=None), 2), (dict(y=None), 2), (dict(y=arr(11)), 2), (dict(y=arr(10, kind=F16)), 2), (dict(r=arr(9)), 2),
    (dict(r=arr(10, kind=BF16)), 2), (dict(x=arr(10, data=None)), 2), (dict(p=-0.1), 1), (dict(p=1.1), 1),
    (dict(p=float("nan")), 1), (dict(step=ctypes.c_void_p(4)), 2), (dict(x=arr(), y=arr()), 2),
    (dict(x=arr(1, 1, 1, 1, 1, 1), y=arr(1, 1, 1, 1, 1, 1)), 2), (dict(x=arr(1 << 21, 1 << 21), y=arr(1 << 21, 1 << 21)), 2)])
def test_dropout_refuses(change, code):
    assert drop(**change) == code
    if "r" not in change:
        args = dict(x=arr(10), y=arr(10), p=0.5, step=None, **{})
        args.update(change)
        assert F.lib().fbfft_dropout_bprop(args["x"], args["y"], args["p"], 1, 2, args["step"], None) == code


def test_dropout_refuses_what_no_launch_holds():
    for kind in (F32, F16, BF16):
        for n in (1 << 35, 1 << 40):
            assert drop(x=arr(n, kind=kind), y=arr(n, kind=kind)) == 1
            assert F.lib().fbfft_dropout_bprop(arr(n, kind=kind), arr(n, kind=kind), 0.5, 1, 2, None, None) == 1


def test_dropout_of_nothing():
    assert drop(x=arr(0, data=None), y=arr(0, data=None)) == 0
    assert drop(x=arr(3, 0, 2), y=arr(3, 0, 2), p=1.0) == 0


def test_workspace_sizes():
    L = F.lib()
    for bad in [(2, 1, 8, 9, 2), (0, 0, 8, 9, 2), (0, 1, 8, 9, 3), (1, 1, 8, 0, 2), (1, 1 << 40, 8, 9, 2), (-1, 1, 8, 9, 2)]:
        assert L.fbfft_group_norm_workspace(*bad) == 0
    assert L.fbfft_group_norm_workspace(1, 2, 8, 9, 2) > 0
    for bad in [(2, 4, 4, 4, 0), (0, -1, 4, 4, 0), (0, 4, 4, 4, 3), (1, 1 << 39, 4, 4, 0), (1, 4, 1 << 39, 4, 0)]:
        assert L.fbfft_linear_workspace(*bad) == 0
    assert L.fbfft_linear_workspace(1, 4, 4, 4, 1) > 0


def test_python_wrappers_refuse():
    x = torch.zeros((2, 8, 3, 3))
    with pytest.raises(ValueError):
        F.group_norm_fprop(x, None, None, x, 2, None)  # not on the GPU
    with pytest.raises(ValueError):
        F.group_norm_fprop(x, None, None, x, 2, None, activation="tanh")
    with pytest.raises(ValueError):
        F.linear_fprop(x[0, 0], x[0, 0], None, x[0, 0], None)
    with pytest.raises(ValueError):
        F.dropout_fprop(x, x, 0.5, 1, 2)
    with pytest.raises(TypeError):
        F.array(torch.zeros(3, dtype=torch.float64))
    with pytest.raises(ValueError):
        F.array(torch.zeros((1,) * 6))
    with pytest.raises(TypeError):
        F.linear_workspace(0, 1, 1, 1, torch.float64)


def test_words_that_products_read_lie_in_their_operands():
    """tests/cpp/linear_check.cpp: every word that a product of 16-bit operands moves straight to LDS
    (fbcuda_amd/csrc/linear_step.h) over ragged rows and k, both layouts and ranges of k."""
    import os
    import subprocess
    at = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp")
    subprocess.check_call(["make", "-C", at, "-B", "linear_check"], stdout=subprocess.DEVNULL, stderr=subprocess.DEVNULL)
    out = subprocess.run([os.path.join(at, "linear_check")], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "OK", out.stdout

"""Plain forms, in 64 bits on the CPU, of the operators around a convolution layer, and the bounds that the tests hold
results to.

A bound is made of two parts: half a unit in the last place of the result's type (U), and a number of fp32 roundings
(2^-24 each) of the quantities that meet in a result, whose sizes the plain form returns next to the result."""
import math

import numpy as np
import torch

U = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
# the spacing of the smallest numbers, half of it lost at most
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
R = 2.0 ** -24
TYPES = [torch.float32, torch.float16, torch.bfloat16]
NAMES = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16"}
ACTS = ["none", "relu", "silu", "gelu"]


def randn(gen, *shape, std=1.0, mean=0.0):
    return torch.randn(*shape, generator=gen, dtype=torch.float64) * std + mean


def within(got, want, bound):
    """Asserts |got - want| <= bound everywhere, NaN and infinities in the same places."""
    got, want = got.detach().cpu().double(), want.double()
    assert got.shape == want.shape
    fine = torch.isfinite(want)
    assert torch.equal(fine, torch.isfinite(got))
    assert torch.equal(torch.isnan(want), torch.isnan(got))
    off = torch.where(fine, (got - want).abs(), torch.zeros_like(want))
    over = off - torch.where(fine, bound.expand_as(want), torch.ones_like(want))
    assert not bool((over > 0).any()), "off by %.3e where %.3e is allowed (%d of %d values)" % (
        off.flatten()[over.argmax()], bound.expand_as(want).flatten()[over.argmax()], int((over > 0).sum()), over.numel())


def rounded(want, dtype):
    return U[dtype] * want.abs() + TINY[dtype]


def act(z, name):
    if name == "relu":
        return torch.where(z < 0, torch.zeros_like(z), z)
    if name == "silu":
        return z / (1 + torch.exp(-z))
    if name == "gelu":
        return 0.5 * z * torch.special.erfc(-z * math.sqrt(0.5))
    return z


def act_slope(z, name):
    if name == "relu":
        return (z > 0).double()
    if name == "silu":
        u = 1 / (1 + torch.exp(-z))
        return u * (1 + z * (1 - u))
    if name == "gelu":
        return 0.5 * torch.special.erfc(-z * math.sqrt(0.5)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _param(p, c, otherwise):
    p = torch.full((c,), float(otherwise), dtype=torch.float64) if p is None else p.detach().cpu().double()
    return p[None, :, None, None]


def norm(x, weight, bias, groups, eps, name):
    """(output, mean, rstd, bound of the output's fp32 part)"""
    x = x.detach().cpu().double()
    b, c = x.shape[:2]
    flat = x.reshape(b, groups, -1)
    mean = flat.mean(-1)
    rstd = 1 / torch.sqrt((flat - mean[..., None]).square().mean(-1) + eps)
    w, s = _param(weight, c, 1), _param(bias, c, 0)
    each = lambda v: v.repeat_interleave(c // groups, 1)[:, :, None, None]  # noqa: E731
    xh = (x - each(mean)) * each(rstd)
    z = xh * w + s
    # rounding of the mean, of differences, products and sums, and the activation's own
    size = (xh * w).abs() + s.abs() + (each(mean) * each(rstd) * w).abs() + z.abs() + 1
    return act(z, name), mean, rstd, 16 * R * size


def norm_grads(x, weight, bias, mean, rstd, gy, groups, name):
    """((gradInput, bound), (gradWeight, bound), (gradBias, bound))"""
    x, gy, mean, rstd = (v.detach().cpu().double() for v in (x, gy, mean, rstd))
    b, c = x.shape[:2]
    w, s = _param(weight, c, 1), _param(bias, c, 0)
    each = lambda v: v.repeat_interleave(c // groups, 1)[:, :, None, None]  # noqa: E731
    over = lambda v: each(v.reshape(b, groups, -1).mean(-1))  # noqa: E731
    xh = (x - each(mean)) * each(rstd)
    z = xh * w + s
    dz = gy * act_slope(z, name)
    dx = each(rstd) * (dz * w - over(dz * w) - xh * over(dz * w * xh))
    # of dz: the activation's slope changes by at most 1.2 times what z is off by
    size = gy.abs() * (1 + z.abs() + (xh * w).abs() + s.abs() + (each(mean) * each(rstd) * w).abs())
    dsize = each(rstd) * (size * w.abs() + over(size * w.abs()) + xh.abs() * over(size * w.abs() * (1 + xh.abs())))
    sums = (0, 2, 3)
    return ((dx, 32 * R * dsize), ((dz * xh).sum(sums), 64 * R * (size * (1 + xh.abs())).sum(sums)),
            (dz.sum(sums), 64 * R * size.sum(sums)))


def _chain(k):
    """fp32 roundings of a sum of k products, in units of the sum of their sizes: a random walk's share of k."""
    return R * (8 + 2 * math.sqrt(k))


def linear(x, w, bias, residual, name):
    """(output, its bound, z, its bound); bounds of the fp32 parts"""
    x, w = x.detach().cpu().double(), w.detach().cpu().double()
    z, size = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, size = z + bias.detach().cpu().double(), size + bias.detach().cpu().double().abs()
    zb = _chain(x.shape[1]) * size + R * z.abs()
    y = act(z, name)
    yb = 1.2 * zb + 8 * R * (1 + z.abs())
    if residual is not None:
        r = residual.detach().cpu().double()
        y, yb = y + r, yb + R * (y.abs() + r.abs())
    return y, yb, z, zb


def linear_grads(x, w, gy, z, name, dtype):
    """((gradInput, bound), (gradWeight, bound), (gradBias, bound)); dz is rounded to dtype before the products"""
    x, w, gy = (v.detach().cpu().double() for v in (x, w, gy))
    dz = gy if z is None else gy * act_slope(z.detach().cpu().double(), name)
    own = 16 * R * gy.abs() * (1 + (0 if z is None else z.detach().cpu().double().abs()))
    size = dz.abs() * (1 + 0) + own
    lost = own + (0 if z is None else U[dtype] * dz.abs() + TINY[dtype])
    m, n = gy.shape
    return ((dz @ w, lost @ w.abs() + _chain(n) * (size @ w.abs())),
            (dz.t() @ x, lost.t() @ x.abs() + _chain(m) * (size.t() @ x.abs())),
            (dz.sum(0), own.sum(0) + _chain(m) * size.sum(0)))


def halves(count, seed, offset):
    """The 16-bit numbers of elements 0 ... count-1."""
    return torch.from_numpy(halves_at(np.arange(count), seed, offset))


def halves_at(index, seed, offset):
    """The 16-bit numbers of these elements: Philox4x32-10 in numpy."""
    low, up = np.uint64(0xFFFFFFFF), np.uint64(32)
    index = index.astype(np.uint64)
    i = index >> np.uint64(3)
    offset %= 2 ** 64
    a, b = i & low, i >> up
    c, d = np.full_like(i, offset & 0xFFFFFFFF), np.full_like(i, offset >> 32)
    for r in range(10):
        k0, k1 = (np.uint64(((seed >> s) + r * inc) & 0xFFFFFFFF) for s, inc in ((0, 0x9E3779B9), (32, 0xBB67AE85)))
        p, q = a * np.uint64(0xD2511F53), c * np.uint64(0xCD9E8D57)
        a, b, c, d = (q >> up) ^ b ^ k0, q & low, (p >> up) ^ d ^ k1, p & low
    words = np.stack([a, b, c, d], 1)
    j = (index & np.uint64(7)).astype(np.int64)
    word = words[np.arange(len(index)), j // 2]
    return (np.where(j % 2, word >> np.uint64(16), word) & np.uint64(0xFFFF)).astype(np.int64)


def dropout(x, residual, p, seed, offset):
    """(output, bound of its fp32 part)"""
    cut = math.floor(p * 65536 + 0.5)
    x = x.detach().cpu().double()
    keep = (halves(x.numel(), seed, offset) >= cut).view(x.shape)
    y = torch.where(keep, x * (65536 / (65536 - cut) if cut < 65536 else 0.0), torch.zeros_like(x))
    bound = 2 * R * torch.nan_to_num(y, posinf=0.0, neginf=0.0, nan=0.0).abs()
    if residual is not None:
        r = residual.detach().cpu().double()
        y, bound = y + r, bound + R * torch.nan_to_num(y + r, posinf=0.0, neginf=0.0, nan=0.0).abs()
    return y, bound

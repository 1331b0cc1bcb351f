"""Plain forms, in 64 bits on the CPU, of the operators around a linear layer, and the bounds that the tests hold results
to: half a unit in the last place of the result's type, and fp32 roundings (R each) of what meets in a result."""
import math

import torch

from operators_util import R, TINY, U

BLOCK = 32


def chain(k):
    """fp32 roundings of a sum of k terms, in units of the sum of their sizes: a random walk's share of k."""
    return R * (8 + 2 * math.sqrt(k))


def _param(p, n, otherwise):
    return torch.full((n,), float(otherwise), dtype=torch.float64) if p is None else p.detach().cpu().double()


def layer_norm(x, weight, bias, eps):
    """((output, bound), (mean, bound), (rstd, bound)); bounds of the fp32 parts"""
    x = x.detach().cpu().double()
    n = x.shape[1]
    w, b = _param(weight, n, 1), _param(bias, n, 0)
    mean = x.mean(-1, keepdim=True)
    var = (x - mean).square().mean(-1, keepdim=True)
    rstd = 1 / torch.sqrt(var + eps)
    xh = (x - mean) * rstd
    off = chain(n) * x.abs().mean(-1, keepdim=True)  # of the mean
    # of rstd, relative: its sum's roundings, those of every x - mean, and the mean's error squared
    lost = (x.abs() + mean.abs()) * R
    less = 0.5 * chain(n) + 4 * R + rstd.square() * (off.square() + (2 * (x - mean).abs() * lost).mean(-1, keepdim=True))
    y = xh * w + b
    bound = w.abs() * (xh.abs() * (less + 4 * R) + rstd * (off + lost)) + R * (b.abs() + 2 * y.abs())
    return (y, bound), (mean[:, 0], off[:, 0]), (rstd[:, 0], (rstd * less)[:, 0])


def layer_norm_grads(x, weight, mean, rstd, g):
    """((gradInput, bound), (gradWeight, bound), (gradBias, bound)); bounds of the fp32 parts"""
    x, g, mean, rstd = (v.detach().cpu().double() for v in (x, g, mean, rstd))
    m, n = x.shape
    w, mean, rstd = _param(weight, n, 1), mean[:, None], rstd[:, None]
    xh, h = (x - mean) * rstd, g * w
    exh = R * ((x.abs() + mean.abs()) * rstd + 2 * xh.abs())
    over = lambda v: v.mean(-1, keepdim=True)  # noqa: E731
    s1, s2 = over(h), over(h * xh)
    e1, e2 = chain(n) * over(h.abs()), chain(n) * over((h * xh).abs()) + over(h.abs() * exh)
    bound = rstd * (4 * R * (h.abs() + s1.abs() + (xh * s2).abs()) + e1 + xh.abs() * e2 + exh * s2.abs())
    return ((rstd * (h - s1 - xh * s2), bound),
            ((g * xh).sum(0), chain(m) * (g * xh).abs().sum(0) + (g.abs() * exh).sum(0)),
            (g.sum(0), chain(m) * g.abs().sum(0)))


# ---- Newton-Schulz ----

QUINTIC = (3.4445, -4.7750, 2.0315)


def orthogonal(g, triples, eps, scale, moved=None, alone=False):
    """The formula on [batch][rows][cols]; moved(v, k, unit): what becomes of a value that is held between products, from
    sums of k products, in pieces whose unit is `unit`.  alone: the factors a I + B of all steps first, and X in the end."""
    moved = moved or (lambda v, k, unit=1024: v)
    x = g.detach().cpu().double()
    turn = x.shape[1] > x.shape[2]
    x = x.transpose(1, 2) if turn else x
    x = x / (x.square().sum((1, 2), keepdim=True).sqrt() + eps)
    p, q = x.shape[1:]
    if alone:
        same = lambda v, k, unit=1024: (lambda w: w.tril() + w.tril(-1).transpose(1, 2))(moved(v, k, unit))  # noqa: E731
        x = moved(x, 1)
        gram, m = same(x @ x.transpose(1, 2), q), None
        for i, (a, b, c) in enumerate(triples):
            poly = same(b * gram + c * (gram @ gram), p)
            m = same(poly + a * torch.eye(p, dtype=torch.float64) if m is None else a * m + poly @ m, p, 64)
            if i + 1 < len(triples):
                half = same(a * gram + poly @ gram, p)
                gram = same(a * half + poly @ half, p)
        x = m @ x
    else:
        for i, (a, b, c) in enumerate(triples):
            x = moved(x, 1 if i == 0 else p)
            gram = moved(x @ x.transpose(1, 2), q)
            poly = moved(b * gram + c * (gram @ gram), p)
            x = a * x + poly @ x
    x = moved(x, p) * scale
    return x.transpose(1, 2) if turn else x


def orthogonal_bound(g, triples, eps, scale):
    """How far 22 bits of every value between the products, and 32-bit sums of them, may leave the result off: the formula
    with every such value moved by a random part of its rounding, 2^-22 of itself and 2^-25 of the pieces' unit (the smallest
    second piece), and of its sum's, 2^-24 sqrt(k) of its row's and column's size, which the root of the matrix's mean square
    stands for.  Eight such moves, three times the largest; (the rounding to the result's type apart).  bfloat16 matrices
    with three times as many columns as rows, or rows as columns, may be computed alone."""
    gen = torch.Generator().manual_seed(1)

    def moved(v, k, unit=1024):
        part = lambda: torch.rand(v.shape, generator=gen, dtype=torch.float64) * 2 - 1  # noqa: E731
        size = v.square().mean((1, 2), keepdim=True).sqrt()
        return v + part() * (2.0 ** -22 * v.abs() + 2.0 ** -25 / unit) + part() * 2.0 ** -24 * math.sqrt(k) * size

    want = orthogonal(g, triples, eps, scale)
    short, long = (-(-n // 32) for n in sorted(g.shape[1:]))
    forms = [False, True] if g.dtype == torch.bfloat16 and long >= 3 * short else [False]
    offs = [orthogonal(g, triples, eps, scale, moved, form) - want for form in forms for _ in range(8)]
    norms = torch.stack([o.square().sum((1, 2)).sqrt() for o in offs]).amax(0)
    return want, 3 * norms, 3 * torch.stack([o.abs().amax((1, 2)) for o in offs]).amax(0)


# ---- 4-bit rows ----

VALUES = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def quantized(x):
    """(codes [rows][16 blocks], scales [rows][blocks]) in uint8 of [rows][cols], from the definition."""
    x = x.detach().cpu().double()
    rows, cols = x.shape
    blocks = -(-cols // BLOCK)
    v = torch.zeros((rows, blocks * BLOCK), dtype=torch.float64)
    v[:, :cols] = x
    v = v.view(rows, blocks, BLOCK)
    fine = torch.isfinite(v).all(-1)
    clean = torch.where(fine[..., None], v, torch.zeros_like(v))
    most = clean.abs().amax(-1)
    # frexp: a magnitude in [0.5, 1) times 2^e, so floor(log2) is e - 1
    e = torch.where(most > 0, torch.frexp(most)[1].double() - 3, torch.full_like(most, -127.0)).clamp(min=-127)
    a = clean / torch.exp2(e)[..., None]
    size = a.abs().clamp(max=6)
    code, best = torch.zeros(size.shape, dtype=torch.long), size
    for i, v in enumerate(VALUES[1:], 1):
        far = (size - v).abs()
        nearer = (far < best) | ((far == best) & (i % 2 == 0))  # of two that are as near, the even code
        code, best = torch.where(nearer, torch.full_like(code, i), code), torch.minimum(far, best)
    code = code + 8 * torch.signbit(a).long()
    code = torch.where(fine[..., None], code, torch.zeros_like(code))
    scales = torch.where(fine, (e + 127).long(), torch.full(e.shape, 255))
    return (code[..., 0::2] + 16 * code[..., 1::2]).reshape(rows, -1).to(torch.uint8), scales.to(torch.uint8)


def values_of(codes, scales, cols):
    """What they stand for, in 64 bits."""
    codes, scales = codes.cpu(), scales.cpu()
    table = torch.tensor(VALUES + [-v for v in VALUES], dtype=torch.float64)
    pairs = torch.stack((codes & 15, codes >> 4), -1).flatten(1).long()
    scale = torch.where(scales == 255, torch.full(scales.shape, float("nan"), dtype=torch.float64),
                        torch.exp2(scales.double() - 127))
    return (table[pairs] * scale.repeat_interleave(BLOCK, 1))[:, :cols]


__all__ = ["R", "TINY", "U", "chain", "layer_norm", "layer_norm_grads", "orthogonal", "orthogonal_bound", "quantized",
           "values_of", "QUINTIC", "BLOCK"]

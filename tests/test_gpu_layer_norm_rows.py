"""Layer norm of many rows, where lanes hold several words of a row, and of results that leave past the caches: against the formula in 64
bits, computed on the GPU."""
import pytest
import torch

import fbcuda_amd as F
from gpu_util import dev
from layers_util import chain
from operators_util import NAMES, R, TINY, TYPES, U

pytestmark = pytest.mark.gpu

EPS = 1e-5


def within(got, want, bound):
    assert bool(((got.double() - want).abs() <= bound).all())


def rounded(want, dtype):
    return U[dtype] * want.abs() + TINY[dtype]


def make(m, n, dtype, gap):
    gen = torch.Generator(device=dev()).manual_seed(m + n)
    randn = lambda *shape: torch.randn(*shape, generator=gen, device=dev())  # noqa: E731
    rows = lambda v: torch.zeros((m, n + gap), dtype=dtype, device=dev())[:, gap // 2:gap // 2 + n].copy_(v)  # noqa: E731
    x = rows(randn(m, n) * (0.5 + randn(m, 1).abs()) + 0.5 * randn(m, 1))
    return x, 1 + 0.3 * randn(n), 0.3 * randn(n), rows(randn(m, n)), rows(torch.full((), 7.0, device=dev()))


def check(m, n, dtype, kind=torch.float32, gap=0):
    """kind: the parameters' type.  The bounds: roundings in fp32 (R each) of what meets in a result, as in layers_util."""
    x, w, b, g, y = make(m, n, dtype, gap)
    w, b = w.to(kind), b.to(kind)
    mean, rstd = (torch.full((m,), 7.0, device=dev()) for _ in range(2))
    space = lambda q: torch.empty(F.layer_norm_workspace(q, m, n), dtype=torch.uint8, device=dev())  # noqa: E731
    assert F.layer_norm_fprop(x, w, b, y, space(0), eps=EPS, mean=mean, rstd=rstd) == F.Success
    torch.cuda.synchronize()
    v, w64, b64 = x.double(), w.double(), b.double()
    over = lambda t: t.mean(-1, keepdim=True)  # noqa: E731
    mu = over(v)
    r = 1 / torch.sqrt(over((v - mu).square()) + EPS)
    xh = (v - mu) * r
    off, lost = chain(n) * over(v.abs()), (v.abs() + mu.abs()) * R
    less = 0.5 * chain(n) + 4 * R + r.square() * (off.square() + over(2 * (v - mu).abs() * lost))
    want = xh * w64 + b64
    within(y, want, rounded(want, dtype) + w64.abs() * (xh.abs() * (less + 4 * R) + r * (off + lost)) + R * (b64.abs() + 2 * want.abs()))
    within(mean, mu[:, 0], (off + R * mu.abs())[:, 0])
    within(rstd, r[:, 0], (r * less)[:, 0])

    gw, gb = (torch.full((n,), 7.0, dtype=kind, device=dev()) for _ in range(2))
    assert F.layer_norm_bprop(x, w, mean, rstd, g, y, gw, gb, space(1)) == F.Success
    torch.cuda.synchronize()
    mu, r, d = mean.double()[:, None], rstd.double()[:, None], g.double()
    xh, h = (v - mu) * r, d * w64
    exh = R * ((v.abs() + mu.abs()) * r + 2 * xh.abs())
    s1, s2 = over(h), over(h * xh)
    e1, e2 = chain(n) * over(h.abs()), chain(n) * over((h * xh).abs()) + over(h.abs() * exh)
    want = r * (h - s1 - xh * s2)
    within(y, want, rounded(want, dtype) + r * (4 * R * (h.abs() + s1.abs() + (xh * s2).abs()) + e1 + xh.abs() * e2 + exh * s2.abs()))
    want = (d * xh).sum(0)
    within(gw, want, rounded(want, kind) + chain(m) * (d * xh).abs().sum(0) + (d.abs() * exh).sum(0))
    want = d.sum(0)
    within(gb, want, rounded(want, kind) + chain(m) * d.abs().sum(0))


# 1024 rows and more: a wave to a row, two and four words to a lane
@pytest.mark.parametrize("dtype", TYPES, ids=NAMES.get)
@pytest.mark.parametrize("gap", [0, 7])
@pytest.mark.parametrize("shape", [(1024, 257), (1025, 300), (1100, 512), (1027, 513), (1200, 600), (1031, 777), (1024, 1024), (1500, 1025),
                                   (1033, 1300), (2100, 2041), (1025, 2048), (1024, 2049)], ids=str)
def test_several_words_to_a_lane(shape, gap, dtype):
    check(*shape, dtype, gap=gap)
    check(*shape, dtype, kind=dtype, gap=gap)


# results of 48 MiB and more, from rows of a few lanes to rows that take a workgroup
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=NAMES.get)
@pytest.mark.parametrize("words", [1, 3, 4, 7, 13, 30, 61, 64, 65, 110, 129, 200, 256, 300, 505, 999, 1025, 2040, 2049, 4090, 4097])
def test_results_that_leave_past_the_caches(words, dtype):
    size = 4 if dtype == torch.float32 else 2
    n = words * 16 // size - (words % 2)  # every second one ends inside a word
    check((48 << 20) // (n * size) + 2, n, dtype, gap=(words // 2) % 2 * 5)

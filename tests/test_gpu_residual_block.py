"""The operators as examples/residual_block.py runs them together: its loss falls, and the gradients of its first step
are those of the same block in 64 bits with torch's own differentiation."""
import importlib.util
import math
import os

import pytest
import torch

from operators_util import halves

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
spec = importlib.util.spec_from_file_location("residual_block", os.path.join(ROOT, "examples", "residual_block.py"))
E = importlib.util.module_from_spec(spec)
spec.loader.exec_module(E)


def test_the_loss_falls():
    block = E.ResidualBlock()
    losses = E.train(block, *E.data(block), 20)
    assert all(math.isfinite(v) for v in losses)
    assert losses[-1] < 0.9 * losses[0]
    # the same seeds draw the same masks, and no sum depends on the order in which workgroups end
    again = E.ResidualBlock()
    assert E.train(again, *E.data(again), 20) == losses


def test_gradients_of_a_step():
    block = E.ResidualBlock(batch=3, cin=5, channels=12, size=11, kernel=3, groups=3, p=0.25, seed=4)
    x, target = E.data(block, batch=3, cin=5, size=11)
    off = block.forward(x, 6) - target
    block.backward(x, off * (2 / off.numel()), 6)
    p = {k: v.cpu().double().requires_grad_() for k, v in block.params.items()}
    c = torch.nn.functional.conv2d(x.cpu().double(), p["filters"])
    b, ch = c.shape[:2]
    flat = c.reshape(b, 3, -1)
    xh = ((flat - flat.mean(-1, keepdim=True)) / (flat.var(-1, unbiased=False, keepdim=True) + 1e-5).sqrt()).view_as(c)
    h = torch.nn.functional.silu(xh * p["gamma"].view(1, ch, 1, 1) + p["beta"].view(1, ch, 1, 1))
    h = h.permute(0, 2, 3, 1).reshape(-1, ch)
    z = h @ p["weight"].t() + p["bias"]
    keep = (halves(z.numel(), 4, 6) >= 16384).view(z.shape)
    y = torch.where(keep, torch.nn.functional.gelu(z) / 0.75, torch.zeros_like(z)) + h
    loss = (y - target.cpu().double()).square().mean()
    loss.backward()
    assert abs(float(off.square().mean()) - loss.item()) < 1e-5 * loss.item()
    for k, v in p.items():
        # fp32 through five operators, and the convolution's transforms at 1e-4
        far = float((block.grads[k].cpu().double() - v.grad).norm() / v.grad.norm())
        assert far < 1e-4, "%s: %.2e" % (k, far)
